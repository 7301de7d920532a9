// kda_rotary.hip -- rotary positions on several axes, for queries and keys in one launch.
//
// A pair (x, y) of channels turns by the angle of its axis' position p and its own
// frequency: (x cos - y sin, x sin + y cos); the gradient turns back.  Every element is
// read and written once, which is what bounds it.  Angles are formed in fp64 as
// fractions of a turn (in fp32 a position of 2^20 leaves an angle off by a 16th of
// a radian), cos and sin in fp32.  A thread forms those of V pairs of one token once
// and takes them through the token's heads (or a part of them, where there are few
// tokens), four rows' loads in flight: their cost is shared and nothing goes through LDS.
// Measured: 65537 x (16 + 4) x 128 bf16 129 us, 5.2 TB/s (a row at a time 159); 25088 x
// (6 + 6) x 64 in three sections 17 us, 4.5 TB/s; 196 x 12 x 64 4.8 us.
#include "kda_hip.h"
#include "kda_internal.h"

namespace kda {

namespace {

constexpr int MAX_D = 256, AXES = KDA_ROTARY_AXES;

struct RotaryArgs {
    const void *src[2];
    void* dst[2];
    int64_t batch[2], token[2], head[2];
    int heads[2];
    const void* pos;
    int64_t p_axis, p_batch, p_token;
    int type;
    uint32_t grid_h, grid_w;
    int64_t start;
    uint32_t T, groups, parts, unit0, units;  // groups of V pairs a row; parts of `per` heads each; units [unit0, units) of B T parts
    int D, per;
    float sign;
    int axes, ends[AXES];              // pairs before each axis' end
    uint16_t lo[MAX_D / 2];            // a group's first channel, and (halves) the other members'
    uint16_t hi[MAX_D / 2];
    double turns[MAX_D / 2];
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};
template <typename ST>
__device__ __forceinline__ float to_f(ST x) {
    if constexpr (std::is_same<ST, float>::value) return x;
    else return bf2f(x);
}
template <typename ST>
__device__ __forceinline__ ST of_f(float x) {
    if constexpr (std::is_same<ST, float>::value) return x;
    else return f2bf(x);
}

// (x, y) turned.  No angle: copied, whatever the other one is, and a zero with its sign.
__device__ __forceinline__ void turned(float& x, float& y, float c, float s) {
    const float u = s == 0.f ? x * c : fmaf(x, c, -(y * s)), v = s == 0.f ? y * c : fmaf(y, c, x * s);
    x = u;
    y = v;
}

// V pairs of one row: channels lo and hi (halves), or from lo on
template <typename ST, int V, bool HALVES>
struct Row {
    static constexpr int N = HALVES ? V : V == 1 ? 1 : 16 / (int)sizeof(ST), M = 2 * V / N;   // channels a piece, pieces
    typedef Vec<ST, N> P;
    P p[M];
    __device__ __forceinline__ static int at(int i, int lo, int hi) { return HALVES ? (i ? hi : lo) : lo + i * N; }
    __device__ __forceinline__ void load(const ST* s, int lo, int hi) {
#pragma unroll
        for (int i = 0; i < M; ++i) p[i] = *reinterpret_cast<const P*>(s + at(i, lo, hi));
    }
    __device__ __forceinline__ void store(ST* d, int lo, int hi, const float (&cs)[V], const float (&sn)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            ST &x = HALVES ? p[0].v[i] : p[2 * i / N].v[2 * i % N], &y = HALVES ? p[1].v[i] : p[(2 * i + 1) / N].v[(2 * i + 1) % N];
            float xf = to_f<ST>(x), yf = to_f<ST>(y);
            turned(xf, yf, cs[i], sn[i]);
            x = of_f<ST>(xf);
            y = of_f<ST>(yf);
        }
#pragma unroll
        for (int i = 0; i < M; ++i) *reinterpret_cast<P*>(d + at(i, lo, hi)) = p[i];
    }
};

template <typename ST, int V, bool HALVES>
__global__ __launch_bounds__(256) void kda_rotary_kernel(const RotaryArgs a) {
    const uint32_t rows = 256u / a.groups, group = threadIdx.x % a.groups, unit = a.unit0 + blockIdx.x * rows + threadIdx.x / a.groups;
    if (threadIdx.x >= rows * a.groups || unit >= a.units) return;
    const uint32_t tok = a.parts == 1 ? unit : unit / a.parts, part = unit - tok * a.parts;
    const uint32_t b = tok / a.T, t = tok - b * a.T;

    float cs[V], sn[V];
    double p[AXES];
#pragma unroll
    for (int x = 0; x < AXES; ++x) {
        p[x] = 0.0;
        if (x < a.axes) {
            if (a.pos) {
                const int64_t at = x * a.p_axis + (int64_t)b * a.p_batch + (int64_t)t * a.p_token;
                p[x] = a.type == 0   ? (double)static_cast<const int32_t*>(a.pos)[at]
                       : a.type == 1 ? (double)static_cast<const int64_t*>(a.pos)[at]
                                     : (double)static_cast<const float*>(a.pos)[at];
            } else {
                const int64_t n = a.start + t;
                int64_t row, frame;
                if (n >> 32) {
                    row = n / a.grid_w;
                    frame = row / a.grid_h;
                } else {
                    row = (uint32_t)n / a.grid_w;
                    frame = (uint32_t)row / a.grid_h;
                }
                p[x] = x == 0 ? (double)frame : x == 1 ? (double)(row - frame * a.grid_h) : (double)(n - row * a.grid_w);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int pair = (int)group * V + i;
        double pos = 0.0;
#pragma unroll
        for (int x = AXES - 1; x >= 0; --x)
            if (x < a.axes && pair < a.ends[x]) pos = p[x];
        const double turn = pos * a.turns[pair];
        const float f = (float)(turn - rint(turn));
        sincospif(2.f * f, &sn[i], &cs[i]);
        sn[i] *= a.sign;
    }
    const int lo = a.lo[group], hi = HALVES ? a.hi[group] : 0;
    const int first = (int)part * a.per, behind = min(first + a.per, a.heads[0] + a.heads[1]);
    // (the tensors in turn: chosen by the head, their addresses would be loads in front of each row's)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int skip = k ? a.heads[0] : 0, end = min(behind - skip, a.heads[k]);
        const ST* s = static_cast<const ST*>(a.src[k]) + (int64_t)b * a.batch[k] + (int64_t)t * a.token[k];
        ST* d = static_cast<ST*>(a.dst[k]) + (int64_t)tok * a.heads[k] * a.D;
        int h = max(first - skip, 0);
        auto batch = [&](auto size) {   // that many rows' loads, then their stores
            constexpr int R = size();
            for (; h + R <= end; h += R) {
                Row<ST, V, HALVES> r[R];
#pragma unroll
                for (int i = 0; i < R; ++i) r[i].load(s + (h + i) * a.head[k], lo, hi);
#pragma unroll
                for (int i = 0; i < R; ++i) r[i].store(d + (int64_t)(h + i) * a.D, lo, hi, cs, sn);
            }
        };
        batch(std::integral_constant<int, 4>());
        batch(std::integral_constant<int, 2>());
        batch(std::integral_constant<int, 1>());
    }
}

template <typename ST, int V, bool HALVES>
hipError_t launch(RotaryArgs a, hipStream_t st) {
    const uint32_t rows = 256u / a.groups;
    // (a launch has fewer than 2^32 threads)
    for (uint32_t blocks = (a.units + rows - 1) / rows; blocks;) {
        const uint32_t n = std::min(blocks, 1u << 23);
        hipLaunchKernelGGL((kda_rotary_kernel<ST, V, HALVES>), dim3(n), dim3(256), 0, st, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        a.unit0 += n * rows;
        blocks -= n;
    }
    return hipSuccess;
}

}  // namespace

}  // namespace kda

using namespace kda;

extern "C" int kda_rotary(const kda_rotary_args* args, void* stream) {
    if (!args) return api_fail(KDA_E_INVALID, "args is NULL");
    const kda_rotary_args& r = *args;
    if (r.dtype != KDA_DTYPE_F32 && r.dtype != KDA_DTYPE_BF16)
        return api_fail(KDA_E_UNSUPPORTED, "dtype=%lld: expected 0 (fp32) or 1 (bf16)", (long long)r.dtype);
    if (r.D < 2 || r.D > MAX_D || r.D % 2 != 0)
        return api_fail(KDA_E_UNSUPPORTED, "D=%lld: expected an even number from 2 to %d", (long long)r.D, MAX_D);
    if (r.B < 0 || r.T < 0 || r.B > 0x7fffffff || r.T > 0x7fffffff || r.B * r.T > 0x7fffffff)
        return api_fail(KDA_E_INVALID, "B=%lld T=%lld", (long long)r.B, (long long)r.T);
    if (r.axes < 1 || r.axes > AXES || (!r.positions && r.axes > 3))
        return api_fail(KDA_E_INVALID, "axes=%lld: expected 1 to %d", (long long)r.axes, r.positions ? AXES : 3);
    if (!r.positions && (r.grid_h < 1 || r.grid_w < 1 || r.grid_h > 0x7fffffff || r.grid_w > 0x7fffffff || r.start < 0))
        return api_fail(KDA_E_INVALID, "grid %lld x %lld from %lld, and no positions", (long long)r.grid_h, (long long)r.grid_w,
                        (long long)r.start);
    if (r.positions && (r.type < 0 || r.type > 2)) return api_fail(KDA_E_UNSUPPORTED, "type=%lld: expected 0, 1 or 2", (long long)r.type);
    RotaryArgs a = {};
    const int es = r.dtype == KDA_DTYPE_BF16 ? 2 : 4, halves = !r.interleaved;
    // the widest pieces that every operand and section is made of
    int V = halves && es == 2 ? 8 : 4, at = 0;
    const int m = halves ? 1 : 2;   // elements of a pair in a piece
    const auto fits = [&](int64_t n) { while (V > 1 && n % (m * V) != 0) V = V == 8 ? 4 : 1; };
    for (int x = 0; x < r.axes; ++x) {
        if (r.sections[x] < 0 || r.sections[x] % 2 != 0 || (at += (int)r.sections[x]) > r.D)
            return api_fail(KDA_E_INVALID, "sections[%d]=%lld: even, and no more than D=%lld together", x, (long long)r.sections[x],
                            (long long)r.D);
        a.ends[x] = at / 2;
        if (halves) fits(r.sections[x] / 2);
    }
    if (at && !r.turns) return api_fail(KDA_E_INVALID, "turns is NULL");
    fits(halves ? (r.D - at) / 2 : r.D);
    const kda_decay_rows* in[2] = {&r.q, &r.k};
    void* out[2] = {r.q_out, r.k_out};
    for (int j = 0; j < 2; ++j) {
        if (j && !in[j]->p) continue;
        const char* name = j ? "k" : "q";
        if (in[j]->heads < 1 || in[j]->heads > 65535) return api_fail(KDA_E_INVALID, "%s has %lld heads", name, (long long)in[j]->heads);
        if (r.B * r.T > 0 && (!in[j]->p || !out[j] || ((uintptr_t)in[j]->p | (uintptr_t)out[j]) % es != 0))
            return api_fail(KDA_E_INVALID, "%s or its output is NULL or not aligned to its elements", name);
        for (const int64_t n : {(int64_t)((uintptr_t)in[j]->p / es), (int64_t)((uintptr_t)out[j] / es), in[j]->batch, in[j]->token,
                                in[j]->head})
            fits(n);
        a.src[j] = in[j]->p; a.dst[j] = out[j];
        a.batch[j] = in[j]->batch; a.token[j] = in[j]->token; a.head[j] = in[j]->head;
        a.heads[j] = (int)in[j]->heads;
    }
    if (r.B * r.T == 0) return KDA_OK;
    a.pos = r.positions;
    a.p_axis = r.axis; a.p_batch = r.batch; a.p_token = r.token;
    a.type = (int)r.type; a.grid_h = (uint32_t)r.grid_h; a.grid_w = (uint32_t)r.grid_w; a.start = r.start;
    a.T = (uint32_t)r.T; a.D = (int)r.D;
    a.groups = (uint32_t)(r.D / 2 / V);
    a.sign = r.sign < 0 ? -1.f : 1.f;
    a.axes = (int)r.axes;
    for (int p = 0; p < r.D / 2; ++p) a.turns[p] = p < at / 2 ? r.turns[p] : 0.0;
    for (int g = 0; g < (int)a.groups; ++g) {
        const int p = g * V;
        a.lo[g] = (uint16_t)(2 * p);
        if (!halves) continue;
        int x = 0, begin = 0;
        while (x < r.axes && p >= a.ends[x]) begin = a.ends[x++];
        const int len = (x < r.axes ? a.ends[x] : (int)r.D / 2) - begin;   // pairs of the section
        a.lo[g] = (uint16_t)(2 * begin + (p - begin));
        a.hi[g] = (uint16_t)(a.lo[g] + len);
    }
    // a token's heads in parts where tokens alone leave the card empty
    const int heads = a.heads[0] + a.heads[1];
    const int64_t tokens = r.B * r.T;
    int parts = (int)std::min<int64_t>(heads, std::max<int64_t>(1, 262144 / (tokens * a.groups)));
    a.per = (heads + parts - 1) / parts;
    parts = (heads + a.per - 1) / a.per;
    a.parts = (uint32_t)parts;
    a.units = (uint32_t)(tokens * parts);   // (parts > 1 only below 2^18 threads)
    const hipStream_t st = static_cast<hipStream_t>(stream);
    hipError_t e;
    if (es == 2) {
        if (halves) e = V == 8 ? launch<uint16_t, 8, true>(a, st) : V == 4 ? launch<uint16_t, 4, true>(a, st) : launch<uint16_t, 1, true>(a, st);
        else e = V == 4 ? launch<uint16_t, 4, false>(a, st) : launch<uint16_t, 1, false>(a, st);
    } else {
        if (halves) e = V == 4 ? launch<float, 4, true>(a, st) : launch<float, 1, true>(a, st);
        else e = V == 4 ? launch<float, 4, false>(a, st) : launch<float, 1, false>(a, st);
    }
    return e == hipSuccess ? KDA_OK : api_hip_fail(e, "kda_rotary");
}
