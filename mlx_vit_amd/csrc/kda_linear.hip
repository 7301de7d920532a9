// kda_linear.hip -- linear maps with their epilogue: y = act(x W^T + b) + r, the
// products of their backward pass, and the C ABI around them.
//
//   forward   y[m][n] = act(sum_k x[m][k] W[n][k] + b[n]) + r[m][n], z (before act) on request
//   dgrad     dx[m][k] = (sum_n dz[m][n] W[n][k]) * act'(zin[m][k])
//   wgrad     dW[n][k] = sum_m dz[m][n] x[m][k], db[n] = sum_m dz[m][n]   (fp32; bf16: kda_wgrad.hip)
//
// All are one product C[m][n] = sum_k A[m][k] B(k, n); the operand whose rows
// run across the contracted index (W in dgrad, both in wgrad) reaches the MFMA
// through transposing LDS reads, so nothing is transposed in memory.
//
// What bounds them: 2 M N K operations against the matrix unit (1391 to 1634
// TFLOP/s of bf16 in an 8192^3 product by the library here, as the card's clock
// allows), the rows' bytes where K or N is a few hundred (the 25088 x 1536 hidden layer of a block: 77 MB, 15 us a pass at a
// copy's 5.1 TB/s), the epilogue's instructions beside them, and a load's latency
// where there are fewer tiles than CUs.  Measured (forward, bias and activation
// within, twenty in a graph): 16384 x 2048 -> 8192 gelu 495 us, 1111 TFLOP/s (without
// activation 453; the library's bare product 373); 25088 x 384 -> 1536 gelu 55 us and
// 1536 -> 384 with the residual 39 (the library's bare products 56 and 32); 196 x 384 ->
// 1536 4.5 us; 1 x 384 -> 174 3.2 us.
#include "kda_hip.h"
#include "kda_internal.h"

namespace kda {

namespace {

struct GemmArgs {
    const void *a, *b;
    void* c;
    const void *bias, *res, *zin;
    void* zout;
    int64_t lda, ldb, ldc, ldr, ldzi, ldzo;
    int M, N, K;
    int mt, nt;             // tiles
    int vec;                // C, bias, res, zin, zout: 16-byte accesses, N % 8 == 0 (wgrad's parts: N % 4)
    int vec_a, vec_b;       // fp32: rows of A, B can be read four floats at a time
    int splits, k_per;      // fp32 wgrad: parts of the contracted index, k_per (a multiple of the step) each
    float *part, *bpart;    // and their partial sums, [split][M][N] and [split][M]; dgrad with an activation:
                            // bpart, C's column sums before rounding, [row of waves][N]
};

// ----------------------------------------------------------------------------
// activations: 0 none, 1 gelu (z Phi(z)), 2 silu (z sigma(z))
// ----------------------------------------------------------------------------

// Results rounded to bf16 take a fit for gelu, because the epilogue is VALU-bound
// there: with e = e^{-z^2/2}, t = 1 / (1 + 0.338 |z|),
//   Phi(-|z|) = e P(t),  P the minimax polynomial of degree 5 for e^{z^2/2} Phi(-|z|),
// 1.6e-6 of its value off up to |z| = 3.5 and 1e-5 up to 6, so that
//   gelu  = z Phi(z): within 1e-5 of its value down to z = -6 (a 200th of a bf16 half
//           step), where it is 6e-9; 1e-11 below;
//   gelu' = Phi(z) + z phi(z), below zero e (P(t) - |z| / sqrt(2 pi)): within 3e-6 of
//           its terms, so a unit far below zero gets a gradient that vanishes with e.
// 20 and 21 issue slots a value (exp2 and rcp four each); a degree less is off by 1e-4.
// fp32 results take the same with a polynomial of degree 8 in w = 0.36 |z| / (1 + 0.36
// |z|), which is 1/2 at w = 0: 8.4e-9 of its value off up to |z| = 2.5, so that what is
// left is fp32 arithmetic (measured: Phi within 1.0e-7, at z = -5 within 2e-6 of its
// value; (1 + erf) / 2 of fp32 values within 1.1e-7, of which nothing is left at -5).
// sigma of an fp32 result takes the accurate functions: the rounding of log2(e) z alone
// puts |z| 2^-24 of its value on the other (a 1000th of a bf16 half step at z = -40)
template <bool F32>
__device__ __forceinline__ float sigma(float z) {
    if constexpr (F32) return 1.f / (1.f + expf(-z));
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
}
// e^{z^2/2} Phi(-a), a = |z|
template <bool F32>
__device__ __forceinline__ float tail(float a) {
    if constexpr (F32) {
        const float c = 0.36f * a, w = c * __builtin_amdgcn_rcpf(1.f + c);
        float p = fmaf(-2.8067263e-02f, w, 4.4282120e-02f);
        p = fmaf(p, w, 2.8220793e-02f);
        p = fmaf(p, w, -6.2233186e-03f);
        p = fmaf(p, w, -1.5057352e-01f);
        p = fmaf(p, w, -1.0048330e-01f);
        p = fmaf(p, w, 8.2085037e-01f);
        p = fmaf(p, w, -1.1081734f);
        return fmaf(p, w, 0.5f);
    } else {
        const float t = __builtin_amdgcn_rcpf(fmaf(0.338f, a, 1.f));
        float p = fmaf(-1.1298490e-01f, t, 3.6227307e-01f);
        p = fmaf(p, t, -8.4105216e-02f);
        p = fmaf(p, t, 2.1490058e-01f);
        p = fmaf(p, t, 1.1856889e-01f);
        return fmaf(p, t, 1.3469618e-03f);
    }
}
// An infinite z is multiplied with 0 = e: by a finite value; e keeps a NaN.
constexpr float FAR = 64.f;
template <bool F32>
__device__ __forceinline__ float gelu(float z) {
    const float a = F32 ? fminf(fabsf(z), FAR) : fabsf(z);   // (bf16's tail is finite everywhere)
    const float x = __builtin_amdgcn_exp2f(-0.72134752044448170f * (z * z)) * tail<F32>(a);
    return z * (z < 0.f ? x : 1.f - x);
}
template <bool F32>
__device__ __forceinline__ float gelu_grad(float z) {
    const float a = fminf(fabsf(z), FAR), e = __builtin_amdgcn_exp2f(-0.72134752044448170f * (z * z));
    const float x = e * fmaf(-0.39894228040143268f, a, tail<F32>(a));
    return z < 0.f ? x : 1.f - x;
}
// F32: for results kept in fp32
template <int ACT, bool F32>
__device__ __forceinline__ float act(float z) {
    if constexpr (ACT == 1) {
        return gelu<F32>(z);
    } else if constexpr (ACT == 2) {
        return z * sigma<F32>(z);
    } else {
        return z;
    }
}
template <int ACT, bool F32>
__device__ __forceinline__ float act_grad(float z) {
    if constexpr (ACT == 1) {
        return gelu_grad<F32>(z);
    } else if constexpr (ACT == 2) {
        // (bf16's z may be past its range: infinite)
        if constexpr (!F32) z = __builtin_elementwise_maximum(__builtin_elementwise_minimum(z, 65504.f), -65504.f);
        const float s = sigma<F32>(z);
        return s * fmaf(z, 1.f - s, 1.f);
    } else {
        return 1.f;
    }
}

// four columns at p (n of them exist): vec: one access
template <typename T>
__device__ __forceinline__ float4 ldc4(const T* p, int n, bool vec) {
    if (vec) return ld4<T>(p);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (n > 0) v.x = ld1<T>(p);
    if (n > 1) v.y = ld1<T>(p + 1);
    if (n > 2) v.z = ld1<T>(p + 2);
    if (n > 3) v.w = ld1<T>(p + 3);
    return v;
}
template <typename T>
__device__ __forceinline__ void stc4(T* p, const float4& v, int n, bool vec) {
    if (vec) {
        if constexpr (std::is_same<T, float>::value) *reinterpret_cast<float4*>(p) = v;
        else *reinterpret_cast<uint2*>(p) = make_uint2(pack2bf(v.x, v.y), pack2bf(v.z, v.w));
        return;
    }
    if (n > 0) st1<T>(p, v.x);
    if (n > 1) st1<T>(p + 1, v.y);
    if (n > 2) st1<T>(p + 2, v.z);
    if (n > 3) st1<T>(p + 3, v.w);
}

// What z is kept in beside bf16 results: fp16, three more bits in the same room.  As
// bf16 it put a fifth of its rounding's size on top of dz's own in every gradient
// (off by 1.46 half steps where 1.41 is two roundings).  Past fp16's range it is
// infinite, where both derivatives are at their ends.
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
template <typename T>
using Pre = typename std::conditional<std::is_same<T, float>::value, float, _Float16>::type;

// eight columns at p (n of them exist): vec: 16-byte accesses
template <typename T>
__device__ __forceinline__ void ldc8(const T* p, int n, bool vec, float (&v)[8]) {
    if constexpr (std::is_same<T, _Float16>::value) {
        if (vec) {
            const half8v h = *reinterpret_cast<const half8v*>(p);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (float)h[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < n ? (float)p[e] : 0.f;
        }
        return;
    } else {
        if (vec) {
            if constexpr (std::is_same<T, float>::value) {
                const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
                v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
                v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
            } else {
                const uint4 x = *reinterpret_cast<const uint4*>(p);
                v[0] = bf_lo(x.x); v[1] = bf_hi(x.x); v[2] = bf_lo(x.y); v[3] = bf_hi(x.y);
                v[4] = bf_lo(x.z); v[5] = bf_hi(x.z); v[6] = bf_lo(x.w); v[7] = bf_hi(x.w);
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? ld1<T>(p + e) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void stc8(T* p, const float (&v)[8], int n, bool vec) {
    if constexpr (std::is_same<T, _Float16>::value) {
        half8v h;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = (_Float16)v[e];
        if (vec) *reinterpret_cast<half8v*>(p) = h;
        else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < n) p[e] = h[e];
    } else {
        if (vec) {
            if constexpr (std::is_same<T, float>::value) {
                *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                *reinterpret_cast<uint4*>(p) =
                    make_uint4(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7]));
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) st1<T>(p + e, v[e]);
    }
}

// Where an epilogue reads and writes: column n of row m in each matrix, moved down a
// few rows at a time (a multiplication by each row stride for every eight values
// was a fifth of the epilogue's instructions)
template <typename T, bool DG>
struct Place {
    typedef typename std::conditional<DG, Pre<T>, T>::type In;
    const In* in;   // DG: zin, else the residual
    Pre<T>* z;
    T* c;
    __device__ __forceinline__ Place(const GemmArgs& a, int m, int n)
        : in(static_cast<const In*>(DG ? a.zin : a.res) + (size_t)m * (DG ? a.ldzi : a.ldr) + n),
          z(static_cast<Pre<T>*>(a.zout) + (size_t)m * a.ldzo + n), c(static_cast<T*>(a.c) + (size_t)m * a.ldc + n) {}
    __device__ __forceinline__ void down(const GemmArgs& a, int rows) {
        in += rows * (DG ? a.ldzi : a.ldr);
        if constexpr (!DG) z += rows * a.ldzo;
        c += rows * a.ldc;
    }
};

// The epilogue of eight columns from `at`, of which `left` exist.  DG: times act'(zin)
// and added to `bias`, the rows' sums (no activation: nothing); else bias, z out,
// activation, residual
template <typename T, int ACT, bool DG, bool F32>
__device__ __forceinline__ void finish8(const GemmArgs& a, const Place<T, DG>& at, int left, float (&v)[8], float (&bias)[8]) {
    const bool vec = a.vec;
    float t[8];
    if constexpr (DG) {
        if constexpr (ACT != 0) {
            ldc8<Pre<T>>(at.in, left, vec, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] *= act_grad<ACT, F32>(t[e]);
                bias[e] += v[e];
            }
        }
    } else {
        if (a.res) ldc8<T>(at.in, left, vec, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += bias[e];
        if (a.zout) stc8<Pre<T>>(at.z, v, left, vec);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = act<ACT, F32>(v[e]);
        if (a.res)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += t[e];
    }
    stc8<T>(at.c, v, left, vec);
}
template <typename T, bool DG>
__device__ __forceinline__ void bias8(const GemmArgs& a, int n, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (!DG && a.bias && n < a.N) ldc8<T>(static_cast<const T*>(a.bias) + n, a.N - n, a.vec, v);
}

// The epilogue of a wave's 16 FN columns from n0 and 16 FM rows from m0, R rows (16
// or 32) at a time through 64 FN R bytes of LDS of its own: the accumulators hold
// four columns of 16 rows a fragment, and leave as whole rows (128 bytes of bf16
// at FN = 4) of 16-byte pieces.  The 16-byte piece c of row r lies at c ^ (r's low
// bits), so that both the fragments' writes (16 rows of a piece) and the reads
// are spread over the banks.  acc[i][j]: columns 16 i, rows 16 j.
template <typename T, int ACT, bool DG, bool F32, int R, int FN, int FM>
__device__ __forceinline__ void finish_wave(const GemmArgs& a, int m0, int n0, const f32x4 (&acc)[FN][FM], char* lds,
                                            int wave_row = 0) {
    constexpr int RB = 64 * FN, KEY = 4 * FN - 1, LR = 2 * FN, RI = 64 / LR;   // row bytes, lanes a row, rows a read
    const int l = lane_id(), r16 = l & 15, g4 = l >> 4, q = l % LR;
    const int n = n0 + 8 * q;
    float bias[8];
    bias8<T, DG>(a, n, bias);
    int m = m0 + l / LR;
    Place<T, DG> at(a, m, n);
#pragma unroll
    for (int h = 0; h < FM; h += R / 16) {
        wave_sync();   // the last part's reads come first
#pragma unroll
        for (int j = h; j < h + R / 16; ++j) {
            const int r = 16 * (j - h) + r16;
#pragma unroll
            for (int i = 0; i < FN; ++i)
                *reinterpret_cast<f32x4*>(lds + RB * r + (((4 * i + g4) ^ (r16 & KEY)) << 4)) = acc[i][j];
        }
        wave_sync();
#pragma unroll
        for (int it = 0; it < R / RI; ++it) {
            const int r = RI * it + l / LR;
            const f32x4 x = *reinterpret_cast<const f32x4*>(lds + RB * r + (((2 * q) ^ (r & KEY)) << 4));
            const f32x4 y = *reinterpret_cast<const f32x4*>(lds + RB * r + (((2 * q + 1) ^ (r & KEY)) << 4));
            float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            if (m < a.M && n < a.N) finish8<T, ACT, DG, F32>(a, at, a.N - n, v, bias);
            m += RI;
            at.down(a, RI);
        }
    }
    if constexpr (DG && ACT != 0) {
        if (a.bpart) {   // the lanes of a column
#pragma unroll
            for (int e = 0; e < 8; ++e) {
#pragma unroll
                for (int d = LR; d < 64; d <<= 1) bias[e] += __shfl_xor(bias[e], d);
                if (l < LR && n + e < a.N) a.bpart[(size_t)wave_row * a.N + n + e] = bias[e];
            }
        }
    }
}

// tile (mi, ni) of block bid: each XCD takes a run of consecutive tiles, ordered
// in groups of 8 tile rows (a column of a group shares B's tile)
__device__ __forceinline__ void tile_of(int bid, int nb, int mt, int nt, int& mi, int& ni) {
    const int xcd = bid % 8, q = nb / 8, rem = nb % 8;
    const int t = xcd * q + min(xcd, rem) + bid / 8;
    const int per = 8 * nt, g = t / per, r = t - g * per, rows = min(8, mt - 8 * g);
    ni = r / rows;
    mi = 8 * g + (r - ni * rows);
}

// ----------------------------------------------------------------------------
// bf16: tiles by LDS DMA
// ----------------------------------------------------------------------------

// chunk key of row r: rows of RB bytes along the contracted index (a fragment
// read takes 16 rows of one chunk), or rows across it (a transposing read takes
// rows 8 g .. 8 g + 3 of 32 bytes; of 128-byte rows two share a bank)
template <int RB>
__device__ __forceinline__ int key_k(int r) {
    // of 64-byte rows: a 16-byte read's 16 lanes are 0-3 and 12-15 of one quarter of the
    // wave and 4-11 of the next, so the four keys pair up accordingly
    return RB == 128 ? (r >> 1) & 7 : -(r >> 2) & 3;
}
__device__ __forceinline__ int key_t(int r) { return ((r & 3) << 1) | (r & 8); }

template <int RB>
__device__ __forceinline__ bf16x8 frag_k(const char* tile, int row0, int chunk) {
    const int l = lane_id(), r = row0 + (l & 15), g = l >> 4;
    return __builtin_bit_cast(bf16x8,
                              *reinterpret_cast<const uint4*>(tile + r * RB + (((chunk + g) ^ key_k<RB>(r)) << 4)));
}
template <int RB>
__device__ __forceinline__ bf16x8 frag_t(const char* tile, int n0, int k0) {
    const int l = lane_id(), j = l & 15, g = l >> 4, r = k0 + 8 * g + (j >> 2), b = 2 * (n0 + 4 * (j & 3));
    const int at = (((b >> 4) ^ (key_t(r) & (RB / 16 - 1))) << 4) + (b & 15);   // row r + 4 has the same key
    const short4v x = ld_tr4(reinterpret_cast<const uint16_t*>(tile + r * RB + at));
    const short4v y = ld_tr4(reinterpret_cast<const uint16_t*>(tile + (r + 4) * RB + at));
    return __builtin_bit_cast(bf16x8, short8v{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]});
}

// This wave's part of a tile's DMA (W waves): ROWS rows of RB bytes; instruction
// i of the tile fills 1 KB.  TR: the rows run across the contracted index.
template <int ROWS, int RB, int W, bool TR>
struct Dma {
    static constexpr int NI = ROWS * RB / 1024, PER = NI / W;
    static_assert(NI % W == 0, "whole instructions for each wave");
    uint32_t off[PER];
    __device__ __forceinline__ static void place(int i, int w, int& r, int& c) {
        const int p = 1024 * (w + W * i) + 16 * lane_id();
        r = p / RB;
        c = ((p % RB) >> 4) ^ (TR ? key_t(r) & (RB / 16 - 1) : key_k<RB>(r));
    }
    // rows and 16-byte chunks past the last read the last (not stored, or zeroed below)
    __device__ __forceinline__ void init(int64_t ld, int last_row, int last_chunk, int w) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int r, c;
            place(i, w, r, c);
            off[i] = (uint32_t)min(r, last_row) * (uint32_t)(2 * ld) + 16u * (uint32_t)min(c, last_chunk);
        }
    }
    __device__ __forceinline__ void issue(const char* base, uint32_t lds, int w) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) dma16_s32(base, off[i], lds + 1024u * (uint32_t)(w + W * i));
    }
};

// Zero the columns (elements) at and past `valid` of a tile of rows along the
// contracted index, or the rows at and past it of one across it
template <int ROWS, int RB, bool TR, int THREADS>
__device__ __forceinline__ void zero_tail(char* tile, int valid) {
    if constexpr (TR) {
        for (int i = threadIdx.x; i < (ROWS - valid) * (RB / 16); i += THREADS)
            *reinterpret_cast<uint4*>(tile + valid * RB + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
    } else {
        for (int i = threadIdx.x; i < ROWS * (RB / 16); i += THREADS) {
            const int r = i / (RB / 16), c = i % (RB / 16), left = valid - 8 * c;   // valid elements of chunk c
            char* p = tile + r * RB + ((c ^ key_k<RB>(r)) << 4);
            if (left <= 0) *reinterpret_cast<uint4*>(p) = make_uint4(0u, 0u, 0u, 0u);
            else
                for (int e = left; e < 8; ++e) reinterpret_cast<uint16_t*>(p)[e] = 0;
        }
    }
}

// C tile of BM x BN by WR x WC waves, 64 of the contracted index a step, NB
// buffers.  BT: B's rows run across the contracted index (dgrad).  WPE: waves a
// SIMD that the registers have to leave room for.
//
// AHEAD: a step is two halves of 32, and a wave reads a half's fragments before the
// products of the half before, so that the matrix unit need not wait for LDS.
// There is one barrier a step, in its middle: by then a wave holds its second
// half in registers and its share of the next step has landed, so behind it the
// next step's first half can be read and this step's buffer filled with the step
// NB after it.  (16384 x 2048 x 8192 in tiles of 128 x 128: 622 -> 526 us.)  It
// takes a second set of fragments, which sixteen waves of 64 x 64 have no
// registers for: there four waves a SIMD hide the reads.  (Eight waves of 128 x 64 with
// fragments a quarter of a step ahead instead: 8192^3 833 us against 865, 16384 x 2048
// -> 8192 499 and 503, but 12544 x 768 -> 3200 92 and 88, where eight waves are fewer for
// the epilogue.)
template <int BM, int BN, int WR, int WC, int WPE, int NB, bool AHEAD, bool BT, int ACT, bool DG>
__global__ __launch_bounds__(64 * WR * WC, WPE) void kda_linear_bf16_kernel(const GemmArgs a) {
    constexpr int BK = 64, W = WR * WC, RBA = 2 * BK, RBB = BT ? 2 * BN : 2 * BK, ROWB = BT ? BK : BN;
    constexpr int SA = BM * RBA, STAGE = SA + ROWB * RBB;
    constexpr int FM = BM / WR / 16, FN = BN / WC / 16;
    static_assert(W * 64 * FN * 32 <= NB * STAGE && FM % 2 == 0 && FN <= 4, "the epilogue's rows");
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), r16 = l & 15, g4 = l >> 4;
    const int wm = (w / WC) * (BM / WR), wn = (w % WC) * (BN / WC);
    int mi, ni;
    tile_of((int)blockIdx.x, (int)gridDim.x, a.mt, a.nt, mi, ni);
    const int m0 = mi * BM, n0 = ni * BN;
    Dma<BM, RBA, W, false> da;
    Dma<ROWB, RBB, W, BT> db;
    constexpr int NOCLAMP = 1 << 20;
    da.init(a.lda, a.M - 1 - m0, NOCLAMP, w);
    if constexpr (BT) db.init(a.ldb, NOCLAMP, (a.N - 1 - n0) / 8, w);
    else db.init(a.ldb, a.N - 1 - n0, NOCLAMP, w);
    constexpr int L = decltype(da)::PER + decltype(db)::PER;
    const uint32_t base = lds_addr(lds);
    const char* ga = static_cast<const char*>(a.a) + (size_t)m0 * (2 * a.lda);
    const char* gb = static_cast<const char*>(a.b) + (BT ? (size_t)n0 * 2 : (size_t)n0 * (2 * a.ldb));
    const int64_t stepb = BT ? 2 * BK * a.ldb : 2 * BK;
    const int steps = a.K / BK, tail = a.K % BK;
    auto issue = [&](int buf) {
        const uint32_t st = base + (uint32_t)(buf * STAGE);
        da.issue(ga, st, w);
        db.issue(gb, st + SA, w);
        ga += 2 * BK;
        gb += stepb;
    };
    f32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = zero4();
    // A fragment's place within its half depends on the lane alone (frag_k's key on
    // r16): buffer and fragment are immediate offsets
    const char *pa[2], *pb[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int at = r16 * 128 + (((4 * h + g4) ^ key_k<128>(r16)) << 4);
        pa[h] = lds + wm * RBA + at;
        pb[h] = lds + SA + wn * 128 + at;   // !BT
    }
    struct Frags {
        bf16x8 a[FM], b[FN];
    };
    auto read = [&](Frags& f, int buf, int h) {
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            if constexpr (BT) f.b[i] = frag_t<RBB>(lds + buf * STAGE + SA, wn + 16 * i, 32 * h);
            else f.b[i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(pb[h] + buf * STAGE + 16 * i * 128));
        }
#pragma unroll
        for (int j = 0; j < FM; ++j)
            f.a[j] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(pa[h] + buf * STAGE + 16 * j * 128));
    };
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
            for (int i = 0; i < FN; ++i)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.b[i], f.a[j], acc[i][j], 0, 0, 0);
    };
    // Before each barrier this wave's share of the step has landed; behind it every
    // wave's has, and every wave has read the step before (AHEAD: its second half is
    // in registers)
    if constexpr (AHEAD) {
        static_assert(NB == 2 || NB == 4, "the waits");
        if (steps > 0) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
                if (b < steps) issue(b);
            if (steps >= NB) dma_wait<(NB - 1) * L>();
            else dma_wait<0>();
            lds_barrier();
            Frags f, g;
            read(f, 0, 0);
            auto step = [&](int s, int buf) {
                read(g, buf, 1);
                multiply(f);
                if (s + 1 < steps) {
                    dma_wait_chunks<L>(min(NB - 2, steps - 2 - s));   // what is issued behind step s + 1
                    lds_barrier();
                    if (s + NB < steps) issue(buf);
                    read(f, (buf + 1) % NB, 0);
                }
                multiply(g);
            };
            int s = 0;
            for (; s + NB <= steps; s += NB)
#pragma unroll
                for (int b = 0; b < NB; ++b) step(s + b, b);
#pragma unroll
            for (int b = 0; b < NB - 1; ++b)
                if (s + b < steps) step(s + b, b);
        }
    } else {
        static_assert(NB == 2, "two buffers");
        if (steps > 0) issue(0);
#pragma unroll 1
        for (int s = 0; s < steps; ++s) {
            dma_wait<0>();
            lds_barrier();
            if (s + 1 < steps) issue(1 - (s & 1));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frags f;
                read(f, s & 1, h);
                multiply(f);
            }
        }
    }
    if (tail > 0) {   // the part of a step: what lies past K zero in both operands
        lds_barrier();
        da.init(a.lda, a.M - 1 - m0, (tail - 1) / 8, w);
        if constexpr (BT) db.init(a.ldb, tail - 1, (a.N - 1 - n0) / 8, w);
        else db.init(a.ldb, a.N - 1 - n0, (tail - 1) / 8, w);
        issue(0);
        dma_wait<0>();
        lds_barrier();
        zero_tail<BM, RBA, false, 64 * W>(lds, tail);
        zero_tail<ROWB, RBB, BT, 64 * W>(lds + SA, tail);
        lds_barrier();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            Frags f;
            read(f, 0, h);
            multiply(f);
        }
    }
    lds_barrier();   // every wave has read the last step
    finish_wave<uint16_t, ACT, DG, false, 32>(a, m0 + wm, n0 + wn, acc, lds + 2048 * FN * w, mi * WR + w / WC);
}

// ----------------------------------------------------------------------------
// fp32: each operand split exactly into three bf16 parts on its way to LDS
// ----------------------------------------------------------------------------

// x = h + m + l, each the next 8 bits of x's 24 (truncation, so nothing
// overflows and every difference is exact); the four values' parts packed.
// An infinite x gives a NaN part: its products are NaN where fp32 arithmetic (and a
// forward in pieces of 16 x 16, see few) may have an infinity.
// flip: the sign bit to change in each.
__device__ __forceinline__ void split3(const float4& x, uint32_t flip, uint2& h, uint2& m, uint2& l) {
    const uint32_t v[4] = {__float_as_uint(x.x) ^ flip, __float_as_uint(x.y) ^ flip, __float_as_uint(x.z) ^ flip,
                           __float_as_uint(x.w) ^ flip};
    uint32_t a[4], b[4], c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        a[e] = v[e] & 0xffff0000u;
        const float r = __uint_as_float(v[e]) - __uint_as_float(a[e]);
        b[e] = __float_as_uint(r) & 0xffff0000u;
        c[e] = __float_as_uint(r - __uint_as_float(b[e]));
    }
    constexpr uint32_t HI = 0x07060302u;   // the high halves of two registers
    h = make_uint2(__builtin_amdgcn_perm(a[1], a[0], HI), __builtin_amdgcn_perm(a[3], a[2], HI));
    m = make_uint2(__builtin_amdgcn_perm(b[1], b[0], HI), __builtin_amdgcn_perm(b[3], b[2], HI));
    l = make_uint2(__builtin_amdgcn_perm(c[1], c[0], HI), __builtin_amdgcn_perm(c[3], c[2], HI));
}

// An EDGE x 32 (or, TR, 32 x EDGE) tile of fp32 rows through TH threads' registers
// into three bf16 planes
template <int EDGE, int TH, bool TR>
struct Stage32 {
    static constexpr int RB = TR ? 2 * EDGE : 64, PLANE = 64 * EDGE, TPR = TR ? EDGE / 4 : 8;   // threads a row
    static constexpr int STEP = TH / TPR, PER = 8 * EDGE / TH;                                  // rows apart, pieces a thread
    float4 v[PER];
    uint32_t off[PER];
    // Byte offsets of this thread's pieces in a whole step; across the contracted
    // index, what is past the last (`edge` exist) reads the last: not stored
    __device__ __forceinline__ void init(int64_t ld, int edge) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            off[i] = 4u * (TR ? (uint32_t)row(i) * (uint32_t)ld + (uint32_t)min(col(), edge - 4)
                              : (uint32_t)min(row(i), edge - 1) * (uint32_t)ld + (uint32_t)col());
    }
    __device__ __forceinline__ void load_whole(const float* base) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            v[i] = *reinterpret_cast<const float4*>(reinterpret_cast<const char*>(base) + off[i]);
    }
    // row and first column of this thread's piece i
    __device__ __forceinline__ static int row(int i) { return (int)threadIdx.x / TPR + STEP * i; }
    __device__ __forceinline__ static int col() { return 4 * ((int)threadIdx.x % TPR); }
    // rows, cols: how many of them exist past (r0, c0); what does not is zero
    __device__ __forceinline__ void load(const float* base, int64_t ld, int rows, int cols, bool vec) {
        const int c = col();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int r = row(i);
            v[i] = r < rows && c < cols ? ldc4<float>(base + (size_t)r * ld + c, cols - c, vec && c + 4 <= cols)
                                        : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    __device__ __forceinline__ void store(char* tile, uint32_t flip) const {
        const int b = 2 * col();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int r = row(i);
            char* p = tile + r * RB + (((b >> 4) ^ (TR ? key_t(r) & (RB / 16 - 1) : key_k<RB>(r))) << 4) + (b & 15);
            uint2 h, m, l;
            split3(v[i], flip, h, m, l);
            *reinterpret_cast<uint2*>(p) = h;
            *reinterpret_cast<uint2*>(p + PLANE) = m;
            *reinterpret_cast<uint2*>(p + 2 * PLANE) = l;
        }
    }
};

// C tile of BM x BN by WR x WC waves, 32 of the contracted index a step.  AT, BT:
// the operand's rows run across the contracted index.  PART: one of a.splits
// parts of it, into a.part (and with a.bpart A's column sums).
//
// Six bf16 products for one: at 1634 TFLOP/s of those no more than 272 of fp32's,
// where the library's fp32 products reach 154 at 8192^3 and 85 at 6272 x 384 <-> 1536.
// Here 6272 x 384 -> 1536 with gelu takes 50 us (147 TFLOP/s), 4096^3 617 (223; the
// library 911).  What bounds it is the way to LDS: each value is loaded, split (nine
// instructions) and stored once a tile, in one buffer, the next step's loads in
// flight over the products.
template <int BM, int BN, int WR, int WC, bool AT, bool BT, int ACT, bool DG, bool PART>
__global__ __launch_bounds__(64 * WR * WC, 2) void kda_linear_f32_kernel(const GemmArgs a) {
    constexpr int BK = 32, TH = 64 * WR * WC, FM = BM / WR / 16, FN = BN / WC / 16;
    constexpr int RBA = AT ? 2 * BM : 64, RBB = BT ? 2 * BN : 64, PA = 64 * BM, PB = 64 * BN, LDS = 3 * (PA + PB);
    static_assert(TH / 64 * 64 * FN * 16 <= LDS, "the epilogue's rows");
    __shared__ __attribute__((aligned(1024))) char lds[LDS];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), r16 = l & 15, g4 = l >> 4;
    const int wm = (w / WC) * (BM / WR), wn = (w % WC) * (BN / WC);
    const int tiles = a.mt * a.nt, split = PART ? (int)blockIdx.x / tiles : 0;
    int mi, ni;
    tile_of((int)blockIdx.x - split * tiles, tiles, a.mt, a.nt, mi, ni);
    const int m0 = mi * BM, n0 = ni * BN;
    const int k0 = PART ? split * a.k_per : 0, k1 = PART ? min(a.K, k0 + a.k_per) : a.K;
    const float *A = static_cast<const float*>(a.a), *B = static_cast<const float*>(a.b);
    Stage32<BM, TH, AT> sa;
    Stage32<BN, TH, BT> sb;
    const bool whole_a = a.vec_a && (!AT || a.M % 4 == 0), whole_b = a.vec_b && (!BT || a.N % 4 == 0);
    sa.init(a.lda, a.M - m0);
    sb.init(a.ldb, a.N - n0);
    auto load = [&](int k) {
        const float* pa = AT ? A + (size_t)k * a.lda + m0 : A + (size_t)m0 * a.lda + k;
        const float* pb = BT ? B + (size_t)k * a.ldb + n0 : B + (size_t)n0 * a.ldb + k;
        const bool whole = k + BK <= k1;
        if (whole && whole_a) sa.load_whole(pa);
        else if constexpr (AT) sa.load(pa, a.lda, k1 - k, a.M - m0, a.vec_a);
        else sa.load(pa, a.lda, a.M - m0, k1 - k, a.vec_a);
        if (whole && whole_b) sb.load_whole(pb);
        else if constexpr (BT) sb.load(pb, a.ldb, k1 - k, a.N - n0, a.vec_b);
        else sb.load(pb, a.ldb, a.N - n0, k1 - k, a.vec_b);
    };
    f32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = zero4();
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool sums = PART && a.bpart && ni == 0;
    load(k0);
    for (int k = k0; k < k1; k += BK) {
        if (k > k0) lds_barrier();   // every wave has read the step before
        const bool odd = ((k - k0) / BK) & 1;
        sa.store(lds, odd ? 0x80000000u : 0u);
        sb.store(lds + 3 * PA, 0u);
        if (sums)
#pragma unroll
            for (int i = 0; i < Stage32<BM, TH, AT>::PER; ++i) {
                sum.x += sa.v[i].x; sum.y += sa.v[i].y; sum.z += sa.v[i].z; sum.w += sa.v[i].w;
            }
        lds_barrier();
        if (k + BK < k1) load(k + BK);
        const float sign = odd ? -1.f : 1.f;
        // products of parts down to 2^-16 of the largest: hh, hm, mh, hl, lh, mm
        bf16x8 fb[3][FN];
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                const char* t = lds + 3 * PA + p * PB;
                if constexpr (BT) fb[p][i] = frag_t<RBB>(t, wn + 16 * i, 0);
                else fb[p][i] = frag_k<RBB>(t, wn + 16 * i, 0);
            }
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            bf16x8 fa[3];
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                if constexpr (AT) fa[p] = frag_t<RBA>(lds + p * PA, wm + 16 * j, 0);
                else fa[p] = frag_k<RBA>(lds + p * PA, wm + 16 * j, 0);
            }
            // The matrix unit rounds its sums downwards, which a sum over many rows of the
            // results shows (a bias gradient over 6272 rows: off by 1.1e-6, 4e-7 in fp32
            // arithmetic).  So a step's products sum from zero, smallest first, join the
            // accumulator by an ordinary addition, and every other step is formed of A
            // negated and subtracted, which turns its rounding upwards.
            f32x4 t[FN];
#pragma unroll
            for (int q = 0; q < 6; ++q) {
                constexpr int QB[6] = {0, 2, 1, 0, 1, 0}, QA[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
                for (int i = 0; i < FN; ++i)
                    t[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[QB[q]][i], fa[QA[q]], q == 0 ? zero4() : t[i], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(sign, t[i][e], acc[i][j][e]);
        }
    }
    if constexpr (PART) {
        float* part = a.part + (size_t)split * a.M * a.N;
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            const int n = n0 + wn + 16 * i + 4 * g4;
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                const int m = m0 + wm + 16 * j + r16;
                if (m < a.M && n < a.N)
                    stc4<float>(part + (size_t)m * a.N + n, make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]),
                                a.N - n, a.vec);
            }
        }
        if (sums) {   // the threads of a column in order
            lds_barrier();
            reinterpret_cast<float4*>(lds)[threadIdx.x] = sum;
            lds_barrier();
            if (threadIdx.x < BM && m0 + (int)threadIdx.x < a.M) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < 4 * TH / BM; ++i) s += reinterpret_cast<const float*>(lds)[BM * i + threadIdx.x];
                a.bpart[(size_t)split * a.M + m0 + threadIdx.x] = s;
            }
        }
    } else {
        constexpr int R = 64 * FN * 32 * TH / 64 <= LDS && FM % 2 == 0 ? 32 : 16;
        lds_barrier();
        finish_wave<float, ACT, DG, true, R>(a, m0 + wm, n0 + wn, acc, lds + 64 * FN * R * w);
    }
}

// dw and db: the parts' sums in order
__global__ __launch_bounds__(256) void kda_linear_sum_parts_kernel(const float* __restrict__ part, const float* __restrict__ bpart,
                                                                   float* __restrict__ dw, float* __restrict__ db, size_t nk,
                                                                   int n, int splits) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < nk + (db ? n : 0); i += (size_t)gridDim.x * 256) {
        const bool w = i < nk;
        const float* src = w ? part + i : bpart + (i - nk);
        const size_t step = w ? nk : (size_t)n;
        float s = src[0];
        for (int q = 1; q < splits; ++q) s += src[q * step];
        if (w) dw[i] = s;
        else db[i - nk] = s;
    }
}

// ----------------------------------------------------------------------------
// few rows: operands straight from memory, the waves share the contracted index
// ----------------------------------------------------------------------------

// eight elements k.. of a row; past K zero
__device__ __forceinline__ bf16x8 row8(const uint16_t* row, int k, int K) {
    short8v v = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (k + e < K) v[e] = (short)row[k + e];
    return __builtin_bit_cast(bf16x8, v);
}
// acc += a step of the contracted index: 32 of it in bf16, 16 in fp32
__device__ __forceinline__ f32x4 few_step(const uint4& x, const uint4& y, f32x4 acc, uint16_t) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, y), __builtin_bit_cast(bf16x8, x), acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 few_step(const uint4& x, const uint4& y, f32x4 acc, float) {
    const float4 p = __builtin_bit_cast(float4, x), q = __builtin_bit_cast(float4, y);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(q.x, p.x, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(q.y, p.y, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(q.z, p.z, acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(q.w, p.w, acc, 0, 0, 0);
}

constexpr int FEW_WAVES = 8, FEW_AHEAD = 4;

// 16 rows x 16 columns a workgroup; wave w takes steps w, w + 8, ... of the
// contracted index, FEW_AHEAD of them loaded before the first is used, and the
// partial tiles meet in LDS.  Bound by the weights' bytes where there are many of
// them (1 x 2048 -> 8192: 33.6 MB in 7.7 us, 4.4 TB/s) and by the chain of a launch, a
// load and the LDS round where there are few (1 x 384 -> 174: 3 us).
template <typename T, int ACT>
__global__ __launch_bounds__(64 * FEW_WAVES) void kda_linear_few_kernel(const GemmArgs a) {
    constexpr int E = 16 / sizeof(T), STEP = 4 * E;   // elements of a lane, of a step
    __shared__ f32x4 part[FEW_WAVES][64];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), r16 = l & 15, g4 = l >> 4;
    const int m0 = 16 * ((int)blockIdx.x / a.nt), n0 = 16 * ((int)blockIdx.x % a.nt);
    const T* ra = static_cast<const T*>(a.a) + (size_t)min(m0 + r16, a.M - 1) * a.lda;
    const T* rb = static_cast<const T*>(a.b) + (size_t)min(n0 + r16, a.N - 1) * a.ldb;
    f32x4 acc = zero4();
    const int whole = a.vec_a && a.vec_b ? a.K / STEP : 0, steps = (a.K + STEP - 1) / STEP;
    int i = w;
    for (; i < whole; i += FEW_AHEAD * FEW_WAVES) {
        uint4 x[FEW_AHEAD], y[FEW_AHEAD];
#pragma unroll
        for (int u = 0; u < FEW_AHEAD; ++u) {
            x[u] = y[u] = make_uint4(0, 0, 0, 0);
            if (i + u * FEW_WAVES < whole) {
                const int k = STEP * (i + u * FEW_WAVES) + E * g4;
                x[u] = *reinterpret_cast<const uint4*>(ra + k);
                y[u] = *reinterpret_cast<const uint4*>(rb + k);
            }
        }
#pragma unroll
        for (int u = 0; u < FEW_AHEAD; ++u) acc = few_step(x[u], y[u], acc, T());
    }
    // a step that ends past K, or all of them where rows begin off 16 bytes
    for (i = whole + (w + FEW_WAVES - whole % FEW_WAVES) % FEW_WAVES; i < steps; i += FEW_WAVES) {
        const int k = STEP * i + E * g4;
        if constexpr (std::is_same<T, float>::value) {
            acc = few_step(__builtin_bit_cast(uint4, ldc4<float>(ra + k, a.K - k, false)),
                           __builtin_bit_cast(uint4, ldc4<float>(rb + k, a.K - k, false)), acc, T());
        } else {
            acc = few_step(__builtin_bit_cast(uint4, row8(ra, k, a.K)), __builtin_bit_cast(uint4, row8(rb, k, a.K)), acc, T());
        }
    }
    part[w][l] = acc;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    // row m, columns n..n+7: two lanes' pieces of each wave
    const int r = threadIdx.x >> 1, c = 2 * (threadIdx.x & 1);
    f32x4 x = part[0][16 * c + r], y = part[0][16 * (c + 1) + r];
#pragma unroll
    for (int i = 1; i < FEW_WAVES; ++i) {
        x += part[i][16 * c + r];
        y += part[i][16 * (c + 1) + r];
    }
    const int m = m0 + r, n = n0 + 4 * c;
    if (m >= a.M || n >= a.N) return;
    float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}, bias[8];
    bias8<T, false>(a, n, bias);
    finish8<T, ACT, false, std::is_same<T, float>::value>(a, Place<T, false>(a, m, n), a.N - n, v, bias);
}

// (Bound by memory: 25088 x 1536 reads and writes 231 MB in 38.5 us, 6.0 TB/s.)
// dz = dy act'(z) (ACT 0: dy), rows of ld_dz elements whose columns from N to the
// next multiple of eight are zero; `rows` rows x 256 columns a workgroup.  part: the
// columns' sums before dz is rounded, [row of workgroups][N].
template <typename T, int ACT>
__global__ __launch_bounds__(256) void kda_linear_act_bwd_kernel(const T* __restrict__ dy, const Pre<T>* __restrict__ z,
                                                                 T* __restrict__ dz, float* __restrict__ part,
                                                                 int64_t ld_dy, int64_t ld_z, int64_t ld_dz, int M, int N,
                                                                 int rows, int vec_in) {
    constexpr bool F32 = std::is_same<T, float>::value;
    __shared__ float sums[8][256];
    const int nb = (N + 255) / 256, rb = (int)blockIdx.x / nb, r0 = threadIdx.x >> 5, c = threadIdx.x & 31;
    const int n = 256 * ((int)blockIdx.x - rb * nb) + 8 * c, left = N - n;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (left > 0)
        for (int m = rows * rb + r0; m < min(M, rows * rb + rows); m += 8) {
            float g[8], x[8];
            ldc8<T>(dy + (size_t)m * ld_dy + n, left, vec_in, g);
            if constexpr (ACT != 0) {
                ldc8<Pre<T>>(z + (size_t)m * ld_z + n, left, vec_in, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    g[e] *= act_grad<ACT, F32>(x[e]);
                    s[e] += g[e];
                }
            }
            stc8<T>(dz + (size_t)m * ld_dz + n, g, 8, true);
        }
    if (!part) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[r0][8 * c + e] = s[e];
    __syncthreads();
    const int col = 256 * ((int)blockIdx.x - rb * nb) + (int)threadIdx.x;
    if (col >= N) return;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += sums[i][threadIdx.x];
    part[(size_t)rb * N + col] = t;
}

// db: the column sums of `rows` rows of partial sums, in a fixed order (32 columns x 8
// runs of rows a workgroup)
__global__ __launch_bounds__(256) void kda_linear_colsum_kernel(const float* __restrict__ part, uint16_t* __restrict__ db,
                                                                int rows, int N) {
    __shared__ float sums[8][32];
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5, n = 32 * (int)blockIdx.x + c;
    float s = 0.f;
    if (n < N) {
        const int per = (rows + 7) / 8, r1 = min(rows, per * (g + 1));
#pragma unroll 4
        for (int r = per * g; r < r1; ++r) s += part[(size_t)r * N + n];
    }
    sums[g][c] = s;
    __syncthreads();
    if (g != 0 || n >= N) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sums[i][c];
    db[n] = f2bf(s);
}

// one or two matrices copied into rows of a multiple of eight columns, zero past theirs
struct PadArgs {
    const uint16_t* src[2];
    uint16_t* dst[2];
    int64_t ld[2];
    int rows[2], cols[2];
};
__global__ __launch_bounds__(256) void kda_linear_pad_kernel(const PadArgs a) {
    const int j = blockIdx.y, groups = (a.cols[j] + 7) / 8;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < (size_t)a.rows[j] * groups; i += (size_t)gridDim.x * 256) {
        const int m = (int)(i / groups), n = 8 * (int)(i - (size_t)m * groups);
        float v[8];
        ldc8<uint16_t>(a.src[j] + (size_t)m * a.ld[j] + n, a.cols[j] - n, false, v);
        stc8<uint16_t>(a.dst[j] + 8 * i, v, 8, true);
    }
}

// the first K columns of rows of ld elements, as contiguous rows
__global__ __launch_bounds__(256) void kda_linear_compact_kernel(const uint16_t* __restrict__ src, uint16_t* __restrict__ dst,
                                                                 int64_t ld, int K, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256)
        dst[i] = src[i / K * ld + i % K];
}

// ----------------------------------------------------------------------------
// launches
// ----------------------------------------------------------------------------
// rows that can be read and written 16 bytes at a time
bool groups_ok(const void* p, int64_t ld, int es) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % (16 / es) == 0);
}

template <int BM, int BN, int WR, int WC, int WPE, int NB, bool AHEAD, bool BT, int ACT, bool DG>
hipError_t launch_tiles(GemmArgs& a, hipStream_t st) {
    constexpr size_t LDS = NB * (BM + BN) * 128;
    const auto kernel = kda_linear_bf16_kernel<BM, BN, WR, WC, WPE, NB, AHEAD, BT, ACT, DG>;
    if constexpr (LDS > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS);
        if (e != hipSuccess) return e;
    }
    a.mt = (a.M + BM - 1) / BM;
    a.nt = (a.N + BN - 1) / BN;
    hipLaunchKernelGGL(kernel, dim3((unsigned)a.mt * a.nt), dim3(64 * WR * WC), LDS, st, a);
    return hipGetLastError();
}

// bf16 tiles, by how many there are for 256 CUs (us):
//                               256 x 256   128 x 128   64 x 64
//   16384 x 8192, K 2048              503         526       740
//   25088 x  384, K 1536               38          41        47
//   12544 x  768, K 768                22          25        26   (147 of the largest)
//   25088 x 1536, K 384, gelu          64          55        64
//   the same, times gelu'(z)           72          59        64
//    4096 x 1024, K 1024               25          11        14
//    2048 x 2048, K 512                16           8.0       9.3
//    2048 x 1024, K 1024               24          10         7.8
//    6272 x  384, K 1536               33          19        15
// One workgroup of 256 x 256 fills a CU, so nothing runs beside its epilogue: it
// takes half the data a product, and pays where the steps outweigh the epilogue
// and most CUs have one.
int bf16_tile(int M, int N, int K) {   // its edge
    const int64_t m256 = (M + 255) / 256, n256 = (N + 255) / 256, m128 = (M + 127) / 128, n128 = (N + 127) / 128;
    return m256 * n256 >= 144 && K >= 512 ? 256 : m128 * n128 >= 192 ? 128 : 64;
}
// Four buffers instead of two for tiles of 64 x 64: where a CU has one of them, a step
// takes as long as a load, and four steps' loads then overlap (us, 2 | 4 buffers:
// 64 tiles, K 8192, 55 | 27; 128, K 2048, 16.3 | 9.3; 256, K 1024, 6.6 | 6.2; 294, K 1536,
// 12.7 | 11.5); more tiles hide each other's loads and need the room, and few steps fill
// no four buffers (588, K 768, 8.7 | 10.3; 312, K 384, 4.9 | 5.3; 96, K 384, 4.0 | 4.1)
bool deep(int M, int N, int K) { return ((int64_t)M + 63) / 64 * ((N + 63) / 64) <= 320 && K >= 512; }
template <bool BT, int ACT, bool DG>
hipError_t launch_bf16(GemmArgs& a, hipStream_t st) {
    switch (bf16_tile(a.M, a.N, a.K)) {
        case 256: return launch_tiles<256, 256, 4, 4, 4, 2, false, BT, ACT, DG>(a, st);
        case 128: return launch_tiles<128, 128, 2, 4, 4, 2, true, BT, ACT, DG>(a, st);
    }
    return deep(a.M, a.N, a.K) ? launch_tiles<64, 64, 2, 2, 4, 4, true, BT, ACT, DG>(a, st)
                               : launch_tiles<64, 64, 2, 2, 4, 2, true, BT, ACT, DG>(a, st);
}
// rows of waves of such a product, each with its column sums
int wave_rows(int M, int N, int K) {
    const int t = bf16_tile(M, N, K);
    return (M + t - 1) / t * (t == 256 ? 4 : 2);
}

// fp32 tiles, by how many there are for 256 CUs (6272 rows: 384 -> 1536, 588 tiles of
// 128 x 128: 65 us, 1176 of 128 x 64: 52, 2352 of 64 x 64: 56; 1536 -> 384, a quarter
// as many: 94, 74, 62; 4096 x 4096 x 4096, 1024 of 128 x 128: 663, 727, 815)
template <bool BT, int ACT, bool DG>
hipError_t launch_f32(GemmArgs& a, hipStream_t st) {
    const int64_t m128 = (a.M + 127) / 128, n128 = (a.N + 127) / 128, n64 = (a.N + 63) / 64;
    if (m128 * n128 >= 1024) {
        a.mt = (int)m128;
        a.nt = (int)n128;
        hipLaunchKernelGGL((kda_linear_f32_kernel<128, 128, 2, 2, false, BT, ACT, DG, false>), dim3((unsigned)a.mt * a.nt),
                           dim3(256), 0, st, a);
    } else if (m128 * n64 >= 512) {
        a.mt = (int)m128;
        a.nt = (int)n64;
        hipLaunchKernelGGL((kda_linear_f32_kernel<128, 64, 2, 2, false, BT, ACT, DG, false>), dim3((unsigned)a.mt * a.nt),
                           dim3(256), 0, st, a);
    } else {
        a.mt = (a.M + 63) / 64;
        a.nt = (int)n64;
        hipLaunchKernelGGL((kda_linear_f32_kernel<64, 64, 2, 2, false, BT, ACT, DG, false>), dim3((unsigned)a.mt * a.nt),
                           dim3(256), 0, st, a);
    }
    return hipGetLastError();
}

// Pieces of 16 x 16 instead of tiles: while they are few enough for all CUs at once,
// and twice as many up to 8 rows, whose x the CUs' caches hold.  In fp32 the pieces
// have the fp32 matrix unit's products and no splitting.  us, pieces | tiles:
//   rows, product          pieces        bf16             fp32
//      1, 384 -> 1536          96      3.3    4.3      3.9   12.1
//    128, 384 -> 384          192      3.6    4.5      4.5   12.5
//     32, 8192 -> 2048        256     17.2   27.5     33.2  203.3
//     64, 384 -> 1536         384      4.2    4.5      5.8   12.6
//     48, 8192 -> 2048        384     31.0   27.5
//      8, 2048 -> 8192        512      9.0    9.4     15.9   53.8
//     16, 2048 -> 8192        512     10.3    9.4     17.9   53.9
//      1, 4096 -> 16384      1024     24.0   20.6     48.4  118.7
//     32, 2048 -> 8192       1024     17.8    9.8     31.7   54.4
//    128, 8192 -> 2048       1024     58.7   27.3    114.9  204.5
//      8, 1024 -> 32768      2048     18.8   14.0     31.3   57.0
//     64, 2048 -> 8192       2048     33.1   10.0     59.7   54.7
bool few(int M, int N, int bf16) {
    return ((int64_t)M + 15) / 16 * ((N + 15) / 16) <= (bf16 ? 256 : 1024) * (M <= 8 ? 2 : 1);
}

template <int ACT>
hipError_t launch_fwd(GemmArgs& a, int bf16, hipStream_t st) {
    if (few(a.M, a.N, bf16)) {
        a.nt = (a.N + 15) / 16;
        a.mt = (a.M + 15) / 16;
        const dim3 grid((unsigned)a.mt * a.nt), block(64 * FEW_WAVES);
        if (bf16) hipLaunchKernelGGL((kda_linear_few_kernel<uint16_t, ACT>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((kda_linear_few_kernel<float, ACT>), grid, block, 0, st, a);
        return hipGetLastError();
    }
    return bf16 ? launch_bf16<false, ACT, false>(a, st) : launch_f32<false, ACT, false>(a, st);
}

template <int ACT>
hipError_t launch_dgrad(GemmArgs& a, int bf16, hipStream_t st) {
    return bf16 ? launch_bf16<true, ACT, true>(a, st) : launch_f32<true, ACT, true>(a, st);
}

hipError_t dgrad(int act, int bf16, GemmArgs& a, hipStream_t st) {
    return act == 1 ? launch_dgrad<1>(a, bf16, st) : act == 2 ? launch_dgrad<2>(a, bf16, st) : launch_dgrad<0>(a, bf16, st);
}

// Rows a workgroup of it takes, by how many there are for 256 CUs (a backward pass
// without dx, us, 64 rows | 16: 1571 x 395, 50 of 64 rows, 35 | 26; 4096 x 1024, 256,
// 32 | 29; 3136 x 1536, 294, 34 | 31; 8192 x 1024, 512, 39 | 40; 12544 x 1536, 1176,
// 52 | 58): more workgroups against fewer partial sums
int act_rows(int M, int N) { return ((int64_t)M + 63) / 64 * ((N + 255) / 256) >= 512 ? 64 : 16; }
int act_parts(int M, int N) { return (int)(((int64_t)M + act_rows(M, N) - 1) / act_rows(M, N)); }

template <typename T>
hipError_t launch_act_bwd(const void* dy, const void* z, void* dz, float* part, int64_t ld_dy, int64_t ld_z, int64_t ld_dz,
                          int M, int N, int act, hipStream_t st) {
    constexpr int ES = sizeof(T);
    const int vec = N % 8 == 0 && groups_ok(dy, ld_dy, ES) && groups_ok(act ? z : nullptr, ld_z, ES);
    const dim3 grid((unsigned)act_parts(M, N) * ((N + 255) / 256)), block(256);
    const T* pdy = static_cast<const T*>(dy);
    const Pre<T>* pz = static_cast<const Pre<T>*>(z);
    T* pdz = static_cast<T*>(dz);
    const auto kernel = act == 1   ? kda_linear_act_bwd_kernel<T, 1>
                        : act == 2 ? kda_linear_act_bwd_kernel<T, 2>
                                   : kda_linear_act_bwd_kernel<T, 0>;
    hipLaunchKernelGGL(kernel, grid, block, 0, st, pdy, pz, pdz, part, ld_dy, ld_z, ld_dz, M, N, act_rows(M, N), vec);
    return hipGetLastError();
}

hipError_t launch_colsum(const float* part, void* db, int rows, int N, hipStream_t st) {
    hipLaunchKernelGGL(kda_linear_colsum_kernel, dim3((N + 31) / 32), dim3(256), 0, st, part, static_cast<uint16_t*>(db), rows, N);
    return hipGetLastError();
}

// Parts of the m rows that wgrad's sum is split into: a workgroup on each of 256
// CUs, at least 8 steps each (6272 rows, 1536 x 384: 7 parts in tiles of 128 x 128
// by eight waves 50 us, 14 by four waves 53 and twice the partial sums)
void wgrad_plan(int M, int N, int K, int* splits, int* per) {
    const int tiles = ((N + 127) / 128) * ((K + 127) / 128), steps = (M + 31) / 32;
    const int s = std::max(1, std::min(256 / std::max(tiles, 1), steps / 8));
    *per = (steps + s - 1) / s * 32;
    *splits = (M + *per - 1) / *per;
}

// a matrix: pointer, row stride, columns
struct Mat {
    const void* p;
    int64_t ld;
    int n;
};
// the weight gradient dw [n][k] (and db [n]) of one map
struct Wgrad {
    Mat dz, x;
    void *dw, *db;
};

int64_t up8(int64_t n) { return (n + 7) & ~(int64_t)7; }
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// rows that the LDS DMA can read: 16-byte aligned, whole pieces
bool dma_ok(const Mat& m) { return reinterpret_cast<uintptr_t>(m.p) % 16 == 0 && m.ld % 8 == 0 && m.n % 8 == 0; }

// bytes of `count` gradients' partial sums and padded results
size_t wgrads_bytes(const Wgrad* g, int count, int M, int bf16) {
    size_t n = 0;
    if (bf16) {
        WgradProblem q[2] = {};
        for (int j = 0; j < count; ++j) {
            q[j] = WgradProblem{g[j].dz.p, g[j].x.p, g[j].dw, g[j].db, g[j].dz.ld, g[j].x.ld, g[j].dz.n, up8(g[j].x.n)};
            if (g[j].x.n % 8 != 0) n += up256((size_t)g[j].dz.n * up8(g[j].x.n) * 2);
        }
        return n + up256(wgrad_ws_floats(q, count, M) * sizeof(float));
    }
    for (int j = 0; j < count; ++j) {
        int splits, per;
        wgrad_plan(M, g[j].dz.n, g[j].x.n, &splits, &per);
        n = std::max(n, up256(((size_t)splits * g[j].dz.n * (g[j].x.n + 1)) * sizeof(float)));
    }
    return n;
}

hipError_t wgrad_f32(const Wgrad& g, int M, char* ws, hipStream_t st) {
    const int N = g.dz.n, K = g.x.n;
    GemmArgs a = {};   // C[n][k] = sum_m A[m][n] B[m][k]
    a.a = g.dz.p; a.b = g.x.p;
    a.lda = g.dz.ld; a.ldb = g.x.ld;
    a.M = N; a.N = K; a.K = M;
    a.mt = (N + 127) / 128;
    a.nt = (K + 127) / 128;
    wgrad_plan(M, N, K, &a.splits, &a.k_per);
    a.part = reinterpret_cast<float*>(ws);
    float* bpart = a.part + (size_t)a.splits * N * K;
    a.bpart = g.db ? bpart : nullptr;
    a.vec = K % 4 == 0;
    a.vec_a = reinterpret_cast<uintptr_t>(a.a) % 16 == 0 && a.lda % 4 == 0;
    a.vec_b = reinterpret_cast<uintptr_t>(a.b) % 16 == 0 && a.ldb % 4 == 0;
    hipLaunchKernelGGL((kda_linear_f32_kernel<128, 128, 4, 2, true, true, 0, false, true>), dim3((unsigned)(a.mt * a.nt * a.splits)),
                       dim3(512), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const size_t total = (size_t)N * K + N;
    hipLaunchKernelGGL(kda_linear_sum_parts_kernel, dim3((unsigned)std::min<size_t>((total + 255) / 256, 4096)), dim3(256), 0,
                       st, a.part, bpart, static_cast<float*>(g.dw), static_cast<float*>(g.db), (size_t)N * K, N, a.splits);
    return hipGetLastError();
}

hipError_t wgrads(const Wgrad* g, int count, int M, int bf16, char* ws, hipStream_t st) {
    if (count == 0) return hipSuccess;
    hipError_t e = hipSuccess;
    if (!bf16) {
        for (int j = 0; j < count && e == hipSuccess; ++j) e = wgrad_f32(g[j], M, ws, st);
        return e;
    }
    WgradProblem q[2];
    for (int j = 0; j < count; ++j) {
        const int64_t k = up8(g[j].x.n);
        q[j] = WgradProblem{g[j].dz.p, g[j].x.p, g[j].dw, g[j].db, g[j].dz.ld, g[j].x.ld, g[j].dz.n, k};
        if (k != g[j].x.n) {
            q[j].dw = ws;
            ws += up256((size_t)g[j].dz.n * k * 2);
        }
    }
    e = launch_wgrad(q, count, M, reinterpret_cast<float*>(ws), st);
    for (int j = 0; j < count && e == hipSuccess; ++j)
        if (q[j].dw != g[j].dw) {
            const size_t n = (size_t)g[j].dz.n * g[j].x.n;
            hipLaunchKernelGGL(kda_linear_compact_kernel, dim3((unsigned)std::min<size_t>((n + 255) / 256, 2048)), dim3(256), 0,
                               st, static_cast<const uint16_t*>(q[j].dw), static_cast<uint16_t*>(g[j].dw), q[j].k, g[j].x.n, n);
            e = hipGetLastError();
        }
    return e;
}

// dx = dz w (* act'(z))
GemmArgs dgrad_args(const Mat& dz, const Mat& w, const void* z, int64_t ld_z, void* dx, int64_t ld_dx, int M, int es) {
    GemmArgs a = {};   // C[m][k] = sum_n A[m][n] B[n][k]
    a.a = dz.p; a.b = w.p; a.c = dx; a.zin = z;
    a.lda = dz.ld; a.ldb = w.ld; a.ldc = ld_dx; a.ldzi = ld_z;
    a.M = M; a.N = w.n; a.K = dz.n;
    a.vec = w.n % 8 == 0 && groups_ok(dx, ld_dx, es) && groups_ok(z, ld_z, es);
    a.vec_a = reinterpret_cast<uintptr_t>(a.a) % 16 == 0 && a.lda % 4 == 0;
    a.vec_b = reinterpret_cast<uintptr_t>(a.b) % 16 == 0 && a.ldb % 4 == 0;
    return a;
}

int check_map(int M, int N, int K, int act, int dtype) {
    if (dtype != KDA_DTYPE_F32 && dtype != KDA_DTYPE_BF16)
        return api_fail(KDA_E_UNSUPPORTED, "dtype=%d: expected 0 (fp32) or 1 (bf16)", dtype);
    if (act < KDA_ACT_NONE || act > KDA_ACT_SILU)
        return api_fail(KDA_E_UNSUPPORTED, "act=%d: expected 0 (none), 1 (gelu) or 2 (silu)", act);
    if (M < 0 || N < 1 || K < 1 || N > (1 << 20) || K > (1 << 20))
        return api_fail(KDA_E_INVALID, "M=%d N=%d K=%d: expected M >= 0, N and K from 1 to 2^20", M, N, K);
    // tiles of 64 x 128 by at most 512 threads: below 2^32 threads
    if (((int64_t)M + 63) / 64 * ((std::max(N, K) + 127) / 128) > (1 << 22))
        return api_fail(KDA_E_UNSUPPORTED, "M=%d N=%d K=%d: more than 2^22 tiles of 64 x 128", M, N, K);
    return KDA_OK;
}

// a matrix's pointer and row stride; dma: rows are read 16 bytes at a time
int check_rows(const void* p, const char* name, int64_t ld, int cols, int dtype, bool dma) {
    const int es = dtype == KDA_DTYPE_BF16 ? 2 : 4;
    if (!p) return api_fail(KDA_E_INVALID, "%s is NULL", name);
    if (reinterpret_cast<uintptr_t>(p) % (dma ? 16 : es) != 0)
        return api_fail(KDA_E_INVALID, "%s is not %d-byte aligned", name, dma ? 16 : es);
    if (ld < (dma ? up8(cols) : cols) || ld > (1 << 21) || (dma && ld % 8 != 0))
        return api_fail(KDA_E_INVALID, "%s: row stride %lld for %d columns", name, (long long)ld, cols);
    return KDA_OK;
}
int check_opt(const void* p, const char* name, int64_t ld, int cols, int dtype) {
    return p ? check_rows(p, name, ld, cols, dtype, false) : KDA_OK;
}
int check_ws(const void* ws, size_t have, size_t need) {
    if (need == 0) return KDA_OK;
    if (!ws || reinterpret_cast<uintptr_t>(ws) % 16 != 0)
        return api_fail(KDA_E_INVALID, "workspace is NULL or not 16-byte aligned");
    if (have < need) return api_fail(KDA_E_WORKSPACE, "workspace has %zu bytes, needs %zu", have, need);
    return KDA_OK;
}

#define LIN_TRY(x)                       \
    do {                                 \
        const int rc_ = (x);             \
        if (rc_ != KDA_OK) return rc_;   \
    } while (0)
#define LIN_HIP(x, what)                                       \
    do {                                                       \
        const hipError_t e_ = (x);                             \
        if (e_ != hipSuccess) return api_hip_fail(e_, what);   \
    } while (0)

// dz's bytes in the workspace: where an activation's derivative is applied, or dy cannot be read as it is
size_t dz_bytes(const Mat& dy, int M, int act, int bf16) {
    return act || (bf16 && !dma_ok(dy)) ? up256((size_t)M * up8(dy.n) * (bf16 ? 2 : 4)) : 0;
}
// dy act'(z) as dz_bytes' part of the workspace, or dy itself; part: launch_act_bwd's
hipError_t make_dz(Mat* dy, const void* z, int64_t ld_z, int M, int act, int bf16, char** ws, float* part, hipStream_t st) {
    const size_t n = dz_bytes(*dy, M, act, bf16);
    if (n == 0) return hipSuccess;
    const Mat dz = {*ws, up8(dy->n), dy->n};
    const hipError_t e = bf16 ? launch_act_bwd<uint16_t>(dy->p, z, *ws, part, dy->ld, ld_z, dz.ld, M, dy->n, act, st)
                              : launch_act_bwd<float>(dy->p, z, *ws, part, dy->ld, ld_z, dz.ld, M, dy->n, act, st);
    *ws += n;
    *dy = dz;
    return e;
}

// A bf16 bias gradient behind an activation sums dz before it is rounded: from its
// rounded values the sum would be off by as much again as its own rounding.
bool sums_apart(int act, int bf16) { return act && bf16; }

}  // namespace

}  // namespace kda

using namespace kda;

extern "C" {

int kda_linear_fwd(const void* x, int64_t ld_x, const void* w, int64_t ld_w, const void* bias, const void* residual,
                   int64_t ld_r, void* y, int64_t ld_y, void* z, int64_t ld_z, int M, int N, int K, int act, int dtype,
                   void* stream) {
    LIN_TRY(check_map(M, N, K, act, dtype));
    if (M == 0) return KDA_OK;
    const int es = dtype == KDA_DTYPE_BF16 ? 2 : 4;
    const bool dma = dtype == KDA_DTYPE_BF16 && !few(M, N, 1);
    LIN_TRY(check_rows(x, "x", ld_x, K, dtype, dma));
    LIN_TRY(check_rows(w, "w", ld_w, K, dtype, dma));
    LIN_TRY(check_opt(bias, "bias", N, N, dtype));
    LIN_TRY(check_opt(residual, "residual", ld_r, N, dtype));
    LIN_TRY(check_rows(y, "y", ld_y, N, dtype, false));
    LIN_TRY(check_opt(z, "z", ld_z, N, dtype));
    GemmArgs a = {};
    a.a = x; a.b = w; a.c = y; a.bias = bias; a.res = residual; a.zout = z;
    a.lda = ld_x; a.ldb = ld_w; a.ldc = ld_y; a.ldr = ld_r; a.ldzo = ld_z;
    a.M = M; a.N = N; a.K = K;
    a.vec = N % 8 == 0 && groups_ok(y, ld_y, es) && groups_ok(bias, 0, es) && groups_ok(residual, ld_r, es) && groups_ok(z, ld_z, es);
    a.vec_a = groups_ok(x, ld_x, es);
    a.vec_b = groups_ok(w, ld_w, es);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    LIN_HIP(act == 1   ? launch_fwd<1>(a, es == 2, st)
            : act == 2 ? launch_fwd<2>(a, es == 2, st)
                       : launch_fwd<0>(a, es == 2, st),
            "kda_linear_fwd");
    return KDA_OK;
}

int kda_linear_pad(const void* src0, int64_t ld0, int rows0, int cols0, void* dst0, const void* src1, int64_t ld1, int rows1,
                   int cols1, void* dst1, void* stream) {
    PadArgs a = {};
    const void* src[2] = {src0, src1};
    void* dst[2] = {dst0, dst1};
    const int64_t ld[2] = {ld0, ld1};
    const int rows[2] = {rows0, rows1}, cols[2] = {cols0, cols1};
    int n = 0;
    size_t most = 0;
    for (int j = 0; j < 2; ++j) {
        if (!src[j] && !dst[j]) continue;
        if (rows[j] < 0 || cols[j] < 1 || cols[j] > (1 << 20)) return api_fail(KDA_E_INVALID, "matrix %d: %d x %d", j, rows[j], cols[j]);
        LIN_TRY(check_rows(src[j], "src", ld[j], cols[j], KDA_DTYPE_BF16, false));
        if (!dst[j] || reinterpret_cast<uintptr_t>(dst[j]) % 16 != 0)
            return api_fail(KDA_E_INVALID, "dst is NULL or not 16-byte aligned");
        a.src[n] = static_cast<const uint16_t*>(src[j]);
        a.dst[n] = static_cast<uint16_t*>(dst[j]);
        a.ld[n] = ld[j];
        a.rows[n] = rows[j];
        a.cols[n] = cols[j];
        most = std::max(most, (size_t)rows[j] * ((cols[j] + 7) / 8));
        ++n;
    }
    if (n == 0 || most == 0) return KDA_OK;
    hipLaunchKernelGGL(kda_linear_pad_kernel, dim3((unsigned)std::min<size_t>((most + 255) / 256, 4096), n), dim3(256), 0,
                       static_cast<hipStream_t>(stream), a);
    LIN_HIP(hipGetLastError(), "kda_linear_pad");
    return KDA_OK;
}

size_t kda_linear_bwd_workspace_size(const void* dy, int64_t ld_dy, int M, int N, int K, int act, int dtype) {
    if (check_map(M, N, K, act, dtype) != KDA_OK || M == 0) return 0;
    const int bf16 = dtype == KDA_DTYPE_BF16;
    const Mat d = {dy, ld_dy, N};
    const Wgrad g = {d, {nullptr, up8(K), K}, nullptr, const_cast<void*>(dy)};
    const size_t sums = sums_apart(act, bf16) ? up256((size_t)act_parts(M, N) * N * sizeof(float)) : 0;
    return dz_bytes(d, M, act, bf16) + sums + wgrads_bytes(&g, 1, M, bf16);
}

int kda_linear_bwd(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, const void* w, int64_t ld_w, const void* z,
                   int64_t ld_z, void* dx, int64_t ld_dx, void* dw, void* db, int M, int N, int K, int act, int dtype,
                   void* workspace, size_t ws_bytes, void* stream) {
    LIN_TRY(check_map(M, N, K, act, dtype));
    if (M < 1) return api_fail(KDA_E_INVALID, "M=%d: expected at least one row", M);
    const int bf16 = dtype == KDA_DTYPE_BF16, es = bf16 ? 2 : 4;
    LIN_TRY(check_rows(dy, "dy", ld_dy, N, dtype, false));
    if (act) LIN_TRY(check_rows(z, "z", ld_z, N, dtype, false));
    if (dx) {
        LIN_TRY(check_rows(w, "w", ld_w, K, dtype, bf16));
        LIN_TRY(check_rows(dx, "dx", ld_dx, K, dtype, false));
    }
    if (dw) {
        LIN_TRY(check_rows(x, "x", ld_x, K, dtype, bf16));
        LIN_TRY(check_rows(dw, "dw", K, K, dtype, bf16 && K % 8 == 0));
    } else if (db) {
        return api_fail(KDA_E_INVALID, "db without dw");
    }
    LIN_TRY(check_ws(workspace, ws_bytes, kda_linear_bwd_workspace_size(dy, ld_dy, M, N, K, act, dtype)));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    Mat dz = {dy, ld_dy, N};
    float* part = db && sums_apart(act, bf16) ? reinterpret_cast<float*>(ws + dz_bytes(dz, M, act, bf16)) : nullptr;
    LIN_HIP(make_dz(&dz, z, ld_z, M, act, bf16, &ws, part, st), "kda_linear_bwd");
    if (part) {
        const int rows = act_parts(M, N);
        LIN_HIP(launch_colsum(part, db, rows, N, st), "kda_linear_bwd");
        ws += up256((size_t)rows * N * sizeof(float));
        db = nullptr;
    }
    if (dx) {
        GemmArgs a = dgrad_args(dz, {w, ld_w, K}, nullptr, 0, dx, ld_dx, M, es);
        LIN_HIP(dgrad(0, bf16, a, st), "kda_linear_bwd");
    }
    const Wgrad g = {dz, {x, ld_x, K}, dw, db};
    LIN_HIP(wgrads(&g, dw ? 1 : 0, M, bf16, ws, st), "kda_linear_bwd");
    return KDA_OK;
}

size_t kda_mlp_bwd_workspace_size(const void* dy, int64_t ld_dy, int M, int N, int K, int O, int act, int dtype) {
    if (check_map(M, N, K, act, dtype) != KDA_OK || check_map(M, O, N, act, dtype) != KDA_OK || M == 0) return 0;
    const int bf16 = dtype == KDA_DTYPE_BF16;
    const Mat d = {dy, ld_dy, O}, d1 = {nullptr, up8(N), N};
    void* b = const_cast<void*>(dy);
    const Wgrad g[2] = {{d, {nullptr, up8(N), N}, nullptr, b}, {d1, {nullptr, up8(K), K}, nullptr, b}};
    size_t one = wgrads_bytes(g, 2, M, bf16);
    for (int j = 0; j < 2; ++j) one = std::max(one, wgrads_bytes(g + j, 1, M, bf16));
    const size_t sums = sums_apart(act, bf16) ? up256((size_t)wave_rows(M, N, O) * N * sizeof(float)) : 0;
    return dz_bytes(d, M, 0, bf16) + up256((size_t)M * up8(N) * (bf16 ? 2 : 4)) + sums + one;
}

int kda_mlp_bwd(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, const void* w1, int64_t ld_w1, const void* z,
                int64_t ld_z, const void* h, int64_t ld_h, const void* w2, int64_t ld_w2, void* dx, int64_t ld_dx, void* dw1,
                void* db1, void* dw2, void* db2, int M, int N, int K, int O, int act, int dtype, void* workspace,
                size_t ws_bytes, void* stream) {
    LIN_TRY(check_map(M, N, K, act, dtype));
    LIN_TRY(check_map(M, O, N, act, dtype));
    if (M < 1) return api_fail(KDA_E_INVALID, "M=%d: expected at least one row", M);
    const int bf16 = dtype == KDA_DTYPE_BF16, es = bf16 ? 2 : 4;
    const bool first = dx || dw1;
    LIN_TRY(check_rows(dy, "dy", ld_dy, O, dtype, false));
    if (first) {
        LIN_TRY(check_rows(w2, "w2", ld_w2, N, dtype, bf16));
        if (act) LIN_TRY(check_rows(z, "z", ld_z, N, dtype, false));
    }
    if (dx) {
        LIN_TRY(check_rows(w1, "w1", ld_w1, K, dtype, bf16));
        LIN_TRY(check_rows(dx, "dx", ld_dx, K, dtype, false));
    }
    if (dw1) {
        LIN_TRY(check_rows(x, "x", ld_x, K, dtype, bf16));
        LIN_TRY(check_rows(dw1, "dw1", K, K, dtype, bf16 && K % 8 == 0));
    }
    if (dw2) {
        LIN_TRY(check_rows(h, "h", ld_h, N, dtype, bf16));
        LIN_TRY(check_rows(dw2, "dw2", N, N, dtype, bf16 && N % 8 == 0));
    }
    if ((db1 && !dw1) || (db2 && !dw2)) return api_fail(KDA_E_INVALID, "a bias gradient without its weight's");
    LIN_TRY(check_ws(workspace, ws_bytes, kda_mlp_bwd_workspace_size(dy, ld_dy, M, N, K, O, act, dtype)));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    Mat d2 = {dy, ld_dy, O};
    LIN_HIP(make_dz(&d2, nullptr, 0, M, 0, bf16, &ws, nullptr, st), "kda_mlp_bwd");
    const Mat d1 = {ws, up8(N), N};
    if (first) {   // dz1 = (dy w2) act'(z)
        GemmArgs a = dgrad_args(d2, {w2, ld_w2, N}, act ? z : nullptr, ld_z, ws, d1.ld, M, es);
        ws += up256((size_t)M * d1.ld * es);
        const bool apart = db1 && sums_apart(act, bf16);
        if (apart) a.bpart = reinterpret_cast<float*>(ws);
        LIN_HIP(dgrad(act, bf16, a, st), "kda_mlp_bwd");
        if (apart) {
            const int rows = wave_rows(M, N, O);
            LIN_HIP(launch_colsum(a.bpart, db1, rows, N, st), "kda_mlp_bwd");
            ws += up256((size_t)rows * N * sizeof(float));
            db1 = nullptr;
        }
    }
    if (dx) {
        GemmArgs a = dgrad_args(d1, {w1, ld_w1, K}, nullptr, 0, dx, ld_dx, M, es);
        LIN_HIP(dgrad(0, bf16, a, st), "kda_mlp_bwd");
    }
    Wgrad g[2];
    int count = 0;
    if (dw1) g[count++] = Wgrad{d1, {x, ld_x, K}, dw1, db1};
    if (dw2) g[count++] = Wgrad{d2, {h, ld_h, N}, dw2, db2};
    LIN_HIP(wgrads(g, count, M, bf16, ws, st), "kda_mlp_bwd");
    return KDA_OK;
}

}  // extern "C"
