// kda_decay.hip -- linear attention with a decay for each head: the forward and backward
// passes over whole sequences, one token's step, and the C ABI around them.
//
//   S_t = e^{g_t} S_{t-1} + v_t k_t^T,   o_t = S_t q_t        (S[i_v][j_k], fp32)
//
// A sequence is worked through in chunks of C tokens with the state in registers.
// With G_t the sum of g over the chunk up to t,
//   o_t = e^{G_t} S q_t + sum_{s <= t} e^{G_t - G_s} (q_t . k_s) v_s
//   S'  = e^{G_C} S + sum_s e^{G_C - G_s} v_s k_s^T
// so a chunk is four products of the matrix unit.  All of the backward pass is the
// same form again.  With (X, Y, W) in the places of (q, k, v):
//   dq  (do, v, k), the state transposed;
//   dk  (v, do, q) and dv (k, q, do), backwards in time with the decay of the token
//       behind, the state then being dS, the adjoint of S;
//   dg_t = e^{g_t} <S_{t-1}, dS_t>, what reaches tokens from t on from before t,
// put together from what enters, leaves, crosses and passes a chunk (mix2).
//
// A long sequence is shared out into slots of whole chunks, a workgroup each: a pass for what
// every slot adds to the state, a scan over the slots, and the pass for the output.  That
// reads k and v twice, and gives a few long sequences the whole card.
#include "kda_hip.h"
#include "kda_internal.h"

#include <cmath>

namespace kda {

namespace {

// One operand [batch][token][head][D]: strides in elements, `share` heads of the
// state to one of its own
struct Rows {
    const void* p;
    int64_t batch, token, head;
    int share;
};

// A run of tokens that one workgroup takes through in order
struct Slot {
    int tok0, n, seq;   // seq -1: tokens of no sequence, -2: nothing
    int first, last;    // of its sequence
};

struct DecayArgs {
    Rows x, y, w, z;            // z: the fourth operand (mix: q beside dq; mix2: see there)
    const float* g;
    int64_t gb, gt, gh;
    void *out, *out2;           // [B][T][H][D]
    const float* s_in;          // the state that a slot starts from, by slot or by sequence
    float* s_out;               // and ends with: by slot (states), by sequence (else); may be null
    float* dots;                // [H][B T]
    float* peaks;               // [H][chunk_count]: the largest |S| at each chunk's start
    const float *starts, *s_final;   // mix2: the state at the starts (as s_in), and at the sequences' ends
    float* dg;                  // [B][T][H], or null
    double* sums;               // or its sums by slot, [slot][H]
    float* seg;                 // states: e^{sum of g} of each slot and head
    const int4* tab;            // packed: the slots, and the order in which they are taken
    const int* order;
    int in_by_slot;
    int B, T, H, nseq, nslots, per_seq, seg_tokens;
};

__device__ __forceinline__ Slot slot_of(const DecayArgs& a, int j) {
    Slot s;
    if (a.tab) {
        const int4 t = a.tab[j];
        s.tok0 = t.x; s.n = t.y; s.seq = t.z; s.first = t.w & 1; s.last = (t.w >> 1) & 1;
    } else {
        s.seq = j / a.per_seq;
        const int i = j - s.seq * a.per_seq;
        s.tok0 = i * a.seg_tokens;
        s.n = min(a.seg_tokens, a.T - s.tok0);
        s.first = i == 0;
        s.last = i == a.per_seq - 1;
    }
    return s;
}
// Chunks are numbered in their tokens' order, with a gap where a slot's last one is not whole:
// chunk c of slot j, whose first token is number `tok` of all rows
__device__ __forceinline__ int64_t chunk_number(int64_t tok, int j, int c) { return tok / 32 + j + c; }
__host__ __device__ __forceinline__ int64_t chunk_count(int64_t B, int64_t T, int64_t nslots) { return B * T / 32 + nslots + 1; }
// The slot, head and part of the columns of a workgroup.  Workgroups go to the 8 XCDs in
// turn: neighbours, which read the same tokens' keys, are put into one XCD's cache where the grid is
// a multiple of 8 (else they stay as they come); of packed sequences, whose slots differ in
// length, only the parts of one slot and head are, for any grid, so that each XCD begins with whole
// slots and ends with short ones (20000 in 10 sequences x 16 x 128, forward and backward, when it was
// chosen: 806 us in the slots' own order, 779 so, 727 with lengths chosen for it).
template <int SPLIT>
__device__ __forceinline__ void work_of(const DecayArgs& a, int& j, int& h, int& cols) {
    int at;
    if (a.tab) {
        constexpr int GROUP = 8 * SPLIT;
        const int b = (int)blockIdx.x, r = b % GROUP, g = b - r;
        const bool full = g + GROUP <= (int)gridDim.x;
        at = g / SPLIT + (full ? r % 8 : r / SPLIT);
        cols = full ? r / 8 : r % SPLIT;
    } else {
        const int b = xcd_remap((int)blockIdx.x, (int)gridDim.x);
        at = b / SPLIT;
        cols = b % SPLIT;
    }
    j = at / a.H;
    h = at - j * a.H;
    if (a.tab) j = a.order[j];
}

// Products of two operands given as sums of bf16 planes, down to 2^-16 of the
// largest, the smallest first
template <int NA, int NB>
__device__ __forceinline__ f32x4 mmp(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], f32x4 c) {
#pragma unroll
    for (int s = 2; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], c, 0, 0, 0);
    return c;
}

// eight fp32 values as N bf16 planes: with three, exactly
template <int N>
__device__ __forceinline__ void planes8(const float* v, bf16x8 (&f)[N]) {
    uint32_t w[N][4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        float x = v[2 * p], y = v[2 * p + 1];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w[i][p] = pack2bf(x, y);
            if (i + 1 < N) { x -= bf_lo(w[i][p]); y -= bf_hi(w[i][p]); }
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = __builtin_bit_cast(bf16x8, make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]));
}

// Tiles of rows in LDS, RB bytes each: 16-byte piece c of row r lies at c ^ key(r), so that
// neither eight rows' reads of one piece nor a transposing read's four rows of two
// pieces meet in a bank (with fewer than eight pieces to a row and its neighbour's: two bits).
template <int RB>
struct Sw {
    __device__ __forceinline__ static int key(int r) {
        return RB % 128 == 0 ? ((r & 3) << 1) | ((r >> 2) & 1) : (r & 2) | ((r >> 2) & 1);
    }
    __device__ __forceinline__ static int at(int r, int c) { return r * RB + ((c ^ key(r)) << 4); }
    // at(r, 4 k + q), q < 4, with k's part as a constant where k is one
    __device__ __forceinline__ static int at(int r, int q, int k) {
        const int o = r * RB + ((q ^ (key(r) & 3)) << 4);
        return RB % 128 == 0 ? o + (((k & 1) ^ ((r >> 1) & 1)) << 6) + 64 * (k & ~1) : o + 64 * k;
    }
};

// C tokens a chunk; a wave has 16 of W's channels (32, which halves the LDS reads, took
// 190 us instead of 175 over 65536 x 12 x 64: too few waves), a workgroup a SPLIT-th of
// them: the pairs are then formed SPLIT times, but by waves that would wait for them (20000
// packed x 16 x 128, when it was chosen: 115 instead of 128 us forward, dq 147 instead of 185).  bf16 operands are
// one plane, fp32 ones three, and so are the pairs' weights and the state as factors (NP): with two,
// 16 bits, one bf16 output in 450 is rounded the other way, so one in 6000 to 18000, for 1 to 3%
// of the time (65536 x 12 x 64 153.1 -> 154.7 us, 20000 packed x 16 x 128 forward and backward 726 -> 747).
// OCC, OCC2: waves a SIMD that mix and mix2 are held to (fp32, D = 64: mix2 takes registers for
// one where it is let, and the training call 254 us instead of 220, 8 x 1568 x 12).
template <int D_, bool F32_, int SPLIT_ = 1, int C_ = 32>
struct Cfg {
    static constexpr int D = D_, C = C_, SPLIT = SPLIT_, DW = D / SPLIT, NPL = F32_ ? 3 : 1, NP = 3, NW = DW / 16, NTH = 64 * NW;
    static constexpr int RB = 2 * D, PLANE = C * RB, TILE = NPL * PLANE;                       // bytes
    static constexpr int RBW = (2 * DW + 63) / 64 * 64, PLANEW = C * RBW, TILEW = NPL * PLANEW;   // of DW channels
    static constexpr int RP = 2 * C, PPL = C * RP;                                             // of the pairs'
    static constexpr int TT = C / 16, NT = TT * (TT + 1) / 2, DT = D / 16, KD = D / 32, KC = C / 32;
    static constexpr int OCC = F32_ ? 1 : D > 64 ? 3 : 4, OCC2 = F32_ ? (D > 32 ? 2 : 1) : D > 64 ? 2 : 3;
    static constexpr bool F32 = F32_, WITH_DS = D <= 64;
    typedef typename std::conditional<F32_, float, uint16_t>::type ST;
    static constexpr int ES = (int)sizeof(ST), EPV = 16 / ES;
    static_assert(C % 32 == 0 && D % (16 * SPLIT) == 0 && D % 32 == 0, "whole tiles");
};

// C rows of COLS channels on their way from memory to LDS, forwards or backwards in time
template <class K, int COLS, bool REV>
struct Stage {
    static constexpr int VPR = COLS / K::EPV, NV = K::C * VPR, PER = NV / K::NTH;
    static constexpr int RB = COLS == K::D ? K::RB : K::RBW, PLANE = K::C * RB;
    static_assert(NV % K::NTH == 0, "whole pieces");
    uint4 r[PER];
    // n >= 1 rows, the first in memory at p, `step` bytes apart; what is behind them reads the last
    __device__ __forceinline__ void load(const typename K::ST* p, uint32_t step, int n) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int v = (int)threadIdx.x + K::NTH * i, row = v / VPR, c = v - row * VPR, m = min(row, n - 1);
            r[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p) + ((uint32_t)(REV ? n - 1 - m : m) * step + 16 * c));
        }
    }
    // ... and is stored as zeros
    __device__ __forceinline__ void store(char* t, int n) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int v = (int)threadIdx.x + K::NTH * i, row = v / VPR, c = v - row * VPR;
            uint4 x = r[i];
            if (n < K::C) x = row < n ? x : make_uint4(0u, 0u, 0u, 0u);
            if constexpr (!K::F32) {
                *reinterpret_cast<uint4*>(t + Sw<RB>::at(row, c)) = x;
            } else {
                // each part the next 8 bits of 24, cut off, so that nothing overflows
                const uint32_t b[4] = {x.x, x.y, x.z, x.w};
                uint32_t h[4], m[4], l[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    h[e] = b[e] & 0xffff0000u;
                    const float rest = __uint_as_float(b[e]) - __uint_as_float(h[e]);
                    m[e] = __float_as_uint(rest) & 0xffff0000u;
                    l[e] = __float_as_uint(rest - __uint_as_float(m[e]));
                }
                constexpr uint32_t HI = 0x07060302u;
                char* q = t + Sw<RB>::at(row, c >> 1) + 8 * (c & 1);
                *reinterpret_cast<uint2*>(q) =
                    make_uint2(__builtin_amdgcn_perm(h[1], h[0], HI), __builtin_amdgcn_perm(h[3], h[2], HI));
                *reinterpret_cast<uint2*>(q + PLANE) =
                    make_uint2(__builtin_amdgcn_perm(m[1], m[0], HI), __builtin_amdgcn_perm(m[3], m[2], HI));
                *reinterpret_cast<uint2*>(q + 2 * PLANE) =
                    make_uint2(__builtin_amdgcn_perm(l[1], l[0], HI), __builtin_amdgcn_perm(l[3], l[2], HI));
            }
        }
    }
};

// Fragments, the contracted index in the matrix unit's own order (lane l has 8 (l / 16) ..
// + 7 of 32).  Along the rows:
template <int RB, int NPL, int PLANE>
__device__ __forceinline__ void along(const char* t, int row0, int k, bf16x8 (&f)[NPL]) {
    const int l = lane_id(), o = Sw<RB>::at(l & 15, l >> 4, k);
#pragma unroll
    for (int p = 0; p < NPL; ++p)
        f[p] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(t + p * PLANE + row0 * RB + o));
}
// and across them: 16 columns of rows 32 k .., the p-th four of them at o0 (o1: four rows on)
template <int RB, int NPL, int PLANE>
__device__ __forceinline__ void across(const char* t, int k, int o0, int o1, bf16x8 (&f)[NPL]) {
#pragma unroll
    for (int p = 0; p < NPL; ++p) {
        const char* u = t + p * PLANE + 32 * k * RB;
        f[p] = cat4(ld_tr4(reinterpret_cast<const uint16_t*>(u + o0)), ld_tr4(reinterpret_cast<const uint16_t*>(u + o1)));
    }
}
// of W, columns 16 w .. of rows of RB bytes; of Y, tile t: every other four of 32 channels
template <class K, int RB>
__device__ __forceinline__ void w_frag(const char* W, int k, int w, bf16x8 (&f)[K::NPL]) {
    const int l = lane_id(), j = l & 15, row = 8 * (l >> 4) + (j >> 2), piece = 2 * w + ((j & 3) >> 1), b = 8 * (j & 1);
    across<RB, K::NPL, K::C * RB>(W, k, Sw<RB>::at(row, piece) + b, Sw<RB>::at(row + 4, piece) + b, f);
}
template <class K>
__device__ __forceinline__ void y_frag(const char* Y, int k, int t, bf16x8 (&f)[K::NPL]) {
    const int l = lane_id(), j = l & 15, row = 8 * (l >> 4) + (j >> 2), b = 8 * (t & 1);
    across<K::RB, K::NPL, K::PLANE>(Y, k, Sw<K::RB>::at(row, j & 3, t >> 1) + b, Sw<K::RB>::at(row + 4, j & 3, t >> 1) + b, f);
}

// A chunk's decays.  Sums of g are formed in fp64 (a difference of two sums of
// fast decays would lose what lies between neighbours) and kept as pairs of fp32,
// in powers of two.
template <int C>
struct Decays {
    float hi[C], lo[C], up[C], down[C];   // G_t; 2^{G_t}; 2^{G_C - G_t}
    float all, pad[3];                    // 2^{G_C}
};
constexpr double LOG2E = 1.4426950408889634;
// e^-200 is zero in fp32, as e^-inf is, and its sums stay finite
constexpr float G_MIN = -200.f;
__device__ __forceinline__ float decay(float g) { return expf(g < G_MIN ? G_MIN : g); }

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double x) {   // 0 where there is no source lane
    const uint2 u = __builtin_bit_cast(uint2, x);
    return __builtin_bit_cast(double, make_uint2(__builtin_amdgcn_update_dpp(0, u.x, CTRL, ROWS, 0xf, true),
                                                 __builtin_amdgcn_update_dpp(0, u.y, CTRL, ROWS, 0xf, true)));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, true));
}
__device__ __forceinline__ float lane(float x, int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l)); }
// sums over the lanes up to each, of 32; and the last of those, for all lanes
template <typename T>
__device__ __forceinline__ T prefix32(T x) {
    x += dpp<0x111, 0xf>(x);   // row_shr:1, 2, 4, 8
    x += dpp<0x112, 0xf>(x);
    x += dpp<0x114, 0xf>(x);
    x += dpp<0x118, 0xf>(x);
    return x + dpp<0x142, 0xa>(x);   // row_bcast:15, into rows 1 and 3
}
__device__ __forceinline__ double lane(double x, int l) {
    const uint2 u = __builtin_bit_cast(uint2, x);
    return __builtin_bit_cast(double, make_uint2(__builtin_amdgcn_readlane(u.x, l), __builtin_amdgcn_readlane(u.y, l)));
}
__device__ __forceinline__ double lane31(double x) { return lane(x, 31); }
// sums over the lanes behind each, of 32, and over all of them
__device__ __forceinline__ double behind32(double x, double& all) {
    x += dpp<0x101, 0xf>(x);   // row_shl:1, 2, 4, 8
    x += dpp<0x102, 0xf>(x);
    x += dpp<0x104, 0xf>(x);
    x += dpp<0x108, 0xf>(x);
    const double row1 = lane(x, 16);
    all = lane(x, 0) + row1;
    return dpp<0x101, 0xf>(x) + (lane_id() < 16 ? row1 : 0.0);
}
// by one wave: lane r has g of row r (0 behind the last); returns G_C
template <int C>
__device__ __forceinline__ double fill_decays(Decays<C>* d, float g) {
    static_assert(C == 32, "two rows of 16 lanes");
    const int l = lane_id();
    const double x = prefix32((double)(g < G_MIN ? G_MIN : g) * LOG2E), all = lane31(x);
    if (l < C) {
        const float h = (float)x;
        d->hi[l] = h;
        d->lo[l] = (float)(x - (double)h);
        d->up[l] = __builtin_amdgcn_exp2f(h);
        d->down[l] = __builtin_amdgcn_exp2f((float)(all - x));
        if (l == C - 1) d->all = d->up[l];
    }
    return all;
}

// tile id of the lower triangle -> (row of tiles, column)
__device__ __forceinline__ void tile_of(int id, int& ti, int& si) {
    ti = (id >= 1) + (id >= 3) + (id >= 6);
    si = id - ti * (ti + 1) / 2;
}

// raw products of X's rows of tile ti with Y's of tile si: lane (c = l % 16, r = l / 16)
// has X row 16 ti + c with Y rows 16 si + 4 r + i
template <class K>
__device__ __forceinline__ f32x4 pair_tile(const char* X, const char* Y, int ti, int si) {
    f32x4 acc = zero4();
#pragma unroll
    for (int k = 0; k < K::KD; ++k) {
        bf16x8 y[K::NPL], x[K::NPL];
        along<K::RB, K::NPL, K::PLANE>(Y, 16 * si, k, y);
        along<K::RB, K::NPL, K::PLANE>(X, 16 * ti, k, x);
        acc = mmp(y, x, acc);
    }
    return acc;
}
// their weights, and the product with them: nothing of a later token, whatever it is
template <class K>
__device__ __forceinline__ f32x4 mask_tile(const Decays<K::C>& d, int ti, int si) {
    const int l = lane_id(), t = 16 * ti + (l & 15), s0 = 16 * si + 4 * (l >> 4);
    const float h = d.hi[t], o = d.lo[t];
    const float4 hs = *reinterpret_cast<const float4*>(d.hi + s0), ls = *reinterpret_cast<const float4*>(d.lo + s0);
    const float hv[4] = {hs.x, hs.y, hs.z, hs.w}, lv[4] = {ls.x, ls.y, ls.z, ls.w};
    f32x4 m;
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = __builtin_amdgcn_exp2f((h - hv[i]) + (o - lv[i]));
    return m;
}
__device__ __forceinline__ f32x4 masked(const f32x4& p, const f32x4& m, int ti, int si) {
    f32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = ti == si && 4 * (lane_id() >> 4) + i > (lane_id() & 15) ? 0.f : p[i] * m[i];
    return x;
}
// a tile into P[t][s]
template <class K>
__device__ __forceinline__ void put_pair(char* P, const f32x4& v, int ti, int si) {
    const int l = lane_id(), g = l >> 4;
    char* p = P + Sw<K::RP>::at(16 * ti + (l & 15), 2 * si + (g >> 1)) + 8 * (g & 1);
    float x[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int i = 0; i < K::NP; ++i) {
        const uint32_t a = pack2bf(x[0], x[1]), b = pack2bf(x[2], x[3]);
        *reinterpret_cast<uint2*>(p + i * K::PPL) = make_uint2(a, b);
        if (i + 1 < K::NP) { x[0] -= bf_lo(a); x[1] -= bf_hi(a); x[2] -= bf_lo(b); x[3] -= bf_hi(b); }
    }
}
// the tiles above the diagonal that products of 32 columns read
template <class K>
__device__ __forceinline__ void clear_upper(char* P) {
    for (int v = threadIdx.x; v < K::NP * (K::TT / 2) * 16 * 2; v += K::NTH) {
        const int c = v & 1, row = (v >> 1) & 15, b = (v >> 5) % (K::TT / 2), p = (v >> 5) / (K::TT / 2);
        *reinterpret_cast<uint4*>(P + p * K::PPL + Sw<K::RP>::at(32 * b + row, 4 * b + 2 + c)) = make_uint4(0u, 0u, 0u, 0u);
    }
}

// The state, channels 16 w .. + 15 of W for wave w of all: lane (m = l % 16, r = l / 16) holds
// St[32 (j / 2) + 8 r + 4 (j % 2) + i][16 w + m] in s[j][i].  In memory [W's channel][Y's], or
// (swapped) [Y's][W's].
template <class K>
struct State {
    f32x4 s[K::DT];
    __device__ __forceinline__ void load(const float* p, int w, bool swapped) {
        const int l = lane_id(), r = l >> 4, dw = 16 * w + (l & 15);
#pragma unroll
        for (int j = 0; j < K::DT; ++j) {
            const int dy = 32 * (j >> 1) + 8 * r + 4 * (j & 1);
            if (!p) { s[j] = zero4(); continue; }
            if (!swapped) {
                const float4 v = *reinterpret_cast<const float4*>(p + dw * K::D + dy);
                s[j] = f32x4{v.x, v.y, v.z, v.w};
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[j][i] = p[(dy + i) * K::D + dw];
            }
        }
    }
    __device__ __forceinline__ void store(float* p, int w, float scale) const {
        const int l = lane_id(), r = l >> 4, dw = 16 * w + (l & 15);
#pragma unroll
        for (int j = 0; j < K::DT; ++j)
            *reinterpret_cast<float4*>(p + dw * K::D + 32 * (j >> 1) + 8 * r + 4 * (j & 1)) =
                make_float4(scale * s[j][0], scale * s[j][1], scale * s[j][2], scale * s[j][3]);
    }
    // sum of s p over the wave's part, for all lanes; p as load's, swapped
    __device__ __forceinline__ double dot(const float* p, int w) const {
        const int l = lane_id(), r = l >> 4, dw = 16 * w + (l & 15);
        double x = 0.0;
#pragma unroll
        for (int j = 0; j < K::DT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) x += (double)p[(32 * (j >> 1) + 8 * r + 4 * (j & 1) + i) * K::D + dw] * s[j][i];
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m, 64);
        return x;
    }
    // the largest magnitude of the wave's part, and the sum of them, in lane 63
    __device__ __forceinline__ float peak() const {
        float x = 0.f;
#pragma unroll
        for (int j = 0; j < K::DT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) x = fmaxf(x, fabsf(s[j][i]));
        x = fmaxf(x, dpp<0x111, 0xf>(x));
        x = fmaxf(x, dpp<0x112, 0xf>(x));
        x = fmaxf(x, dpp<0x114, 0xf>(x));
        x = fmaxf(x, dpp<0x118, 0xf>(x));
        x = fmaxf(x, dpp<0x142, 0xa>(x));
        return fmaxf(x, dpp<0x143, 0xc>(x));   // row_bcast:31, into rows 2 and 3
    }
    __device__ __forceinline__ float weight() const {
        float x = 0.f;
#pragma unroll
        for (int j = 0; j < K::DT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) x += fabsf(s[j][i]);
        x = prefix32(x);
        return x + dpp<0x143, 0xc>(x);
    }
    // S <- own S + all Y^T (weights W): the chunk's sum from zero, so that what the matrix unit loses
    // (it rounds sums downwards) does not add up over the chunks.  w: w_frag of W.
    __device__ __forceinline__ void add(const char* Y, const bf16x8 (&w)[K::NPL], const float* weights, float own, float all) {
        static_assert(K::KC == 1, "one step of the contracted index");
        const int r = lane_id() >> 4;
        const float4 d0 = *reinterpret_cast<const float4*>(weights + 8 * r), d1 = *reinterpret_cast<const float4*>(weights + 8 * r + 4);
        const float dn[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
        bf16x8 ws[3];
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = (float)w[0][e];
            if constexpr (K::NPL == 3) v[e] += (float)w[1][e] + (float)w[2][e];
            v[e] *= dn[e];
        }
        planes8<3>(v, ws);
#pragma unroll
        for (int j = 0; j < K::DT; ++j) {
            bf16x8 y[K::NPL];
            y_frag<K>(Y, 0, j, y);
            const f32x4 u = mmp(y, ws, zero4());
#pragma unroll
            for (int i = 0; i < 4; ++i) s[j][i] = fmaf(own, s[j][i], all * u[i]);
        }
    }
    // up_t (St^T X_t) for every row: lane (m, r) has row 16 i + m, channels 16 w + 4 r ..
    __device__ __forceinline__ void apply(const char* X, const Decays<K::C>& d, f32x4 (&o)[K::TT]) const {
#pragma unroll
        for (int i = 0; i < K::TT; ++i) o[i] = zero4();
#pragma unroll
        for (int k = 0; k < K::KD; ++k) {
            const f32x4 &x = s[2 * k], &y = s[2 * k + 1];
            const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            bf16x8 f[K::NP];
            planes8<K::NP>(v, f);
#pragma unroll
            for (int i = 0; i < K::TT; ++i) {
                bf16x8 x[K::NPL];
                along<K::RB, K::NPL, K::PLANE>(X, 16 * i, k, x);
                o[i] = mmp(f, x, o[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < K::TT; ++i) o[i] *= d.up[16 * i + (lane_id() & 15)];
    }
};

// A value of W that is not finite would reach the rows before its own too, whose weights are zero:
// seldom, so all of it lies behind a branch, it is taken out of W (w: w_frag) ...
struct Ends {
    bool any;    // in the wave's channels
    int first;   // the first such row of this lane's (C: none)
};
template <class K>
__device__ __forceinline__ Ends take_ends(bf16x8 (&w)[K::NPL]) {
    const uint4 u = __builtin_bit_cast(uint4, w[0]);   // (the first plane has the exponent)
    // bit 15 of a half whose exponent is all ones, carried there
    const auto ends = [](uint32_t x) { return ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u; };
    Ends r = {(bool)__any((int)(ends(u.x) | ends(u.y) | ends(u.z) | ends(u.w))), K::C};
    if (__builtin_expect(r.any, 0)) {
        const int row = 8 * (lane_id() >> 4);
        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 7; e >= 0; --e)
            if (ends(x[e >> 1]) & (e & 1 ? 0x80000000u : 0x8000u)) r.first = row + e;
        r.first = min(r.first, __shfl_xor(r.first, 16, 64));
        r.first = min(r.first, __shfl_xor(r.first, 32, 64));
#pragma unroll
        for (int p = 0; p < K::NPL; ++p) {
            const uint4 v = __builtin_bit_cast(uint4, w[p]);
            uint32_t y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (row + e >= r.first) y[e >> 1] &= e & 1 ? 0xffffu : 0xffff0000u;
            w[p] = __builtin_bit_cast(bf16x8, make_uint4(y[0], y[1], y[2], y[3]));
        }
    }
    return r;
}
// ... and put into its channel of the state behind the chunk, as its decay (no branch: the compiler may
// move what reads a matrix product behind one and then leave out the wait for it), ...
template <class K>
__device__ __forceinline__ float own_of(const Ends& r, float own) {
    return r.first < K::C ? __builtin_nanf("") : own;
}
// ... and of the rows from its own on, before the pairs' part is added
template <class K>
__device__ __forceinline__ void put_ends(const Ends& r, f32x4 (&o)[K::TT]) {
    if (__builtin_expect(r.any, 0)) {
        const int l = lane_id();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int row = __shfl(r.first, 4 * (l >> 4) + c, 64);
#pragma unroll
            for (int i = 0; i < K::TT; ++i)
                if (16 * i + (l & 15) >= row) o[i][c] = __builtin_nanf("");
        }
    }
}

// o_t += sum_s P[t][s] W_s, layout as State::apply
template <class K>
__device__ __forceinline__ void add_pairs(const char* P, const bf16x8 (&w)[K::NPL], f32x4 (&o)[K::TT]) {
#pragma unroll
    for (int i = 0; i < K::TT; ++i) {
        bf16x8 p[K::NP];
        along<K::RP, K::NP, K::PPL>(P, 16 * i, 0, p);
        o[i] = mmp(w, p, o[i]);
    }
}

template <typename T>
__device__ __forceinline__ void put4(T* p, const f32x4& v) {
    if constexpr (std::is_same<T, float>::value)
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else
        *reinterpret_cast<uint2*>(p) = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]));
}
// wave w's channels of the rows of a chunk, the first in memory at out
template <class K, typename OT, bool REV>
__device__ __forceinline__ void put_rows(OT* out, uint32_t step, const f32x4 (&o)[K::TT], int w, int n) {
    const int l = lane_id();
#pragma unroll
    for (int i = 0; i < K::TT; ++i) {
        const int t = 16 * i + (l & 15);
        if (t < n) put4<OT>(out + (uint32_t)(REV ? n - 1 - t : t) * step + 16 * w + 4 * (l >> 4), o[i]);
    }
}
__device__ __forceinline__ float quad_sum(float x) {   // over the four lanes of equal l % 16
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}
__device__ __forceinline__ float dot4(const float4& a, const f32x4& b) {
    return fmaf(a.x, b[0], a.y * b[1]) + fmaf(a.z, b[2], a.w * b[3]);
}

template <typename T>
__device__ __forceinline__ const T* at(const Rows& r, int b, int tok, int h) {
    return static_cast<const T*>(r.p) + b * r.batch + tok * r.token + (h / r.share) * r.head;
}

// rows of no sequence
template <int D, typename OT>
__device__ __forceinline__ void clear_rows(void* out, const DecayArgs& a, const Slot& s, int h) {
    for (int v = threadIdx.x; v < s.n * D; v += blockDim.x)
        static_cast<OT*>(out)[((int64_t)(s.tok0 + v / D) * a.H + h) * D + v % D] = OT(0);
}

template <class K>
constexpr size_t mix_lds(bool states, bool grad, bool dot) {
    return (states ? 1 : grad ? 3 : 2) * (size_t)K::TILE + K::TILEW + (states ? 0 : (size_t)K::NP * K::PPL) + 2 * sizeof(Decays<K::C>) +
           (dot ? (size_t)K::NW * (K::C + 1) * 4 : 0);
}
// four channels of a row of a tile
template <class K>
__device__ __forceinline__ float4 tile4(const char* p) {
    float4 v = ld4<uint16_t>(reinterpret_cast<const uint16_t*>(p));
    if constexpr (K::NPL == 3) {
        const float4 v1 = ld4<uint16_t>(reinterpret_cast<const uint16_t*>(p + K::PLANE)),
                     v2 = ld4<uint16_t>(reinterpret_cast<const uint16_t*>(p + 2 * K::PLANE));
        v = make_float4(v.x + (v1.x + v2.x), v.y + (v1.y + v2.y), v.z + (v1.z + v2.z), v.w + (v1.w + v2.w));
    }
    return v;
}

// mix: out = the operator over a slot's tokens.  STATES: only what the slot adds to the state,
// and its whole decay.  GRAD: out is dq, z is q, and the slots' s_out and seg take what they
// add to dS as well, sum of e^{G_t} do_t q_t^T (WITH_DS, when it was chosen: 8 x 1568 x 12 x 64 34 us, by a pass
// of its own 27 + 15; at D = 128 that leaves registers for two waves a SIMD instead of three, 213 us of
// 20000 packed x 16, by itself 148 + 64); STATES and GRAD: dS alone.  DOT: dots[t] = q_t . (the
// part of out_t that comes from the state before the chunk), by parts of the channels.
//
// A chunk: pairs, state and the state's part of out from LDS; a barrier; the pairs'
// part from P and registers, and the next chunk into LDS; a barrier.  Its loads are in
// flight for a whole chunk.  The last wave, which has the fewest pairs, forms the next
// chunk's decays.
//
// Measured, bf16: 65536 x 12 x 64 STATES 50 us (201 MB at 4.0 TB/s, all that a sum which only
// reads reaches), output 108 us (403 MB at 3.7 TB/s); 8 x 1568 x 12 x 64 15 and 24 us; 20000
// packed x 16 x 128 56 and 122 us.  What bounds the output's pass is the chain through a chunk,
// not one unit: of the latter (117 us when that was measured) the state's sum and its product, most
// of the matrix work, are worth 15 each and 26 together, then stores 28, loads 18, and 34 are
// left without anything else.
template <class K, typename OT, bool STATES, bool GRAD, bool DOT>
__global__ __launch_bounds__(K::NTH, GRAD && !STATES && K::WITH_DS ? K::OCC2 : K::OCC) void kda_decay_mix_kernel(const DecayArgs a) {
    typedef typename K::ST ST;
    constexpr bool DQ = GRAD && !STATES, DS = DQ && K::WITH_DS;
    __shared__ __attribute__((aligned(16))) char lds[mix_lds<K>(STATES, DS, DOT)];
    char* X = lds;
    char* Y = X + (STATES ? 0 : K::TILE);
    char* Z = Y + K::TILE;
    char* W = Z + (DS ? K::TILE : 0);
    char* P = W + K::TILEW;
    Decays<K::C>* dec = reinterpret_cast<Decays<K::C>*>(P + (STATES ? 0 : K::NP * K::PPL));
    float* part = reinterpret_cast<float*>(dec + 2);   // DOT: [NW][C]
    float* peak = part + K::NW * K::C;                 // [NW]

    int j, h, cols;
    work_of<K::SPLIT>(a, j, h, cols);
    const Slot s = slot_of(a, j);
    if (s.seq < 0) {
        if constexpr (!STATES) {
            if (s.seq == -1 && cols == 0) clear_rows<K::D, OT>(a.out, a, s, h);
        }
        return;
    }
    if (STATES && (GRAD ? s.first : s.last)) return;   // no slot needs it
    const int b = a.tab ? 0 : s.seq, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
    const int wv = cols * K::NW + wave;   // of all
    constexpr int DD = K::D * K::D, LAST = K::NW - 1;
    State<K> st, ds;
    st.load(STATES || !a.s_in ? nullptr : a.s_in + ((int64_t)(a.in_by_slot ? j : s.seq) * a.H + h) * DD, wv, DQ);
    const bool adjoint = DS && a.s_out && !s.first;
    if constexpr (DS) ds.load(nullptr, wv, false);
    float before = 1.f;   // e^{sum of g before the chunk}

    const float* g = a.g + b * a.gb + (int64_t)s.tok0 * a.gt + h * a.gh;
    Stage<K, K::D, false> sx, sy, sz;
    Stage<K, K::DW, false> sw;
    float gv = 0.f;
    auto load = [&](int i0) {
        const int n = min(K::C, s.n - i0), t = s.tok0 + i0;
        if constexpr (!STATES) sx.load(at<ST>(a.x, b, t, h), (uint32_t)a.x.token * K::ES, n);
        sy.load(at<ST>(a.y, b, t, h), (uint32_t)a.y.token * K::ES, n);
        if constexpr (DS) sz.load(at<ST>(a.z, b, t, h), (uint32_t)a.z.token * K::ES, n);
        sw.load(at<ST>(a.w, b, t, h) + cols * K::DW, (uint32_t)a.w.token * K::ES, n);
    };
    auto load_g = [&](int i0) {
        const int i = i0 + l;
        gv = l < K::C && i < s.n ? g[(int64_t)i * a.gt] : 0.f;
    };
    auto store = [&](int n) {
        if constexpr (!STATES) sx.store(X, n);
        sy.store(Y, n);
        if constexpr (DS) sz.store(Z, n);
        sw.store(W, n);
    };
    if constexpr (!STATES) clear_upper<K>(P);
    double whole = 0.0;
    if (s.n > 0) {
        load(0);
        if (wave == LAST) {
            load_g(0);
            whole = fill_decays<K::C>(dec, gv);
            load_g(K::C);
        }
        store(s.n);
        if (K::C < s.n) load(K::C);
        lds_barrier();
    }
    for (int i0 = 0; i0 < s.n; i0 += K::C) {
        const int n = min(K::C, s.n - i0);
        const Decays<K::C>& d = dec[i0 / K::C & 1];
        const bool more = i0 + K::C < s.n;
        bf16x8 w[K::NPL];
        f32x4 o[K::TT];
        w_frag<K, K::RBW>(W, 0, wave, w);
        Ends ends;
        if constexpr (!STATES) ends = take_ends<K>(w);
        const int ch = 16 * wv + 4 * (l >> 4);
        float4 z[DOT && !DS ? K::TT : 1];
        if constexpr (DOT && !DS) {
            const ST* p = at<ST>(a.z, b, s.tok0 + i0, h) + ch;
#pragma unroll
            for (int i = 0; i < K::TT; ++i) z[i] = ld4<ST>(p + min(16 * i + (l & 15), n - 1) * (int)a.z.token);
        }
        if constexpr (!STATES) {
#pragma unroll
            for (int k = 0; k < (K::NT + K::NW - 1) / K::NW; ++k) {
                const int id = wave + K::NW * k;
                if (id < K::NT) {
                    int ti, si;
                    tile_of(id, ti, si);
                    put_pair<K>(P, masked(pair_tile<K>(X, Y, ti, si), mask_tile<K>(d, ti, si), ti, si), ti, si);
                }
            }
            st.apply(X, d, o);
            if constexpr (DOT) {
                const float top = st.peak();
                if (l == 63) peak[wave] = top;
#pragma unroll
                for (int i = 0; i < K::TT; ++i) {
                    const int t = 16 * i + (l & 15);
                    if constexpr (DS) z[0] = tile4<K>(Z + Sw<K::RB>::at(t, ch >> 3) + 2 * (ch & 7));
                    const float x = quad_sum(dot4(z[DS ? 0 : i], o[i]));
                    if (l < 16) part[wave * K::C + t] = x;
                }
            }
        }
        if constexpr (STATES && GRAD) {
            st.add(Y, w, d.up, 1.f, before);
            before *= d.all;
        } else {
            st.add(Y, w, d.down, STATES ? d.all : own_of<K>(ends, d.all), 1.f);
        }
        if constexpr (DS) {
            if (adjoint) {
                bf16x8 x[K::NPL];
                w_frag<K, K::RB>(X, 0, wv, x);
                ds.add(Z, x, d.up, 1.f, before);
                before *= d.all;
            }
        }
        if (wave == LAST && more) {
            whole += fill_decays<K::C>(dec + ((i0 / K::C + 1) & 1), gv);
            load_g(i0 + 2 * K::C);
        }
        lds_barrier();
        if (more) {
            store(s.n - i0 - K::C);
            if (i0 + 2 * K::C < s.n) load(i0 + 2 * K::C);
        }
        if constexpr (!STATES) {
            const int64_t row = (int64_t)b * a.T + s.tok0 + i0;
            put_ends<K>(ends, o);
            add_pairs<K>(P, w, o);
            put_rows<K, OT, false>(static_cast<OT*>(a.out) + (row * a.H + h) * K::D, (uint32_t)(a.H * K::D), o, wv, n);
            if constexpr (DOT) {
                const int t = threadIdx.x;
                if (t < n) {
                    float x = 0.f;
#pragma unroll
                    for (int k = 0; k < K::NW; ++k) x += part[k * K::C + t];
                    a.dots[((int64_t)cols * a.H + h) * a.B * a.T + row + t] = x;
                }
                if (t == 0) {
                    float x = peak[0];
#pragma unroll
                    for (int k = 1; k < K::NW; ++k) x = fmaxf(x, peak[k]);
                    a.peaks[((int64_t)cols * a.H + h) * chunk_count(a.B, a.T, a.nslots) +
                            chunk_number((int64_t)b * a.T + s.tok0, j, i0 / K::C)] = x;
                }
            }
        }
        if (more) lds_barrier();
    }
    if (STATES || adjoint) {
        if (wave == LAST && l == 0 && cols == 0) a.seg[(int64_t)j * a.H + h] = __builtin_amdgcn_exp2f((float)whole);
        (STATES ? st : ds).store(a.s_out + ((int64_t)j * a.H + h) * DD, wv, 1.f);
    } else if (!GRAD && a.s_out && s.last) {
        st.store(a.s_out + ((int64_t)s.seq * a.H + h) * DD, wv, 1.f);
    }
}

// What mix2 keeps of a chunk for dg
struct Chunk {
    double enter, leave;      // sums over its tokens: of what comes from before it, of what goes behind it
    double pass;              // what passes it, counted from the slot's end
    float entered, left;      // the first two of magnitudes
    float off, most;          // what pass may be off by; what it cannot exceed
    uint32_t live;            // bit i: token n - 1 - i has a decay that is not zero
    float pad;
};
constexpr int SLOT_CHUNKS = 64;   // of a slot in training: a lane each
template <class K>
constexpr size_t mix2_lds(bool dot) {
    return 4 * (size_t)K::TILE + 2 * (size_t)K::NP * K::PPL + 2 * sizeof(Decays<K::C>) +
           (dot ? SLOT_CHUNKS * sizeof(Chunk) + 2 * (2 * K::TT * K::C * 8 + K::NW * (K::C + 1) * 4) : 0);
}
// What rounding leaves open in a sum of such magnitudes
constexpr float SUM_OFF = 0x1p-22f;
// a number within +-most, and NaN as it is
__device__ __forceinline__ double within(double x, float most) { return x > most ? most : x < -most ? -most : x; }
// mix2: dk and dv of a slot, backwards in time, from q (y), k (x), v (z) and do (w), with
// dS in both orders: dv = mix(k, q, do), dk = mix(v, do, q).
// DOT: dg too, what passes from before token t to t or later.  With a_t and b_t the parts of
// q_t . dq_t and k_t . dk_t that come through the state (a: dots, from mix), E_{ts} =
// e^{G_t - G_s} (q_t . k_s) (do_t . v_s) the chunk's own pairs, s < t, and P what passes all of
// the chunk,
//   dg_t = P + sum of a from t on + sum of b before t + sum of E_{t' s}, t' >= t > s:
// no difference of large sums but in P.  Behind the chunk passes P + sum of b, before it P + sum
// of a, so P follows from <S, dS> at the slot's end, chunk by chunk backwards, and from that
// at its start forwards: each off by what the sums on its way are off by, the smaller is
// taken.  (From one side alone dg is lost where little gets through: with a loss on the last
// token and g = -0.2, 100 tokens before it.)  Nor can P exceed e^{G_C} max|S| sum|dS|,
// which ends what came from large sums nearby: with all of q . dq - k . dk in one sum over
// the slot, dg of fast decays was 2 to 60 times as far off.  Sums in fp64, E's too: in their
// differences a token with a decay of its own would drown in the rounding of the rest.
// PARTS: of dots and peaks, by channels.
//
// dg's work goes on beside the next chunk's pairs, in a wave that has none of them: 20000 packed
// x 16 x 128 326 us, in the last wave but one 353, at the end of a chunk 357.
//
// Measured, bf16: 8 x 1568 x 12 x 64 50 us; 20000 packed x 16 x 128 332 us, where four heads share
// a key and 328 MB of fp32 parts are written, 64 us of it.  Two states of D x D in registers
// leave two waves a SIMD (D <= 64: three), so a chunk's chain of products is seen in full; parts of
// the channels as in mix would form both kinds of pairs twice (343 us for 325 then).
template <class K, typename OT, bool DOT, int PARTS>
__global__ __launch_bounds__(K::NTH, K::OCC2) void kda_decay_mix2_kernel(const DecayArgs a) {
    static_assert(K::SPLIT == 1, "dg takes all channels");
    typedef typename K::ST ST;
    __shared__ __attribute__((aligned(16))) char lds[mix2_lds<K>(DOT)];
    char* Kt = lds;
    char* Q = Kt + K::TILE;
    char* V = Q + K::TILE;
    char* O = V + K::TILE;
    char* PA = O + K::TILE;
    char* PD = PA + K::NP * K::PPL;
    Decays<K::C>* dec = reinterpret_cast<Decays<K::C>*>(PD + K::NP * K::PPL);
    Chunk* chunks = reinterpret_cast<Chunk*>(dec + 2);                        // DOT: by number in the slot
    // of a chunk and the one before: E's sums over the other tokens, of X rows (k, v), [TT column tiles][C], and of Y
    // rows (q, do), [TT row tiles][C]; k . dk by waves, [NW][C]; sum |dS| by waves
    constexpr int EN = K::TT * K::C, PN = K::NW * K::C;
    double* e_own = reinterpret_cast<double*>(chunks + SLOT_CHUNKS);
    double* e_oth = e_own + 2 * EN;
    float* part = reinterpret_cast<float*>(e_oth + 2 * EN);
    float* weight = part + 2 * PN;

    int j, h, cols;
    work_of<1>(a, j, h, cols);
    const Slot s = slot_of(a, j);
    if (s.seq < 0) {
        if (s.seq == -1) {
            clear_rows<K::D, OT>(a.out, a, s, h);
            clear_rows<K::D, OT>(a.out2, a, s, h);
            if (DOT && a.dg)
                for (int i = threadIdx.x; i < s.n; i += K::NTH) a.dg[(int64_t)(s.tok0 + i) * a.H + h] = 0.f;
        }
        if (DOT && a.sums && threadIdx.x == 0) a.sums[(int64_t)j * a.H + h] = 0.0;
        return;
    }
    const int b = a.tab ? 0 : s.seq, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
    // dg's wave: the first one without a tile of pairs, if there is one
    constexpr int DD = K::D * K::D, LAST = K::NW - 1, DGW = K::NT < LAST ? K::NT : LAST;
    const float* s_in = a.s_in ? a.s_in + ((int64_t)(a.in_by_slot ? j : s.seq) * a.H + h) * DD : nullptr;
    State<K> sv, sk;   // dv's: [do][q]; dk's: [q][do]
    sv.load(s_in, wave, false);
    sk.load(s_in, wave, true);
    auto dot_all = [&](const float* p) {   // <p, dS>, for all threads
        double* sums = reinterpret_cast<double*>(lds);
        const double x = sk.dot(p, wave);
        if (l == 0) sums[wave] = x;
        lds_barrier();
        double y = 0.0;
#pragma unroll
        for (int k = 0; k < K::NW; ++k) y += sums[k];
        return y;
    };
    double passing = 0.0;   // <S, dS> behind the chunk
    if constexpr (DOT) {
        if (s_in && (!s.last || a.s_final)) {
            passing = dot_all(s.last ? a.s_final + ((int64_t)s.seq * a.H + h) * DD : a.starts + ((int64_t)(j + 1) * a.H + h) * DD);
            lds_barrier();
        }
    }
    float off = SUM_OFF * fabsf((float)passing);   // of it

    const float* g = a.g + b * a.gb + (int64_t)s.tok0 * a.gt + h * a.gh;
    Stage<K, K::D, true> rk, rq, rv, ro;
    float gv = 0.f;
    // the chunks are those of a pass forwards, so that dots and the sums of mix over them add up:
    // rows [i0, i0 + n) backwards, all but the first C of them
    const int n0 = s.n - (s.n - 1) / K::C * K::C;
    auto load = [&](int i0, int n) {
        const int t = s.tok0 + s.n - i0 - n;
        rk.load(at<ST>(a.x, b, t, h), (uint32_t)a.x.token * K::ES, n);
        rq.load(at<ST>(a.y, b, t, h), (uint32_t)a.y.token * K::ES, n);
        rv.load(at<ST>(a.z, b, t, h), (uint32_t)a.z.token * K::ES, n);
        ro.load(at<ST>(a.w, b, t, h), (uint32_t)a.w.token * K::ES, n);
    };
    auto load_g = [&](int i0, int n) {
        const int i = i0 + l;
        gv = l < n && i > 0 && i < s.n ? g[(int64_t)(s.n - i) * a.gt] : 0.f;
    };
    // dots, peaks and g of the chunk's tokens (those behind the last: of that), on their way until settle
    float av[PARTS], top[PARTS], gt = 0.f;
    double whole = 0.0;
    auto load_a = [&](int i0, int n) {
        const int t = s.n - 1 - i0 - min(l, n - 1);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            av[p] = a.dots[((int64_t)p * a.H + h) * a.B * a.T + (int64_t)b * a.T + s.tok0 + t];
            top[p] = a.peaks[((int64_t)p * a.H + h) * chunk_count(a.B, a.T, a.nslots) +
                             chunk_number((int64_t)b * a.T + s.tok0, j, (s.n - 1 - i0) / K::C)];
        }
        gt = g[(int64_t)t * a.gt];
    };
    auto store = [&](int n) {
        rk.store(Kt, n);
        rq.store(Q, n);
        rv.store(V, n);
        ro.store(O, n);
    };
    clear_upper<K>(PA);
    clear_upper<K>(PD);
    if constexpr (DOT)
        for (int v = threadIdx.x; v < 4 * EN; v += K::NTH) e_own[v] = 0.0;
    if (s.n > 0) {
        load(0, n0);
        if (wave == LAST) {
            load_g(0, n0);
            fill_decays<K::C>(dec, gv);
            load_g(n0, K::C);
        }
        store(n0);
        if (n0 < s.n) load(n0, K::C);
        lds_barrier();
    }
    // dg of the chunk of rows [i0, i0 + n), but for what passes it: one chunk late, beside the next one's pairs
    float all = 1.f;   // e^{sum of g over it}
    auto settle = [&](int i0, int n, int turn) {
        // lane l: token n - 1 - l of the chunk
        float x = 0.f, y = 0.f, size = 0.f, peak = 0.f;
        double cross = 0.0;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            y += av[p];
            peak = fmaxf(peak, top[p]);
        }
        if (l >= n) y = 0.f;
        if (l < n) {
#pragma unroll
            for (int k = 0; k < K::TT; ++k) cross += e_oth[turn * EN + k * K::C + l] - e_own[turn * EN + k * K::C + l];
#pragma unroll
            for (int k = 0; k < K::NW; ++k) x += part[turn * PN + k * K::C + l];
        }
#pragma unroll
        for (int k = 0; k < K::NW; ++k) size += weight[turn * K::NW + k];
        Chunk c;
        const double pairs = prefix32(cross), enter = prefix32((double)y), before = behind32((double)x, c.leave);
        c.enter = lane31(enter);
        c.entered = lane(prefix32(fabsf(y)), 31);
        c.left = lane(prefix32(fabsf(x)), 31);
        c.most = decay(lane(gt, n - 1)) * all * (peak * size);
        c.pass = within(passing - c.leave, c.most);
        c.off = off + SUM_OFF * c.left;
        if (c.most < c.off) c.off = c.most;
        c.live = (uint32_t)__ballot(l < n && !(gt < G_MIN));
        passing = c.pass + c.enter;
        off = c.off + SUM_OFF * c.entered;
        if (l == 0) chunks[(s.n - 1 - i0) / K::C] = c;
        if (l < n) {
            // (nothing passes a decay of zero: exactly; nor do pairs cross the chunk's first token)
            const double v = gt < G_MIN ? 0.0 : enter + before + (l < n - 1 ? pairs : 0.0);
            if (a.dg) a.dg[((int64_t)b * a.T + s.tok0 + s.n - 1 - i0 - l) * a.H + h] = (float)v;
            whole += v;
        }
    };
    int turn = 0;
    for (int i0 = 0, n = n0; i0 < s.n; i0 += n, n = K::C, turn ^= 1) {
        const Decays<K::C>& d = dec[turn];
        const bool more = i0 + n < s.n;
        if constexpr (DOT) {
            if (wave == DGW) {
                if (i0) settle(i0 == n0 ? 0 : i0 - K::C, i0 == n0 ? n0 : K::C, turn ^ 1);
                load_a(i0, n);
                all = d.all;
            }
        }
        bf16x8 wo[K::NPL], wq[K::NPL];
        w_frag<K, K::RB>(O, 0, wave, wo);
        w_frag<K, K::RB>(Q, 0, wave, wq);
        const Ends ends_o = take_ends<K>(wo), ends_q = take_ends<K>(wq);
#pragma unroll
        for (int k = 0; k < (K::NT + K::NW - 1) / K::NW; ++k) {
            const int id = wave + K::NW * k;
            if (id < K::NT) {
                int ti, si;
                tile_of(id, ti, si);
                const f32x4 m = mask_tile<K>(d, ti, si);
                const f32x4 pa = masked(pair_tile<K>(Kt, Q, ti, si), m, ti, si), pd = pair_tile<K>(V, O, ti, si);
                put_pair<K>(PA, pa, ti, si);
                put_pair<K>(PD, masked(pd, m, ti, si), ti, si);
                if constexpr (DOT) {
                    // a token's own pair passes no decay, and would drown what does where decays are fast
                    double e[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) e[i] = ti == si && 4 * (l >> 4) + i >= (l & 15) ? 0.0 : (double)(pa[i] * pd[i]);
                    double own = (e[0] + e[1]) + (e[2] + e[3]);
                    own += __shfl_xor(own, 16, 64);
                    own += __shfl_xor(own, 32, 64);
                    if (l < 16) e_own[turn * EN + si * K::C + 16 * ti + l] = own;
                    // sums over 16 lanes of four numbers, which the first two steps share out
                    const bool b0 = l & 1, b1 = l & 2;
                    const double x = (b0 ? e[2] : e[0]) + dpp<0xb1, 0xf>(b0 ? e[0] : e[2]),   // quad_perm: the other one,
                                 y = (b0 ? e[3] : e[1]) + dpp<0xb1, 0xf>(b0 ? e[1] : e[3]);
                    double oth = (b1 ? y : x) + dpp<0x4e, 0xf>(b1 ? x : y);                   // and the other two
                    oth += dpp<0x128, 0xf>(oth);                                              // row_ror:8, 4
                    oth += dpp<0x124, 0xf>(oth);
                    if ((l & 15) < 4) e_oth[turn * EN + ti * K::C + 16 * si + 4 * (l >> 4) + 2 * b0 + b1] = oth;
                }
            }
        }
        f32x4 o[K::TT], o2[K::TT];
        sv.apply(Kt, d, o);
        sk.apply(V, d, o2);
        if constexpr (DOT) {
            const float x = sk.weight();
            if (l == 63) weight[turn * K::NW + wave] = x;
            const int ch = 16 * wave + 4 * (l >> 4);
#pragma unroll
            for (int i = 0; i < K::TT; ++i) {
                const int t = 16 * i + (l & 15);
                const char* p = Kt + Sw<K::RB>::at(t, ch >> 3) + 2 * (ch & 7);
                const float x = quad_sum(dot4(tile4<K>(p), o2[i]));
                if (l < 16) part[turn * PN + wave * K::C + t] = x;
            }
        }
        sv.add(Q, wo, d.down, own_of<K>(ends_o, d.all), 1.f);
        sk.add(O, wq, d.down, own_of<K>(ends_q, d.all), 1.f);
        if (wave == LAST && more) {
            fill_decays<K::C>(dec + (turn ^ 1), gv);
            load_g(i0 + n + K::C, K::C);
        }
        lds_barrier();
        if (more) {
            store(K::C);
            if (i0 + n + K::C < s.n) load(i0 + n + K::C, K::C);
        }
        const int64_t row = (int64_t)b * a.T + s.tok0 + s.n - i0 - n, out = (row * a.H + h) * K::D;
        put_ends<K>(ends_o, o);
        put_ends<K>(ends_q, o2);
        add_pairs<K>(PA, wo, o);
        add_pairs<K>(PD, wq, o2);
        put_rows<K, OT, true>(static_cast<OT*>(a.out) + out, (uint32_t)(a.H * K::D), o2, wave, n);
        put_rows<K, OT, true>(static_cast<OT*>(a.out2) + out, (uint32_t)(a.H * K::D), o, wave, n);
        if (more) lds_barrier();
    }
    if constexpr (DOT) {
        const float* p = !a.starts ? nullptr : a.starts + ((int64_t)(a.in_by_slot ? j : s.seq) * a.H + h) * DD;
        double from = 0.0;   // what passes the slot's start
        if (p && s.n > 0) from = (double)decay(g[0]) * dot_all(p);
        if (wave == DGW) {
            if (s.n > 0) settle(s.n > n0 ? s.n - K::C : 0, s.n > n0 ? K::C : n0, turn ^ 1);
            float open = SUM_OFF * fabsf((float)from);
            double pass = 0.0;   // lane l: of chunk l
            const int count = (s.n + K::C - 1) / K::C;
            for (int i = 0; i < count; ++i) {
                const Chunk c = chunks[i];
                double x = within(from - c.enter, c.most);
                float o = open + SUM_OFF * c.entered;
                if (c.most < o) o = c.most;
                from = x + c.leave;
                open = o + SUM_OFF * c.left;
                if (c.off <= o) x = c.pass;
                if (l == i) {
                    pass = x;
                    whole += x * __popc(c.live);
                }
            }
            if (a.dg) {
                __threadfence_block();   // its other lanes' stores
                for (int i = l; i - l < s.n; i += 64) {
                    const double x = __shfl(pass, min(i, s.n - 1) / K::C, 64);
                    const int k = i / K::C, n = min(K::C, s.n - k * K::C);
                    if (i < s.n && (chunks[k].live >> (n - 1 - (i - k * K::C)) & 1)) {
                        float* d = a.dg + ((int64_t)b * a.T + s.tok0 + i) * a.H + h;
                        *d = (float)(*d + x);
                    }
                }
            }
            if (a.sums) {
#pragma unroll
                for (int m = 1; m < 64; m <<= 1) whole += __shfl_xor(whole, m, 64);
                if (l == 0) a.sums[(int64_t)j * a.H + h] = whole;
            }
        }
    }
    if (a.s_out && s.first) sv.store(a.s_out + ((int64_t)s.seq * a.H + h) * DD, wave, s.n > 0 ? decay(g[0]) : 1.f);
}

// ----------------------------------------------------------------------------
// between the slots
// ----------------------------------------------------------------------------

// Slots of packed sequences, cu[0 .. nseq] their limits (taken as rising and within
// [0, T], whatever they hold): tab as slot_of reads it, first[i] sequence i's first
// slot.  What lies before the first and behind the last sequence becomes slots of
// no sequence, after the others.  order: the slots as workgroups take them, whole ones
// first, so that the last round is of short ones.
constexpr int PLAN_TH = 1024;
__global__ __launch_bounds__(PLAN_TH) void kda_decay_plan_kernel(const int* cu, int nseq, int T, int seg_tokens, int4* tab,
                                                                 int* first, int* order, int nslots) {
    __shared__ int buf[PLAN_TH];
    __shared__ int carry_end, carry_slots, carry_whole;
    const int t = threadIdx.x;
    if (t == 0) {
        carry_end = min(max(cu[0], 0), T);
        carry_slots = 0;
        carry_whole = 0;
    }
    __syncthreads();   // (without sequences the next read is behind the loop)
    const int begin = min(max(cu[0], 0), T);
    for (int i0 = 0; i0 < nseq; i0 += PLAN_TH) {
        const int i = i0 + t;
        // the largest limit so far
        buf[t] = i < nseq ? min(max(cu[i + 1], 0), T) : 0;
        __syncthreads();
        for (int k = 1; k < PLAN_TH; k <<= 1) {
            const int x = t >= k ? buf[t - k] : 0;
            __syncthreads();
            buf[t] = max(buf[t], x);
            __syncthreads();
        }
        const int lo = max(carry_end, t ? buf[t - 1] : 0), hi = max(carry_end, buf[t]), top = max(carry_end, buf[PLAN_TH - 1]);
        __syncthreads();
        const int n = i < nseq ? hi - lo : 0, slots = i < nseq ? max(1, (n + seg_tokens - 1) / seg_tokens) : 0;
        buf[t] = slots;
        __syncthreads();
        for (int k = 1; k < PLAN_TH; k <<= 1) {
            const int x = t >= k ? buf[t - k] : 0;
            __syncthreads();
            buf[t] += x;
            __syncthreads();
        }
        const int at = carry_slots + buf[t] - slots, total = carry_slots + buf[PLAN_TH - 1];
        __syncthreads();
        const int whole = n / seg_tokens;
        buf[t] = whole;
        __syncthreads();
        for (int k = 1; k < PLAN_TH; k <<= 1) {
            const int x = t >= k ? buf[t - k] : 0;
            __syncthreads();
            buf[t] += x;
            __syncthreads();
        }
        const int whole_at = carry_whole + buf[t] - whole, whole_total = carry_whole + buf[PLAN_TH - 1];
        if (i < nseq) {
            first[i] = at;
            for (int k = 0; k < slots; ++k) {
                tab[at + k] = make_int4(lo + k * seg_tokens, min(seg_tokens, n - k * seg_tokens), i,
                                        (k == 0) | (k == slots - 1) << 1);
                // whole ones from the front; the others, of which at - whole_at came before, from behind
                order[k < whole ? whole_at + k : nslots - 1 - (at - whole_at)] = at + k;
            }
        }
        __syncthreads();
        if (t == 0) {
            carry_end = top;
            carry_slots = total;
            carry_whole = whole_total;
        }
        __syncthreads();
    }
    const int used = carry_slots, end = carry_end, wholes = carry_whole;
    if (t == 0) first[nseq] = used;
    const int lead = (begin + seg_tokens - 1) / seg_tokens, trail = (T - end + seg_tokens - 1) / seg_tokens;
    for (int k = t; k < nslots - used; k += PLAN_TH) {
        int4 v = make_int4(0, 0, -2, 0);
        if (k < lead) v = make_int4(k * seg_tokens, min(seg_tokens, begin - k * seg_tokens), -1, 0);
        else if (k - lead < trail)
            v = make_int4(end + (k - lead) * seg_tokens, min(seg_tokens, T - end - (k - lead) * seg_tokens), -1, 0);
        tab[used + k] = v;
        order[wholes + k] = used + k;
    }
}

// The state at each slot's start (REV: its adjoint at each slot's end), in place of
// what the slots add: one thread takes two elements through a sequence's slots, 16
// loads at a time.  Bound by the latency of its rounds of loads: 12 heads of 64
// over 79 slots (15.5 MB, read and written) 14 us, 32 loads at a time no less.
constexpr int SCAN_PER = 2;
template <bool REV>
__global__ __launch_bounds__(256) void kda_decay_scan_kernel(float* u, const float* seg, const float* s0, const int* first,
                                                             int per_seq, int H, int DD, int parts, int seq0) {
    typedef float vec __attribute__((ext_vector_type(SCAN_PER)));
    const int part = blockIdx.x % parts, sh = blockIdx.x / parts, in = sh / H, h = sh - in * H, seq = seq0 + in;
    const int e = SCAN_PER * (part * 256 + (int)threadIdx.x);
    if (e >= DD) return;
    const int lo = first ? first[seq] : seq * per_seq, count = (first ? first[seq + 1] : lo + per_seq) - lo;
    vec run = 0.f;
    if (s0) run = *reinterpret_cast<const vec*>(s0 + ((int64_t)seq * H + h) * DD + e);
    auto slot = [&](int i) { return (int64_t)(REV ? lo + count - 1 - i : lo + i) * H + h; };
    int i = 0;
    // (the last one adds nothing to a start)
    auto batch = [&](auto size) {
        constexpr int N = size();
        for (; i + N <= count - 1; i += N) {
            vec v[N];
            float f[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                v[k] = *reinterpret_cast<const vec*>(u + slot(i + k) * DD + e);
                f[k] = seg[slot(i + k)];
            }
#pragma unroll
            for (int k = 0; k < N; ++k) {
                *reinterpret_cast<vec*>(u + slot(i + k) * DD + e) = run;
#pragma unroll
                for (int x = 0; x < SCAN_PER; ++x) run[x] = fmaf(f[k], run[x], v[k][x]);
            }
        }
    };
    batch(std::integral_constant<int, 16>());
    batch(std::integral_constant<int, 4>());
    batch(std::integral_constant<int, 1>());
    if (count) *reinterpret_cast<vec*>(u + slot(count - 1) * DD + e) = run;
}

// one decay a head: its gradient is the sum over the slots
__global__ __launch_bounds__(64) void kda_decay_dg_sum_kernel(const double* sums, float* dg, int nslots, int H) {
    double x = 0.0;
    for (int j = threadIdx.x; j < nslots; j += 64) x += sums[(int64_t)j * H + blockIdx.x];
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) x += __shfl_xor(x, k, 64);
    if (threadIdx.x == 0) dg[blockIdx.x] = (float)x;
}

// gradients of a tensor whose heads are shared: sums over the state's heads, rounded once.
// Bound by its bytes: 20000 x 16 x 128 to 4 heads 31 to 33 us, 5.8 TB/s (what mix2 has just
// written is partly still in a cache).
template <typename OT>
__global__ __launch_bounds__(256) void kda_decay_group_kernel(const float* src, OT* dst, int64_t n4, int share, int D) {
    const int per = D / 4;
    for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < n4; v += (int64_t)gridDim.x * 256) {
        const int64_t head = v / per;
        const float* p = src + (head * share) * D + 4 * (v - head * per);
        f32x4 x = zero4();
        for (int k = 0; k < share; ++k) {
            const float4 y = *reinterpret_cast<const float4*>(p + (int64_t)k * D);
            x += f32x4{y.x, y.y, y.z, y.w};
        }
        put4<OT>(dst + 4 * v, x);
    }
}


// ----------------------------------------------------------------------------
// one token
// ----------------------------------------------------------------------------
struct StepArgs {
    Rows q, k, v;               // [row][head][D] (token: unused)
    const float* g;
    int64_t gb, gh;
    float* s;                   // [N][H][D][D]
    const int* slots;           // of each row, or null: its own number
    void* o;                    // [B][H][D]
    int B, H, N;
};

// A wave takes R rows of a state (rows of v's channels) through one token: loads of
// 16 bytes a lane, L lanes a row, all in flight together.  The states' bytes, read and
// written once, are all that counts up to about a thousand rows: 256 x 32 x 128 x 128 (1.07 GB both
// ways) 215 us, 5.0 TB/s; 200 of 12 x 64 x 64 (79 MB) 16 us.  With slots every wave looks through
// all rows for its own, B / 64 rounds of loads, which many small states do not hide: 1024 rows of 12 x
// 64 x 64 74 us (without slots 63), 4096 of 6 x 64 x 64 317 (147), 8192 944 (301).
template <int D>
struct StepCfg {
    static constexpr int L = D == 32 ? 8 : D == 64 ? 16 : 32, RP = 64 / L, R = D == 32 ? 32 : 16, NP = R / RP, PARTS = D / R;
};
template <int D, typename ST>
__global__ __launch_bounds__(256) void kda_decay_step_kernel(const StepArgs a) {
    typedef StepCfg<D> C;
    const int l = lane_id(), unit = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6));
    const int part = unit % C::PARTS, bh = unit / C::PARTS, b = bh / a.H, h = bh - b * a.H;
    if (b >= a.B) return;
    const int col = 4 * (l % C::L), row0 = part * C::R + l / C::L;
    const bool in = col < D;
    const int n = a.slots ? a.slots[b] : b;
    auto out = [&](int r) { return static_cast<ST*>(a.o) + ((int64_t)r * a.H + h) * D; };
    if (n < 0 || n >= a.N) {
        if (l < C::R) st1<ST>(out(b) + part * C::R + l, 0.f);
        return;
    }
    if (a.slots) {   // rows of one state follow each other: the first of them does all
        for (int i = l; i - l < b; i += 64)
            if (__any(i < b && a.slots[min(i, b - 1)] == n)) return;
    }
    float* s = a.s + ((int64_t)n * a.H + h) * D * D + (int64_t)row0 * D + (in ? col : 0);
    float4 x[C::NP];
#pragma unroll
    for (int i = 0; i < C::NP; ++i) x[i] = *reinterpret_cast<const float4*>(s + i * C::RP * D);
    for (int r = b; r < a.B;) {
        const ST *qp = static_cast<const ST*>(a.q.p) + r * a.q.batch + (h / a.q.share) * a.q.head,
                 *kp = static_cast<const ST*>(a.k.p) + r * a.k.batch + (h / a.k.share) * a.k.head,
                 *vp = static_cast<const ST*>(a.v.p) + r * a.v.batch + (h / a.v.share) * a.v.head;
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 q = in ? ld4<ST>(qp + col) : zero, k = in ? ld4<ST>(kp + col) : zero;
        const float f = decay(a.g[r * a.gb + h * a.gh]);
        ST* o = out(r);
#pragma unroll
        for (int i = 0; i < C::NP; ++i) {
            const int row = row0 + i * C::RP;
            const float v = ld1<ST>(vp + row);
            x[i] = make_float4(fmaf(f, x[i].x, v * k.x), fmaf(f, x[i].y, v * k.y), fmaf(f, x[i].z, v * k.z),
                               fmaf(f, x[i].w, v * k.w));
            float y = fmaf(x[i].x, q.x, x[i].y * q.y) + fmaf(x[i].z, q.z, x[i].w * q.w);
            if (!in) y = 0.f;
#pragma unroll
            for (int m = 1; m < C::L; m <<= 1) y += __shfl_xor(y, m, 64);
            if (l % C::L == 0) st1<ST>(o + row, y);
        }
        if (!a.slots) break;
        int next = a.B;
        for (int i0 = r + 1; i0 < a.B && next == a.B; i0 += 64) {
            const uint64_t m = __ballot(i0 + l < a.B && a.slots[min(i0 + l, a.B - 1)] == n);
            if (m) next = i0 + __builtin_ctzll(m);
        }
        r = next;
    }
    if (in)
#pragma unroll
        for (int i = 0; i < C::NP; ++i) *reinterpret_cast<float4*>(s + i * C::RP * D) = x[i];
}

// ----------------------------------------------------------------------------
// host
// ----------------------------------------------------------------------------
typedef kda_decay_args Args;

constexpr int64_t MAX_THREADS = (int64_t)1 << 32;   // of a launch: fewer

int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }

struct Plan {
    int seg_tokens, per_seq, nslots, packed;
    bool multi;   // the states between slots are in memory
};
// How many chunks of 64 tokens a slot has.  Sequences that fill the card by themselves are
// one slot each; else what is shared out costs a pass for the slots' states and a scan
// over them, and the workgroups come in rounds of as many as fit beside each other: the
// least of all counts.  (In chunks' times of a full card, 7.5 us at D = 64, bf16, where it was
// measured: a chunk takes 0.33 in a workgroup alone, a slot's beginning a third of a chunk;
// the pass for the states half of the forward pass, dq 1.2 of it and mix2, of which fewer
// fit, 2.1; the two more launches 0.9 and a slot of the scan 0.02.  8 x 1568 x 12 x 64 takes 48 us
// in slots of 3 chunks, 51 of 2, 50 of 4, 47 of 5, 81 whole, and with gradients 136, 154, 149, 144 and 392;
// 196 x 6 x 64 19 whole or of one chunk; 20000 packed x 16 x 128 forward and backward 792 of 7, 838 of 5,
// 848 of 6, 824 of 12, 906 of 3.  The figures are bf16's at D = 64 and 128; fp32 and heads of 32 and 96
// take them over.  At 8 x 1568 and one sequence of 2048 to 8192 their choice was within 6% of the
// best length for heads of 32 and 96 and small fp32 calls; 12% above it for fp32 8 x 1568 x 12 x 64
// with gradients, 235 us against 209, and 20% for fp32 8 x 1568 x 8 x 128 forward, 145 against 122.)
Plan plan_of(const Args& a, bool train) {
    Plan p;
    p.packed = a.cu != nullptr;
    const int64_t rows = p.packed ? 1 : a.B, chunks = std::max<int64_t>(1, (a.T + 63) / 64);
    // dg goes from chunk to chunk of a slot, whose errors add up, and has a lane for each
    const int64_t most = train ? SLOT_CHUNKS / 2 : chunks;
    const double fit = a.D <= 64 ? 1024 : 384, fit2 = a.D <= 64 ? 768 : 256;
    // rounds of `fit` that `whole` slots and `parts` slots of a `rest` of their length take
    const auto turns = [](double whole, double parts, double rest, double fit) {
        const double full = std::floor(whole / fit), left = whole - full * fit;
        const auto round = [&](double n) { return n > 0.0 ? 0.33 + 0.67 * std::min(1.0, n / fit) : 0.0; };
        if (left == 0.0) return full + rest * round(parts);
        return left + parts <= fit ? full + round(left + rest * parts) : full + 1.0 + rest * round(left + parts - fit);
    };
    double best = 0.0;
    int64_t seg = 0;
    for (int64_t c = 1; c <= most; c = c < 64 || c == chunks ? c + 1 : chunks) {
        const int64_t per = (chunks + c - 1) / c;
        const bool multi = p.packed || per > 1;
        // (packed sequences' last slots, of unknown lengths, are taken last and fill a round)
        const double slots = (double)a.T / (64 * c), all = p.packed ? slots : std::floor(slots), n = (double)rows * a.H;
        const auto t = [&](double f) { return turns(n * all, slots > all ? n : 0.0, slots - all, f); };
        double cost = t(fit) * (multi ? 1.5 : 1.0);
        if (train) cost += t(fit) * (multi ? 1.7 : 1.2) + t(fit2) * 2.1;
        cost *= c + 0.35;
        if (multi) cost += (0.9 + 0.02 * a.D / 64 * per) * (train ? 2 : 1);
        if (!seg || cost < best) {
            best = cost;
            seg = c;
        }
    }
    p.seg_tokens = (int)(64 * seg);
    p.per_seq = p.packed ? 0 : (int)((chunks + seg - 1) / seg);
    const int64_t n = p.packed ? a.nseq + 2 + a.T / p.seg_tokens : a.B * p.per_seq;
    p.nslots = n * a.H >= MAX_THREADS / (4 * a.D) ? -1 : (int)n;   // (4 D threads a slot and head)
    p.multi = p.packed || p.per_seq > 1;
    return p;
}

// Parts in bytes: the slots and the states at their starts, which the backward pass reads
// again (kept); and the backward pass' own
struct Layout {
    int64_t tab = -1, first = -1, order = -1, s = -1, seg = -1, kept = 0;
    int64_t ds = -1, segd = -1, dots = -1, peaks = -1, sums = -1, g0 = -1, g1 = -1, bytes = 0;
};
bool shared(const Args& a, const kda_decay_rows& r) { return r.heads != a.H; }
Layout layout_of(const Args& a, const Plan& p) {
    Layout l;
    auto take = [](int64_t& at, int64_t n) { const int64_t x = at; at += up16(n); return x; };
    if (p.packed) {
        l.tab = take(l.kept, 16 * (int64_t)p.nslots);
        l.first = take(l.kept, 4 * (a.nseq + 1));
        l.order = take(l.kept, 4 * (int64_t)p.nslots);
    }
    const int64_t st = 4 * (int64_t)p.nslots * a.H * a.D * a.D, sg = 4 * (int64_t)p.nslots * a.H, rows = 4 * a.B * a.T * a.H;
    if (p.multi) {
        l.s = take(l.kept, st);
        l.seg = take(l.kept, sg);
        l.ds = take(l.bytes, st);
        l.segd = take(l.bytes, sg);
    }
    if (a.dg) {
        l.dots = take(l.bytes, 2 * rows);   // (of two parts of the channels)
        l.peaks = take(l.bytes, 2 * 4 * a.H * chunk_count(a.B, a.T, p.nslots));
        if (a.dg_heads) l.sums = take(l.bytes, 2 * sg);
    }
    const bool kv = shared(a, a.k) || shared(a, a.v);
    if (kv || shared(a, a.q)) l.g0 = take(l.bytes, rows * a.D);
    if (kv) l.g1 = take(l.bytes, rows * a.D);
    return l;
}

constexpr int MAX_TOKEN_STRIDE = 1 << 24;
int check_operand(const Args& a, const kda_decay_rows& r, const char* name) {
    const int64_t es = a.dtype == KDA_DTYPE_BF16 ? 2 : 4;
    if (!r.p || reinterpret_cast<uintptr_t>(r.p) % 16 != 0)
        return api_fail(KDA_E_INVALID, "%s is NULL or not 16-byte aligned", name);
    if ((r.batch * es) % 16 || (r.token * es) % 16 || (r.head * es) % 16)
        return api_fail(KDA_E_INVALID, "%s: strides %lld, %lld, %lld are not whole 16-byte pieces", name, (long long)r.batch,
                        (long long)r.token, (long long)r.head);
    // (a chunk's rows are addressed by 32 bits)
    if (r.token < 0 || r.token > MAX_TOKEN_STRIDE)
        return api_fail(KDA_E_INVALID, "%s: token stride %lld: expected 0 to %d", name, (long long)r.token, MAX_TOKEN_STRIDE);
    return KDA_OK;
}
int check_sizes(const Args& a) {
    if (a.dtype != KDA_DTYPE_F32 && a.dtype != KDA_DTYPE_BF16)
        return api_fail(KDA_E_UNSUPPORTED, "dtype=%lld: expected 0 (fp32) or 1 (bf16)", (long long)a.dtype);
    if (a.D != 32 && a.D != 64 && a.D != 96 && a.D != 128)
        return api_fail(KDA_E_UNSUPPORTED, "D=%lld: expected 32, 64, 96 or 128", (long long)a.D);
    if (a.B < 0 || a.T < 0 || a.H < 1 || a.H > 65535 || a.B > 0x7fffffff || a.T > 0x7fffffff - 4096 || a.nseq < 0 ||
        a.nseq > 0x7fffffff)
        return api_fail(KDA_E_INVALID, "B=%lld T=%lld H=%lld nseq=%lld", (long long)a.B, (long long)a.T, (long long)a.H,
                        (long long)a.nseq);
    if (a.cu && a.B != 1) return api_fail(KDA_E_INVALID, "B=%lld: packed sequences are one row", (long long)a.B);
    const kda_decay_rows* r[3] = {&a.q, &a.k, &a.v};
    for (int i = 0; i < 3; ++i)
        if (r[i]->heads < 1 || a.H % r[i]->heads != 0)
            return api_fail(KDA_E_INVALID, "%c has %lld heads, which do not divide H=%lld", "qkv"[i], (long long)r[i]->heads,
                            (long long)a.H);
    return KDA_OK;
}
int check_ptr(const void* p, const char* name, int align) {
    if (!p || reinterpret_cast<uintptr_t>(p) % align != 0)
        return api_fail(KDA_E_INVALID, "%s is NULL or not %d-byte aligned", name, align);
    return KDA_OK;
}
#define DEC_TRY(x)                       \
    do {                                 \
        const int rc_ = (x);             \
        if (rc_ != KDA_OK) return rc_;   \
    } while (0)
#define DEC_HIP(x)                                                   \
    do {                                                             \
        const hipError_t e_ = (x);                                   \
        if (e_ != hipSuccess) return api_hip_fail(e_, "kda_decay");  \
    } while (0)

Rows rows_of(const Args& a, const kda_decay_rows& r) { return {r.p, r.batch, r.token, r.head, (int)(a.H / r.heads)}; }

DecayArgs base_of(const Args& a, const Plan& p, const Layout& l, char* kept) {
    DecayArgs d = {};
    d.g = a.g; d.gb = a.g_batch; d.gt = a.g_token; d.gh = a.g_head;
    d.B = (int)a.B; d.T = (int)a.T; d.H = (int)a.H;
    d.nseq = (int)(a.cu ? a.nseq : a.B);
    d.nslots = p.nslots; d.per_seq = p.per_seq; d.seg_tokens = p.seg_tokens;
    d.tab = p.packed ? reinterpret_cast<const int4*>(kept + l.tab) : nullptr;
    d.order = p.packed ? reinterpret_cast<const int*>(kept + l.order) : nullptr;
    d.in_by_slot = p.multi;
    return d;
}

template <class K, typename OT, bool STATES, bool GRAD, bool DOT>
hipError_t launch_mix(const DecayArgs& d, hipStream_t st) {
    hipLaunchKernelGGL((kda_decay_mix_kernel<K, OT, STATES, GRAD, DOT>), dim3((unsigned)(d.nslots * d.H * K::SPLIT)),
                       dim3(K::NTH), 0, st, d);
    return hipGetLastError();
}

// the states at the slots' limits: their starts (u, seg: kept), or (REV) their adjoints at the ends
template <bool REV>
hipError_t launch_scan(const DecayArgs& d, int D, float* u, const float* seg, const int* first, const float* s0, hipStream_t st) {
    const int DD = D * D, parts = (DD / SCAN_PER + 255) / 256;
    const int most = std::max(1, (int)((MAX_THREADS - 1) / 256 / ((int64_t)parts * d.H)));   // sequences a launch
    for (int seq0 = 0; seq0 < d.nseq; seq0 += std::min(most, d.nseq - seq0)) {
        hipLaunchKernelGGL(kda_decay_scan_kernel<REV>, dim3((unsigned)(std::min(most, d.nseq - seq0) * d.H * parts)), dim3(256), 0, st, u,
                           seg, s0, first, d.per_seq, d.H, DD, parts, seq0);
        const hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
    }
    return hipSuccess;
}

hipError_t launch_dg_sum(const double* sums, float* dg, int nslots, int H, hipStream_t st) {
    hipLaunchKernelGGL(kda_decay_dg_sum_kernel, dim3((unsigned)H), dim3(64), 0, st, sums, dg, nslots, H);
    return hipGetLastError();
}

template <typename OT>
hipError_t launch_group(const float* src, void* dst, const Args& a, const kda_decay_rows& r, hipStream_t st) {
    const int64_t n4 = a.B * a.T * r.heads * a.D / 4;
    if (n4 == 0) return hipSuccess;
    hipLaunchKernelGGL(kda_decay_group_kernel<OT>, dim3((unsigned)std::min<int64_t>((n4 + 255) / 256, 8192)), dim3(256), 0, st, src,
                       static_cast<OT*>(dst), n4, (int)(a.H / r.heads), (int)a.D);
    return hipGetLastError();
}

template <int D>
constexpr int SPLIT_OF = D > 64 ? 2 : 1;
template <int D, bool F32>
int forward(const Args& a, hipStream_t st) {
    typedef Cfg<D, F32, SPLIT_OF<D>> K;
    const Plan p = plan_of(a, a.train != 0);
    const Layout l = layout_of(a, p);
    char* kept = static_cast<char*>(a.train ? a.kept : a.workspace);
    DecayArgs d = base_of(a, p, l, kept);
    int* first = p.packed ? reinterpret_cast<int*>(kept + l.first) : nullptr;
    if (p.packed) {
        hipLaunchKernelGGL(kda_decay_plan_kernel, dim3(1), dim3(PLAN_TH), 0, st, a.cu, (int)a.nseq, (int)a.T, p.seg_tokens,
                           reinterpret_cast<int4*>(kept + l.tab), first, reinterpret_cast<int*>(kept + l.order), p.nslots);
        DEC_HIP(hipGetLastError());
    }
    if (p.multi) {
        DecayArgs m = d;
        m.y = rows_of(a, a.k);
        m.w = rows_of(a, a.v);
        m.s_out = reinterpret_cast<float*>(kept + l.s);
        m.seg = reinterpret_cast<float*>(kept + l.seg);
        DEC_HIP((launch_mix<K, float, true, false, false>(m, st)));
        DEC_HIP(launch_scan<false>(m, D, m.s_out, m.seg, first, a.s0, st));
    }
    d.x = rows_of(a, a.q);
    d.y = rows_of(a, a.k);
    d.w = rows_of(a, a.v);
    d.out = a.o;
    d.s_in = p.multi ? reinterpret_cast<float*>(kept + l.s) : a.s0;
    d.s_out = a.s_final;
    DEC_HIP((launch_mix<K, typename K::ST, false, false, false>(d, st)));
    return KDA_OK;
}

template <class K, typename OT, bool DOT, int PARTS>
hipError_t launch_mix2(const DecayArgs& d, hipStream_t st) {
    hipLaunchKernelGGL((kda_decay_mix2_kernel<K, OT, DOT, PARTS>), dim3((unsigned)(d.nslots * d.H)), dim3(K::NTH), 0, st, d);
    return hipGetLastError();
}

template <int D, bool F32, bool DOT>
int backward(const Args& a, hipStream_t st) {
    typedef Cfg<D, F32, SPLIT_OF<D>> K;
    typedef Cfg<D, F32> K2;
    typedef typename K::ST ST;
    const Plan p = plan_of(a, true);
    const Layout l = layout_of(a, p);
    char *ws = static_cast<char*>(a.workspace), *kept = static_cast<char*>(a.kept);
    const DecayArgs base = base_of(a, p, l, kept);
    const Rows q = rows_of(a, a.q), k = rows_of(a, a.k), v = rows_of(a, a.v);
    kda_decay_rows dout = a.dout;
    dout.heads = a.H;
    const Rows o = rows_of(a, dout);
    const auto part = [&](char* at, int64_t n) { return n < 0 ? nullptr : reinterpret_cast<float*>(at + n); };
    float *starts = part(kept, l.s), *dends = part(ws, l.ds), *dots = part(ws, l.dots), *g0 = part(ws, l.g0), *g1 = part(ws, l.g1);
    DecayArgs d = base;
    d.x = o; d.y = v; d.w = k; d.z = q;
    d.s_in = p.multi ? starts : a.s0;
    d.dots = dots;
    d.peaks = part(ws, l.peaks);
    d.s_out = dends;
    d.seg = part(ws, l.segd);
    const auto scan = [&] {
        return launch_scan<true>(base, D, dends, d.seg, reinterpret_cast<const int*>(part(kept, l.first)), a.ds_final, st);
    };
    if (p.multi && !K::WITH_DS) {   // dS of the slots by itself; else with dq
        DecayArgs m = d;
        m.y = q; m.w = o;
        DEC_HIP((launch_mix<K, float, true, true, false>(m, st)));
        DEC_HIP(scan());
    }
    d.out = shared(a, a.q) ? g0 : a.dq;
    if (shared(a, a.q)) {
        DEC_HIP((launch_mix<K, float, false, true, DOT>(d, st)));
        DEC_HIP(launch_group<ST>(g0, a.dq, a, a.q, st));
    } else {
        DEC_HIP((launch_mix<K, ST, false, true, DOT>(d, st)));
    }
    if (p.multi && K::WITH_DS) DEC_HIP(scan());
    d = base;
    d.x = k; d.y = q; d.z = v; d.w = o;
    d.s_in = p.multi ? dends : a.ds_final;
    d.s_out = a.ds0;
    double* sums = reinterpret_cast<double*>(part(ws, l.sums));
    d.dots = dots;
    d.peaks = part(ws, l.peaks);
    d.starts = p.multi ? starts : a.s0;
    d.s_final = a.ds_final ? a.s_final : nullptr;
    d.dg = sums ? nullptr : a.dg;
    d.sums = sums;
    if (shared(a, a.k) || shared(a, a.v)) {
        d.out = g0; d.out2 = g1;
        DEC_HIP((launch_mix2<K2, float, DOT, K::SPLIT>(d, st)));
        DEC_HIP(launch_group<ST>(g0, a.dk, a, a.k, st));
        DEC_HIP(launch_group<ST>(g1, a.dv, a, a.v, st));
    } else {
        d.out = a.dk; d.out2 = a.dv;
        DEC_HIP((launch_mix2<K2, ST, DOT, K::SPLIT>(d, st)));
    }
    if (sums) DEC_HIP(launch_dg_sum(sums, a.dg, d.nslots, d.H, st));
    return KDA_OK;
}

template <int D>
int forward_of(const Args& a, hipStream_t st) {
    return a.dtype == KDA_DTYPE_F32 ? forward<D, true>(a, st) : forward<D, false>(a, st);
}
template <int D>
int backward_of(const Args& a, hipStream_t st) {
    if (a.dg) return a.dtype == KDA_DTYPE_F32 ? backward<D, true, true>(a, st) : backward<D, false, true>(a, st);
    return a.dtype == KDA_DTYPE_F32 ? backward<D, true, false>(a, st) : backward<D, false, false>(a, st);
}

template <int D>
hipError_t launch_step(const StepArgs& a, bool f32, hipStream_t st) {
    const dim3 grid((unsigned)(((int64_t)a.B * a.H * StepCfg<D>::PARTS + 3) / 4));
    if (f32) hipLaunchKernelGGL((kda_decay_step_kernel<D, float>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kda_decay_step_kernel<D, uint16_t>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

int check_ws(const void* p, const char* name, int64_t have, int64_t need) {
    if (!need) return KDA_OK;
    DEC_TRY(check_ptr(p, name, 16));
    if (have < need) return api_fail(KDA_E_WORKSPACE, "%s has %lld bytes, needs %lld", name, (long long)have, (long long)need);
    return KDA_OK;
}
int check_common(const Args& a, bool bwd) {
    DEC_TRY(check_sizes(a));
    const Plan p = plan_of(a, bwd || a.train);
    if (p.nslots < 0) return api_fail(KDA_E_UNSUPPORTED, "B=%lld T=%lld H=%lld: too many workgroups", (long long)a.B, (long long)a.T, (long long)a.H);
    if (a.B * a.T > 0) {
        DEC_TRY(check_operand(a, a.q, "q"));
        DEC_TRY(check_operand(a, a.k, "k"));
        DEC_TRY(check_operand(a, a.v, "v"));
        DEC_TRY(check_ptr(a.g, "g", 4));
    }
    if (a.cu) DEC_TRY(check_ptr(a.cu, "cu", 4));
    if (a.s0) DEC_TRY(check_ptr(a.s0, "s0", 16));
    const Layout l = layout_of(a, p);
    if (bwd || a.train) DEC_TRY(check_ws(a.kept, "kept", a.kept_bytes, l.kept));
    else DEC_TRY(check_ws(a.workspace, "workspace", a.ws_bytes, l.kept));
    if (bwd) DEC_TRY(check_ws(a.workspace, "workspace", a.ws_bytes, l.bytes));
    return KDA_OK;
}

}  // namespace

}  // namespace kda

using namespace kda;

extern "C" {

size_t kda_decay_workspace_size(int pass, const kda_decay_args* args) {
    if (!args || check_sizes(*args) != KDA_OK) return 0;
    const Plan p = plan_of(*args, pass != KDA_PASS_FWD);
    if (p.nslots < 0) return 0;
    const Layout l = layout_of(*args, p);
    return (size_t)(pass == KDA_PASS_BWD ? l.bytes : l.kept);
}

int kda_decay_fwd(const kda_decay_args* args, void* stream) {
    if (!args) return api_fail(KDA_E_INVALID, "args is NULL");
    const Args& a = *args;
    DEC_TRY(check_common(a, false));
    if (a.B * a.T > 0) DEC_TRY(check_ptr(a.o, "o", 16));
    if (a.s_final) DEC_TRY(check_ptr(a.s_final, "s_final", 16));
    if (a.B == 0) return KDA_OK;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    switch (a.D) {
        case 32: return forward_of<32>(a, st);
        case 64: return forward_of<64>(a, st);
        case 96: return forward_of<96>(a, st);
        default: return forward_of<128>(a, st);
    }
}

int kda_decay_bwd(const kda_decay_args* args, void* stream) {
    if (!args) return api_fail(KDA_E_INVALID, "args is NULL");
    const Args& a = *args;
    DEC_TRY(check_common(a, true));
    if (a.B * a.T > 0) {
        DEC_TRY(check_operand(a, a.dout, "dout"));
        DEC_TRY(check_ptr(a.dq, "dq", 16));
        DEC_TRY(check_ptr(a.dk, "dk", 16));
        DEC_TRY(check_ptr(a.dv, "dv", 16));
    }
    if (a.ds_final) DEC_TRY(check_ptr(a.ds_final, "ds_final", 16));
    if (a.ds0) DEC_TRY(check_ptr(a.ds0, "ds0", 16));
    if (a.dg) {
        DEC_TRY(check_ptr(a.dg, "dg", 4));
        if (a.ds_final) DEC_TRY(check_ptr(a.s_final, "s_final (of the forward pass, for dg)", 16));
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (a.B == 0) {
        if (a.dg && a.dg_heads) DEC_HIP(launch_dg_sum(nullptr, a.dg, 0, (int)a.H, st));   // zeros
        return KDA_OK;
    }
    switch (a.D) {
        case 32: return backward_of<32>(a, st);
        case 64: return backward_of<64>(a, st);
        case 96: return backward_of<96>(a, st);
        default: return backward_of<128>(a, st);
    }
}

int kda_decay_step(const kda_decay_args* args, const int32_t* slots, int64_t states, void* stream) {
    if (!args) return api_fail(KDA_E_INVALID, "args is NULL");
    const Args& a = *args;
    DEC_TRY(check_sizes(a));
    if (a.cu || a.T != 1) return api_fail(KDA_E_INVALID, "T=%lld: a step takes one token of each row", (long long)a.T);
    if (a.B == 0) return KDA_OK;
    if (states < 0 || states > 0x7fffffff || (!slots && states != a.B))
        return api_fail(KDA_E_INVALID, "%lld states for %lld rows", (long long)states, (long long)a.B);
    if (a.B * a.H >= MAX_THREADS / 512) return api_fail(KDA_E_UNSUPPORTED, "B=%lld H=%lld: too many workgroups", (long long)a.B, (long long)a.H);
    DEC_TRY(check_operand(a, a.q, "q"));
    DEC_TRY(check_operand(a, a.k, "k"));
    DEC_TRY(check_operand(a, a.v, "v"));
    DEC_TRY(check_ptr(a.g, "g", 4));
    DEC_TRY(check_ptr(a.o, "o", 16));
    if (states) DEC_TRY(check_ptr(a.s0, "s0", 16));
    if (slots) DEC_TRY(check_ptr(slots, "slots", 4));
    StepArgs d = {};
    d.q = rows_of(a, a.q); d.k = rows_of(a, a.k); d.v = rows_of(a, a.v);
    d.g = a.g; d.gb = a.g_batch; d.gh = a.g_head;
    d.s = const_cast<float*>(a.s0); d.slots = slots; d.o = a.o;
    d.B = (int)a.B; d.H = (int)a.H; d.N = (int)states;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool f32 = a.dtype == KDA_DTYPE_F32;
    switch (a.D) {
        case 32: DEC_HIP(launch_step<32>(d, f32, st)); break;
        case 64: DEC_HIP(launch_step<64>(d, f32, st)); break;
        case 96: DEC_HIP(launch_step<96>(d, f32, st)); break;
        default: DEC_HIP(launch_step<128>(d, f32, st));
    }
    return KDA_OK;
}

}  // extern "C"
