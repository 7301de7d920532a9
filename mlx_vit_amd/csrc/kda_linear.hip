// kda_linear.hip -- linear maps with their epilogue: y = act(x W^T + b) + r, the
// products of their backward pass, and the C ABI around them.
//
//   forward   y[m][n] = act(sum_k x[m][k] W[n][k] + b[n]) + r[m][n], z (before act) on request
//   dgrad     dx[m][k] = (sum_n dz[m][n] W[n][k]) * act'(zin[m][k])
//   wgrad     dW[n][k] = sum_m dz[m][n] x[m][k], db[n] = sum_m dz[m][n]   (fp32; bf16: kda_wgrad.hip)
//
// Both are one product C[m][n] = sum_k A[m][k] B(k, n); the operand whose rows
// run along the contracted index (W in dgrad, both in wgrad) reaches the MFMA
// through transposing LDS reads, so nothing is transposed in memory.
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
    int vec;                // C, bias, res, zin, zout: groups of four columns are aligned, N % 4 == 0
    int vec_a, vec_b;       // fp32: rows of A, B can be read four floats at a time
    int splits, k_per;      // fp32 wgrad: parts of the contracted index, k_per (a multiple of the step) each
    float *part, *bpart;    // and their partial sums, [split][M][N] and [split][M]
};

// ----------------------------------------------------------------------------
// activations: 0 none, 1 gelu (z Phi(z)), 2 silu (z sigma(z))
// ----------------------------------------------------------------------------

// Phi(z) and e^{-z^2/2}.  EXACT: the library's erf and exp.  Otherwise, for
// results rounded to bf16, Phi(-|z|) = e^{-u^2} P(t) / 2, u = |z| / sqrt 2,
// t = 1 / (1 + 0.3275911 u), Abramowitz & Stegun 7.1.26 (|error| of erf <=
// 1.5e-7, 1 / 13000 of a bf16 half step of Phi near 1).
template <bool EXACT>
__device__ __forceinline__ float phi_exp(float z, float& e) {
    if constexpr (EXACT) {
        e = expf(-0.5f * z * z);
        return 0.5f * (1.f + erff(z * 0.70710678118654752f));
    } else {
        const float u = fabsf(z) * 0.70710678f, t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, u, 1.f));
        e = __builtin_amdgcn_exp2f(-1.4426950408889634f * u * u);
        float p = fmaf(1.061405429f, t, -1.453152027f);
        p = fmaf(p, t, 1.421413741f);
        p = fmaf(p, t, -0.284496736f);
        p = fmaf(p, t, 0.254829592f);
        const float tail = 0.5f * p * t * e;
        return z >= 0.f ? 1.f - tail : tail;
    }
}
template <bool EXACT>
__device__ __forceinline__ float sigma(float z) {
    if constexpr (EXACT) return 1.f / (1.f + expf(-z));
    else return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
}
template <int ACT, bool EXACT>
__device__ __forceinline__ float act(float z) {
    if constexpr (ACT == 1) {
        float e;
        return z * phi_exp<EXACT>(z, e);
    } else if constexpr (ACT == 2) {
        return z * sigma<EXACT>(z);
    } else {
        return z;
    }
}
template <int ACT, bool EXACT>
__device__ __forceinline__ float act_grad(float z) {
    if constexpr (ACT == 1) {
        float e;
        const float p = phi_exp<EXACT>(z, e);
        return fmaf(z * e, 0.39894228040143268f, p);
    } else if constexpr (ACT == 2) {
        const float s = sigma<EXACT>(z);
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

// The epilogue of four columns n..n+3 of row m: DG: times act'(zin) (zin null:
// nothing); else bias, z out, activation, residual
template <typename T, int ACT, bool DG, bool EXACT>
__device__ __forceinline__ void finish4(const GemmArgs& a, int m, int n, f32x4 acc, const float4& bias) {
    const int left = a.N - n;
    const bool vec = a.vec;
    float4 v = make_float4(acc[0], acc[1], acc[2], acc[3]);
    if constexpr (DG) {
        if constexpr (ACT != 0) {
            const float4 z = ldc4<T>(static_cast<const T*>(a.zin) + (size_t)m * a.ldzi + n, left, vec);
            v.x *= act_grad<ACT, EXACT>(z.x);
            v.y *= act_grad<ACT, EXACT>(z.y);
            v.z *= act_grad<ACT, EXACT>(z.z);
            v.w *= act_grad<ACT, EXACT>(z.w);
        }
    } else {
        v.x += bias.x; v.y += bias.y; v.z += bias.z; v.w += bias.w;
        if (a.zout) stc4<T>(static_cast<T*>(a.zout) + (size_t)m * a.ldzo + n, v, left, vec);
        v.x = act<ACT, EXACT>(v.x);
        v.y = act<ACT, EXACT>(v.y);
        v.z = act<ACT, EXACT>(v.z);
        v.w = act<ACT, EXACT>(v.w);
        if (a.res) {
            const float4 r = ldc4<T>(static_cast<const T*>(a.res) + (size_t)m * a.ldr + n, left, vec);
            v.x += r.x; v.y += r.y; v.z += r.z; v.w += r.w;
        }
    }
    stc4<T>(static_cast<T*>(a.c) + (size_t)m * a.ldc + n, v, left, vec);
}
template <typename T, bool DG>
__device__ __forceinline__ float4 bias4(const GemmArgs& a, int n) {
    if (DG || !a.bias || n >= a.N) return make_float4(0.f, 0.f, 0.f, 0.f);
    return ldc4<T>(static_cast<const T*>(a.bias) + n, a.N - n, a.vec);
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
// read takes 16 rows of one chunk), or rows across it of at least 256 bytes (a
// transposing read takes rows 8 g .. 8 g + 3 of 32 bytes)
template <int RB>
__device__ __forceinline__ int key_k(int r) {
    return RB == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
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
    const int at = (((b >> 4) ^ key_t(r)) << 4) + (b & 15);   // row r + 4 has the same key
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
        c = ((p % RB) >> 4) ^ (TR ? key_t(r) : key_k<RB>(r));
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

// at most n of the last steps' DMA (L instructions each) outstanding
template <int L, int MAX>
__device__ __forceinline__ void wait_steps(int n) {
    if constexpr (MAX > 0) {
        if (n >= MAX) {
            dma_wait<MAX * L>();
            return;
        }
        wait_steps<L, MAX - 1>(n);
    } else {
        dma_wait<0>();
    }
}

// C tile of BM x BN by WR x WC waves, BK of the contracted index a step, NST
// buffers.  BT: B's rows run across the contracted index (dgrad).
template <int BM, int BN, int BK, int NST, int WR, int WC, bool BT, int ACT, bool DG>
__global__ __launch_bounds__(64 * WR * WC, 2) void kda_linear_bf16_kernel(const GemmArgs a) {
    constexpr int W = WR * WC, RBA = 2 * BK, RBB = BT ? 2 * BN : 2 * BK, ROWB = BT ? BK : BN;
    constexpr int SA = BM * RBA, STAGE = SA + ROWB * RBB;
    constexpr int FM = BM / WR / 16, FN = BN / WC / 16;
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
    const int steps = (a.K + BK - 1) / BK, tail = a.K - (steps - 1) * BK;
    auto issue = [&](int s) {
        const uint32_t st = base + (uint32_t)((s % NST) * STAGE);
        if (s == steps - 1 && tail < BK) {
            da.init(a.lda, a.M - 1 - m0, (tail - 1) / 8, w);
            if constexpr (BT) db.init(a.ldb, tail - 1, (a.N - 1 - n0) / 8, w);
            else db.init(a.ldb, a.N - 1 - n0, (tail - 1) / 8, w);
        }
        da.issue(ga, st, w);
        db.issue(gb, st + SA, w);
        ga += 2 * BK;
        gb += stepb;
    };
    for (int s = 0; s < min(steps, NST - 1); ++s) issue(s);
    f32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = zero4();
    // Each step: this wave's share of it has landed (the later steps' stays in
    // flight), barrier -- so every wave's has, and every wave has read the step
    // before, whose buffer is filled next -- then issue and compute.
    for (int s = 0; s < steps; ++s) {
        wait_steps<L, NST - 2>(min(NST - 2, steps - 1 - s));
        lds_barrier();
        char* st = lds + (s % NST) * STAGE;
        if (s == steps - 1 && tail < BK) {
            zero_tail<BM, RBA, false, 64 * W>(st, tail);
            zero_tail<ROWB, RBB, BT, 64 * W>(st + SA, tail);
            lds_barrier();
        }
        if (s + NST - 1 < steps) issue(s + NST - 1);
#pragma unroll
        for (int ks = 0; ks < BK / 32; ++ks) {
            bf16x8 fa[FM], fb[FN];
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                if constexpr (BT) fb[i] = frag_t<RBB>(st + SA, wn + 16 * i, 32 * ks);
                else fb[i] = frag_k<RBB>(st + SA, wn + 16 * i, 4 * ks);
            }
#pragma unroll
            for (int j = 0; j < FM; ++j) fa[j] = frag_k<RBA>(st, wm + 16 * j, 4 * ks);
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FM; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[i], fa[j], acc[i][j], 0, 0, 0);
        }
    }
    // B's fragment first: a lane holds four consecutive columns n of one row m
#pragma unroll
    for (int i = 0; i < FN; ++i) {
        const int n = n0 + wn + 16 * i + 4 * g4;
        const float4 bias = bias4<uint16_t, DG>(a, n);
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int m = m0 + wm + 16 * j + r16;
            if (m < a.M && n < a.N) finish4<uint16_t, ACT, DG, false>(a, m, n, acc[i][j], bias);
        }
    }
}

// ----------------------------------------------------------------------------
// fp32: each operand split exactly into three bf16 parts on its way to LDS
// ----------------------------------------------------------------------------

// x = h + m + l, each the next 8 bits of x's 24 (truncation, so nothing
// overflows and every difference is exact); the four values' parts packed.
// An infinite x gives a NaN part.
__device__ __forceinline__ void split3(const float4& x, uint2& h, uint2& m, uint2& l) {
    const float v[4] = {x.x, x.y, x.z, x.w};
    uint32_t a[4], b[4], c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        a[e] = __float_as_uint(v[e]) & 0xffff0000u;
        const float r = v[e] - __uint_as_float(a[e]);
        b[e] = __float_as_uint(r) & 0xffff0000u;
        c[e] = __float_as_uint(r - __uint_as_float(b[e]));
    }
    constexpr uint32_t HI = 0x07060302u;   // the high halves of two registers
    h = make_uint2(__builtin_amdgcn_perm(a[1], a[0], HI), __builtin_amdgcn_perm(a[3], a[2], HI));
    m = make_uint2(__builtin_amdgcn_perm(b[1], b[0], HI), __builtin_amdgcn_perm(b[3], b[2], HI));
    l = make_uint2(__builtin_amdgcn_perm(c[1], c[0], HI), __builtin_amdgcn_perm(c[3], c[2], HI));
}

// A 128 x 32 (or, TR, 32 x 128) tile of fp32 rows through registers into three
// bf16 planes of 8 KB
template <bool TR>
struct Stage32 {
    static constexpr int RB = TR ? 256 : 64, PLANE = 8192;
    float4 v[4];
    // row and first column of this thread's piece i
    __device__ __forceinline__ static int row(int i) { return TR ? (threadIdx.x >> 5) + 8 * i : (threadIdx.x >> 3) + 32 * i; }
    __device__ __forceinline__ static int col() { return TR ? 4 * (threadIdx.x & 31) : 4 * (threadIdx.x & 7); }
    // rows, cols: how many of them exist past (r0, c0); what does not is zero
    __device__ __forceinline__ void load(const float* base, int64_t ld, int rows, int cols, bool vec) {
        const int c = col();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row(i);
            v[i] = r < rows && c < cols ? ldc4<float>(base + (size_t)r * ld + c, cols - c, vec && c + 4 <= cols)
                                        : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    __device__ __forceinline__ void store(char* tile) const {
        const int b = 2 * col();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row(i);
            char* p = tile + r * RB + (((b >> 4) ^ (TR ? key_t(r) : key_k<RB>(r))) << 4) + (b & 15);
            uint2 h, m, l;
            split3(v[i], h, m, l);
            *reinterpret_cast<uint2*>(p) = h;
            *reinterpret_cast<uint2*>(p + PLANE) = m;
            *reinterpret_cast<uint2*>(p + 2 * PLANE) = l;
        }
    }
};

// C tile of 128 x 128 by 2 x 2 waves, 32 of the contracted index a step.  AT, BT:
// the operand's rows run across the contracted index.  PART: one of a.splits
// parts of it, into a.part (and with a.bpart A's column sums).
template <bool AT, bool BT, int ACT, bool DG, bool PART>
__global__ __launch_bounds__(256, 2) void kda_linear_f32_kernel(const GemmArgs a) {
    constexpr int BK = 32, RBA = AT ? 256 : 64, RBB = BT ? 256 : 64, PL = 8192;
    __shared__ __attribute__((aligned(1024))) char lds[6 * PL];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id(), r16 = l & 15, g4 = l >> 4;
    const int wm = (w >> 1) * 64, wn = (w & 1) * 64;
    const int tiles = a.mt * a.nt, split = PART ? (int)blockIdx.x / tiles : 0;
    int mi, ni;
    tile_of((int)blockIdx.x - split * tiles, tiles, a.mt, a.nt, mi, ni);
    const int m0 = mi * 128, n0 = ni * 128;
    const int k0 = PART ? split * a.k_per : 0, k1 = PART ? min(a.K, k0 + a.k_per) : a.K;
    const float *A = static_cast<const float*>(a.a), *B = static_cast<const float*>(a.b);
    Stage32<AT> sa;
    Stage32<BT> sb;
    auto load = [&](int k) {
        if constexpr (AT) sa.load(A + (size_t)k * a.lda + m0, a.lda, k1 - k, a.M - m0, a.vec_a);
        else sa.load(A + (size_t)m0 * a.lda + k, a.lda, a.M - m0, k1 - k, a.vec_a);
        if constexpr (BT) sb.load(B + (size_t)k * a.ldb + n0, a.ldb, k1 - k, a.N - n0, a.vec_b);
        else sb.load(B + (size_t)n0 * a.ldb + k, a.ldb, a.N - n0, k1 - k, a.vec_b);
    };
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = zero4();
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool sums = PART && a.bpart && ni == 0;
    load(k0);
    for (int k = k0; k < k1; k += BK) {
        if (k > k0) lds_barrier();   // every wave has read the step before
        sa.store(lds);
        sb.store(lds + 3 * PL);
        if (sums)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sum.x += sa.v[i].x; sum.y += sa.v[i].y; sum.z += sa.v[i].z; sum.w += sa.v[i].w;
            }
        lds_barrier();
        if (k + BK < k1) load(k + BK);
        // products of parts down to 2^-16 of the largest: hh, hm, mh, hl, lh, mm
        bf16x8 fb[3][4];
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const char* t = lds + (3 + p) * PL;
                if constexpr (BT) fb[p][i] = frag_t<RBB>(t, wn + 16 * i, 0);
                else fb[p][i] = frag_k<RBB>(t, wn + 16 * i, 0);
            }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bf16x8 fa[3];
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                if constexpr (AT) fa[p] = frag_t<RBA>(lds + p * PL, wm + 16 * j, 0);
                else fa[p] = frag_k<RBA>(lds + p * PL, wm + 16 * j, 0);
            }
            // smallest first
#pragma unroll
            for (int q = 0; q < 6; ++q) {
                constexpr int PB[6] = {0, 2, 1, 0, 1, 0}, PA[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[PB[q]][i], fa[PA[q]], acc[i][j], 0, 0, 0);
            }
        }
    }
    if constexpr (PART) {
        float* part = a.part + (size_t)split * a.M * a.N;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = n0 + wn + 16 * i + 4 * g4;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int m = m0 + wm + 16 * j + r16;
                if (m < a.M && n < a.N)
                    stc4<float>(part + (size_t)m * a.N + n, make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]),
                                a.N - n, a.vec);
            }
        }
        if (sums) {   // the eight threads of a column in order (AT: 32 threads a row)
            lds_barrier();
            reinterpret_cast<float4*>(lds)[threadIdx.x] = sum;
            lds_barrier();
            if (threadIdx.x < 128 && m0 + (int)threadIdx.x < a.M) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) s += reinterpret_cast<const float*>(lds)[128 * i + threadIdx.x];
                a.bpart[(size_t)split * a.M + m0 + threadIdx.x] = s;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = n0 + wn + 16 * i + 4 * g4;
            const float4 bias = bias4<float, DG>(a, n);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int m = m0 + wm + 16 * j + r16;
                if (m < a.M && n < a.N) finish4<float, ACT, DG, true>(a, m, n, acc[i][j], bias);
            }
        }
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

// eight (bf16) or four (fp32) elements k.. of a row; past K zero
__device__ __forceinline__ bf16x8 row8(const uint16_t* row, int k, int K, bool vec) {
    if (vec && k + 8 <= K) return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(row + k));
    short8v v = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (k + e < K) v[e] = (short)row[k + e];
    return __builtin_bit_cast(bf16x8, v);
}

constexpr int FEW_WAVES = 8;

// 16 rows x 16 columns a workgroup; wave w takes steps w, w + 8, ... of the
// contracted index (32 of bf16, 16 of fp32) and the partial tiles meet in LDS
template <typename T, int ACT>
__global__ __launch_bounds__(64 * FEW_WAVES) void kda_linear_few_kernel(const GemmArgs a) {
    __shared__ f32x4 part[FEW_WAVES][64];
    const int w = threadIdx.x >> 6, l = lane_id(), r16 = l & 15, g4 = l >> 4;
    const int m0 = 16 * ((int)blockIdx.x / a.nt), n0 = 16 * ((int)blockIdx.x % a.nt);
    const T* ra = static_cast<const T*>(a.a) + (size_t)min(m0 + r16, a.M - 1) * a.lda;
    const T* rb = static_cast<const T*>(a.b) + (size_t)min(n0 + r16, a.N - 1) * a.ldb;
    f32x4 acc = zero4();
    if constexpr (std::is_same<T, float>::value) {
        for (int k = 16 * w; k < a.K; k += 16 * FEW_WAVES) {
            const int kk = k + 4 * g4;
            const float4 x = ldc4<float>(ra + kk, a.K - kk, a.vec_a && kk + 4 <= a.K);
            const float4 y = ldc4<float>(rb + kk, a.K - kk, a.vec_b && kk + 4 <= a.K);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(y.x, x.x, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(y.y, x.y, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(y.z, x.z, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(y.w, x.w, acc, 0, 0, 0);
        }
    } else {
#pragma unroll 4
        for (int k = 32 * w; k < a.K; k += 32 * FEW_WAVES) {
            const bf16x8 x = row8(ra, k + 8 * g4, a.K, a.vec_a), y = row8(rb, k + 8 * g4, a.K, a.vec_b);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y, x, acc, 0, 0, 0);
        }
    }
    part[w][l] = acc;
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (int i = 1; i < FEW_WAVES; ++i) acc += part[i][l];
    const int m = m0 + r16, n = n0 + 4 * g4;
    if (m < a.M && n < a.N)
        finish4<T, ACT, false, std::is_same<T, float>::value>(a, m, n, acc, bias4<T, false>(a, n));
}

// dz = dy act'(z)
template <typename T, int ACT>
__global__ __launch_bounds__(256) void kda_linear_act_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ z,
                                                                 T* __restrict__ dz, int64_t ld_dy, int64_t ld_z,
                                                                 int64_t ld_dz, int M, int N, int vec) {
    constexpr bool EXACT = std::is_same<T, float>::value;
    const int groups = (N + 3) / 4;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < (size_t)M * groups; i += (size_t)gridDim.x * 256) {
        const int m = (int)(i / groups), n = 4 * (int)(i - (size_t)m * groups), left = N - n;
        const float4 g = ldc4<T>(dy + (size_t)m * ld_dy + n, left, vec), x = ldc4<T>(z + (size_t)m * ld_z + n, left, vec);
        stc4<T>(dz + (size_t)m * ld_dz + n,
                make_float4(g.x * act_grad<ACT, EXACT>(x.x), g.y * act_grad<ACT, EXACT>(x.y),
                            g.z * act_grad<ACT, EXACT>(x.z), g.w * act_grad<ACT, EXACT>(x.w)),
                left, vec);
    }
}

// ----------------------------------------------------------------------------
// launches
// ----------------------------------------------------------------------------
bool groups_ok(const void* p, int64_t ld, int es) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % (4 * es) == 0 && ld % 4 == 0);
}

template <bool BT, int ACT, bool DG>
hipError_t launch_bf16(GemmArgs& a, hipStream_t st) {
    constexpr int BM = 128, BN = 128, BK = 32, NST = 4, WR = 2, WC = 2;
    constexpr size_t LDS = (size_t)NST * (BM + BN) * 2 * BK;
    a.mt = (a.M + BM - 1) / BM;
    a.nt = (a.N + BN - 1) / BN;
    hipLaunchKernelGGL((kda_linear_bf16_kernel<BM, BN, BK, NST, WR, WC, BT, ACT, DG>), dim3((unsigned)a.mt * a.nt),
                       dim3(64 * WR * WC), LDS, st, a);
    return hipGetLastError();
}

template <int ACT>
hipError_t launch_fwd(GemmArgs& a, int bf16, hipStream_t st) {
    if (a.M <= 64) {
        a.nt = (a.N + 15) / 16;
        a.mt = (a.M + 15) / 16;
        const dim3 grid((unsigned)a.mt * a.nt), block(64 * FEW_WAVES);
        if (bf16) hipLaunchKernelGGL((kda_linear_few_kernel<uint16_t, ACT>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((kda_linear_few_kernel<float, ACT>), grid, block, 0, st, a);
        return hipGetLastError();
    }
    if (bf16) return launch_bf16<false, ACT, false>(a, st);
    a.mt = (a.M + 127) / 128;
    a.nt = (a.N + 127) / 128;
    hipLaunchKernelGGL((kda_linear_f32_kernel<false, false, ACT, false, false>), dim3((unsigned)a.mt * a.nt), dim3(256), 0,
                       st, a);
    return hipGetLastError();
}

template <int ACT>
hipError_t launch_dgrad(GemmArgs& a, int bf16, hipStream_t st) {
    if (bf16) return launch_bf16<true, ACT, true>(a, st);
    a.mt = (a.M + 127) / 128;
    a.nt = (a.N + 127) / 128;
    hipLaunchKernelGGL((kda_linear_f32_kernel<false, true, ACT, true, false>), dim3((unsigned)a.mt * a.nt), dim3(256), 0,
                       st, a);
    return hipGetLastError();
}

template <typename T>
hipError_t launch_act_bwd(const void* dy, const void* z, void* dz, int64_t ld_dy, int64_t ld_z, int64_t ld_dz, int M, int N,
                          int act, int vec, hipStream_t st) {
    const size_t n = (size_t)M * ((N + 3) / 4);
    const dim3 grid((unsigned)std::min<size_t>((n + 255) / 256, 4096)), block(256);
    const T *pdy = static_cast<const T*>(dy), *pz = static_cast<const T*>(z);
    if (act == 1)
        hipLaunchKernelGGL((kda_linear_act_bwd_kernel<T, 1>), grid, block, 0, st, pdy, pz, static_cast<T*>(dz), ld_dy, ld_z,
                           ld_dz, M, N, vec);
    else
        hipLaunchKernelGGL((kda_linear_act_bwd_kernel<T, 2>), grid, block, 0, st, pdy, pz, static_cast<T*>(dz), ld_dy, ld_z,
                           ld_dz, M, N, vec);
    return hipGetLastError();
}

// Parts of the m rows that wgrad's sum is split into: two workgroups on each
// of 256 CUs, at least 8 steps each
void wgrad_plan(int M, int N, int K, int* splits, int* per) {
    const int tiles = ((N + 127) / 128) * ((K + 127) / 128), steps = (M + 31) / 32;
    const int s = std::max(1, std::min(512 / std::max(tiles, 1), steps / 8));
    *per = (steps + s - 1) / s * 32;
    *splits = (M + *per - 1) / *per;
}

int check_map(int M, int N, int K, int act, int dtype) {
    if (dtype != KDA_DTYPE_F32 && dtype != KDA_DTYPE_BF16)
        return api_fail(KDA_E_UNSUPPORTED, "dtype=%d: expected 0 (fp32) or 1 (bf16)", dtype);
    if (act < KDA_ACT_NONE || act > KDA_ACT_SILU)
        return api_fail(KDA_E_UNSUPPORTED, "act=%d: expected 0 (none), 1 (gelu) or 2 (silu)", act);
    if (M < 0 || N < 1 || K < 1 || N > (1 << 20) || K > (1 << 20))
        return api_fail(KDA_E_INVALID, "M=%d N=%d K=%d: expected M >= 0, N and K from 1 to 2^20", M, N, K);
    // tiles of 128 x 128 by 256 threads: below 2^32 threads
    if (((int64_t)M + 127) / 128 * ((std::max(N, K) + 127) / 128) > (1 << 23))
        return api_fail(KDA_E_UNSUPPORTED, "M=%d N=%d K=%d: more than 2^23 tiles of 128 x 128", M, N, K);
    return KDA_OK;
}

// a matrix's pointer and row stride; dma: rows are read 16 bytes at a time
int check_rows(const void* p, const char* name, int64_t ld, int cols, int dtype, bool dma) {
    const int es = dtype == KDA_DTYPE_BF16 ? 2 : 4;
    if (!p) return api_fail(KDA_E_INVALID, "%s is NULL", name);
    if (reinterpret_cast<uintptr_t>(p) % (dma ? 16 : es) != 0)
        return api_fail(KDA_E_INVALID, "%s is not %d-byte aligned", name, dma ? 16 : es);
    if (ld < (dma ? (cols + 7) & ~7 : cols) || ld > (1 << 21) || (dma && ld % 8 != 0))
        return api_fail(KDA_E_INVALID, "%s: row stride %lld for %d columns", name, (long long)ld, cols);
    return KDA_OK;
}
int check_opt(const void* p, const char* name, int64_t ld, int cols, int dtype) {
    return p ? check_rows(p, name, ld, cols, dtype, false) : KDA_OK;
}

#define LIN_TRY(x)                       \
    do {                                 \
        const int rc_ = (x);             \
        if (rc_ != KDA_OK) return rc_;   \
    } while (0)

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
    const bool dma = dtype == KDA_DTYPE_BF16 && M > 64;
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
    a.vec = N % 4 == 0 && groups_ok(y, ld_y, es) && groups_ok(bias, 0, es) && groups_ok(residual, ld_r, es) && groups_ok(z, ld_z, es);
    const int row = es == 2 ? 8 : 4;   // elements of a 16-byte read
    a.vec_a = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld_x % row == 0;
    a.vec_b = reinterpret_cast<uintptr_t>(w) % 16 == 0 && ld_w % row == 0;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const hipError_t e = act == 1   ? launch_fwd<1>(a, es == 2, st)
                         : act == 2 ? launch_fwd<2>(a, es == 2, st)
                                    : launch_fwd<0>(a, es == 2, st);
    return e == hipSuccess ? KDA_OK : api_hip_fail(e, "kda_linear_fwd");
}

int kda_linear_dgrad(const void* dz, int64_t ld_dz, const void* w, int64_t ld_w, const void* z, int64_t ld_z, void* dx,
                     int64_t ld_dx, int M, int N, int K, int act, int dtype, void* stream) {
    LIN_TRY(check_map(M, N, K, act, dtype));
    if (M == 0) return KDA_OK;
    const int es = dtype == KDA_DTYPE_BF16 ? 2 : 4;
    const bool dma = dtype == KDA_DTYPE_BF16;
    LIN_TRY(check_rows(dz, "dz", ld_dz, N, dtype, dma));
    LIN_TRY(check_rows(w, "w", ld_w, K, dtype, dma));
    LIN_TRY(check_rows(dx, "dx", ld_dx, K, dtype, false));
    if (act != KDA_ACT_NONE) LIN_TRY(check_rows(z, "z", ld_z, K, dtype, false));
    GemmArgs a = {};   // C[m][k] = sum_n A[m][n] B[n][k]
    a.a = dz; a.b = w; a.c = dx; a.zin = act != KDA_ACT_NONE ? z : nullptr;
    a.lda = ld_dz; a.ldb = ld_w; a.ldc = ld_dx; a.ldzi = ld_z;
    a.M = M; a.N = K; a.K = N;
    a.vec = K % 4 == 0 && groups_ok(dx, ld_dx, es) && groups_ok(a.zin, ld_z, es);
    a.vec_a = reinterpret_cast<uintptr_t>(dz) % 16 == 0 && ld_dz % 4 == 0;
    a.vec_b = reinterpret_cast<uintptr_t>(w) % 16 == 0 && ld_w % 4 == 0;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const hipError_t e = act == 1   ? launch_dgrad<1>(a, es == 2, st)
                         : act == 2 ? launch_dgrad<2>(a, es == 2, st)
                                    : launch_dgrad<0>(a, es == 2, st);
    return e == hipSuccess ? KDA_OK : api_hip_fail(e, "kda_linear_dgrad");
}

size_t kda_linear_wgrad_workspace_size(int M, int N, int K) {
    if (M < 1 || N < 1 || K < 1 || N > (1 << 20) || K > (1 << 20)) return 0;
    int splits, per;
    wgrad_plan(M, N, K, &splits, &per);
    return ((size_t)splits * N * K + (size_t)splits * N) * sizeof(float);
}

int kda_linear_wgrad(const float* dz, int64_t ld_dz, const float* x, int64_t ld_x, float* dw, float* db, int M, int N, int K,
                     void* workspace, size_t ws_bytes, void* stream) {
    LIN_TRY(check_map(M, N, K, KDA_ACT_NONE, KDA_DTYPE_F32));
    if (M < 1) return api_fail(KDA_E_INVALID, "M=%d: expected at least one row", M);
    LIN_TRY(check_rows(dz, "dz", ld_dz, N, KDA_DTYPE_F32, false));
    LIN_TRY(check_rows(x, "x", ld_x, K, KDA_DTYPE_F32, false));
    LIN_TRY(check_rows(dw, "dw", K, K, KDA_DTYPE_F32, false));
    const size_t need = kda_linear_wgrad_workspace_size(M, N, K);
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return api_fail(KDA_E_INVALID, "workspace is NULL or not 16-byte aligned");
    if (ws_bytes < need) return api_fail(KDA_E_WORKSPACE, "workspace has %zu bytes, needs %zu", ws_bytes, need);
    GemmArgs a = {};   // C[n][k] = sum_m A[m][n] B[m][k]
    a.a = dz; a.b = x;
    a.lda = ld_dz; a.ldb = ld_x;
    a.M = N; a.N = K; a.K = M;
    a.mt = (N + 127) / 128;
    a.nt = (K + 127) / 128;
    wgrad_plan(M, N, K, &a.splits, &a.k_per);
    a.part = static_cast<float*>(workspace);
    float* bpart = a.part + (size_t)a.splits * N * K;
    a.bpart = db ? bpart : nullptr;
    a.vec = K % 4 == 0;
    a.vec_a = reinterpret_cast<uintptr_t>(dz) % 16 == 0 && ld_dz % 4 == 0;
    a.vec_b = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld_x % 4 == 0;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL((kda_linear_f32_kernel<true, true, 0, false, true>), dim3((unsigned)(a.mt * a.nt * a.splits)),
                       dim3(256), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return api_hip_fail(e, "kda_linear_wgrad");
    const size_t total = (size_t)N * K + N;
    hipLaunchKernelGGL(kda_linear_sum_parts_kernel, dim3((unsigned)std::min<size_t>((total + 255) / 256, 4096)), dim3(256), 0,
                       st, a.part, bpart, dw, db, (size_t)N * K, N, a.splits);
    e = hipGetLastError();
    return e == hipSuccess ? KDA_OK : api_hip_fail(e, "kda_linear_wgrad");
}

int kda_linear_act_bwd(const void* dy, int64_t ld_dy, const void* z, int64_t ld_z, void* dz, int64_t ld_dz, int M, int N,
                       int act, int dtype, void* stream) {
    LIN_TRY(check_map(M, N, 1, act, dtype));
    if (act == KDA_ACT_NONE) return api_fail(KDA_E_UNSUPPORTED, "act=0 has no gradient kernel");
    if (M == 0) return KDA_OK;
    LIN_TRY(check_rows(dy, "dy", ld_dy, N, dtype, false));
    LIN_TRY(check_rows(z, "z", ld_z, N, dtype, false));
    LIN_TRY(check_rows(dz, "dz", ld_dz, N, dtype, false));
    const int es = dtype == KDA_DTYPE_BF16 ? 2 : 4;
    const int vec = N % 4 == 0 && groups_ok(dy, ld_dy, es) && groups_ok(z, ld_z, es) && groups_ok(dz, ld_dz, es);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const hipError_t e = es == 2 ? launch_act_bwd<uint16_t>(dy, z, dz, ld_dy, ld_z, ld_dz, M, N, act, vec, st)
                                 : launch_act_bwd<float>(dy, z, dz, ld_dy, ld_z, ld_dz, M, N, act, vec, st);
    return e == hipSuccess ? KDA_OK : api_hip_fail(e, "kda_linear_act_bwd");
}

}  // extern "C"
