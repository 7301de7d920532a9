// kda_adamw.hip -- the training step's update over all of a model's tensors:
// the gradients' global norm with the clip factor, AdamW with moments in fp32
// or in 8 bits, and the C ABI around them.
//
//   G = sqrt(sum g^2), c = min(max_norm / (G + 1e-6), 1), g' = c g
//   m <- b1 m + (1 - b1) g',  v <- b2 v + (1 - b2) g'^2
//   p <- p (1 - lr wd) - lr c1 m / (sqrt(v) sqrt(c2) + eps)
//
// (the reference's AdamW, train_mlx_k400.py:548-549, without bias correction
// c1 = c2 = 1).  Everything between the loads and the stores is fp32.
//
// The moments of all tensors lie in one buffer each, a tensor's beginning on a
// multiple of 256 elements.  In 8 bits 256 consecutive elements share a scale:
//   m = s (k / 127) |k / 127|, k in [-127, 127], s the block's largest |m|
//   sqrt(v) = s (k / 255)^2,   k in [0, 255],    s the block's largest sqrt(v)
// Both laws spend their codes on small values (v over ten decades); v's holds
// the root that the update divides by, and a v above zero keeps a code above
// zero, so no weight is divided by eps alone.  The update itself uses the new
// moments before they are rounded to codes.
//
// All are one pass over memory.  A copy of 1 GiB moves 5.1 TB/s here, a sum that
// only reads 3.9: 3.1 10^8 bf16 weights with fp32 moments (22 bytes each) take 1264 us
// at 5.4 TB/s, in 8 bits (10 bytes) 595 at 5.2, the norm (2 bytes) 151 at 4.1, reading
// the 8-bit moments into bf16 (6 bytes) 373 at 5.0.
#include <math.h>

#include "kda_hip.h"
#include "kda_internal.h"

namespace kda {

namespace {

constexpr int QB = 256;            // elements that share a scale
// elements of one tensor a workgroup takes (bf16 weights in 16 tensors, a step with
// the norm, us for 2048 | 4096 | 8192: 2^18 elements 7.1 | 8.2 | 10.5, where the host
// takes 20; 2^23 38.3 | 35.4 | 36.1; 2^26 302 | 310 | 316, in 8 bits 156 | 153 | 157)
constexpr int PER_WG = 4096;
// up to so many partial sums of the norm every workgroup of the update adds them
// itself (8 a thread); beyond, a launch between the two does (us, itself | launch:
// 64 sums 8.2 | 9.1, 256 10.1 | 10.9, 2048 35.4 | 36.7, 8192 168 | 154, 16384 388 | 314)
constexpr int SUM_PARTS = 2048;
constexpr int PER_LAUNCH = 480;    // tensors of one launch: their gradients' addresses travel as kernel arguments

// What does not change from step to step lies in device memory, the plan: the
// tensors, then for each workgroup its tensor.  A step's own part, the gradients'
// addresses, fits one launch for most models (as whole descriptors in the
// arguments, 120 tensors a launch, the default classifier's 436 took four
// launches and 6 us more for each).
struct Tensor {
    void* p;
    int64_t n;
    uint32_t blk0;                 // first block of 256 in the moments
    uint32_t wg0;                  // first workgroup
    int64_t bf16;
};
struct Grads {
    const Tensor* tensors;
    const uint32_t* owner;         // [workgroup] its tensor
    int first;                     // tensor of g[0]
    uint32_t wg;                   // workgroup of block 0
    const void* g[PER_LAUNCH];     // null: the tensor is left out
};
struct StepArgs {
    float b1, omb1, b2, omb2, decay, lr, eps, rc2;
    float* clip;                   // the norm and the clip factor, or null
    const double* part;            // non-null: to be formed from these partial sums
    int parts;
    double max_norm;
    void *m, *v;
    float *ms, *vs, *master;
};
static_assert(sizeof(Grads) + sizeof(StepArgs) <= 4096, "kernel arguments");

// eight elements at p, of which `left` exist
template <typename T>
__device__ __forceinline__ void ld8(const T* p, int64_t left, bool vec, float (&x)[8]) {
    if (vec && left >= 8) {
        if constexpr (std::is_same<T, float>::value) {
            const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
            x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else {
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            x[0] = bf_lo(a.x); x[1] = bf_hi(a.x); x[2] = bf_lo(a.y); x[3] = bf_hi(a.y);
            x[4] = bf_lo(a.z); x[5] = bf_hi(a.z); x[6] = bf_lo(a.w); x[7] = bf_hi(a.w);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = e < left ? ld1<T>(p + e) : 0.f;
}
template <typename T>
__device__ __forceinline__ void st8(T* p, int64_t left, bool vec, const float (&x)[8]) {
    if (vec && left >= 8) {
        if constexpr (std::is_same<T, float>::value) {
            *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
            *reinterpret_cast<uint4*>(p) =
                make_uint4(pack2bf(x[0], x[1]), pack2bf(x[2], x[3]), pack2bf(x[4], x[5]), pack2bf(x[6], x[7]));
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < left) st1<T>(p + e, x[e]);
}

// The largest of 32 lanes' values by their bits: of non-negative floats this is
// the largest value, and a NaN, whose bits are larger than infinity's, wins, so
// that a block with one decodes to NaN instead of to something finite.
__device__ __forceinline__ uint32_t max32(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, true));    // quad_perm [1,0,3,2]
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, true));    // quad_perm [2,3,0,1]
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xF, 0xF, true));   // row_half_mirror
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xF, 0xF, true));   // row_mirror
    return max(x, (uint32_t)__builtin_amdgcn_ds_swizzle((int)x, 0x401F));                  // lane ^ 16
}

constexpr uint32_t MIN_NORMAL = 0x00800000u;

// m and v from their codes, each operation rounded as written (a product with the rounded
// reciprocal: a quotient would differ by a step of fp32 at most)
__device__ __forceinline__ void decode8(const uint2& km, const uint2& kv, float sm, float sv, float (&m)[8], float (&v)[8]) {
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float k = (float)(int8_t)((e < 4 ? km.x : km.y) >> (8 * (e & 3))) * (1.f / 127.f);
        const float q = (float)(uint8_t)((e < 4 ? kv.x : kv.y) >> (8 * (e & 3))) * (1.f / 255.f);
        m[e] = sm * k * fabsf(k);
        const float r = sv * q * q;
        v[e] = r * r;
    }
}

// The code of a companded value, x = top sqrt(value / scale): `fast` is x with the
// hardware's square root and reciprocal, within 9e-5 (3.3e-7 of 255); where it lies
// that near a border between two codes, about once in 3000, x is formed with
// correctly rounded operations.  So the codes are those of fp32 arithmetic operation
// by operation, whatever computes them, and two programs that take the same steps
// keep the same moments.
constexpr float BORDER = 0.5f - 1.5e-4f;

template <typename T, bool SMALL, bool MASTER>
__device__ __forceinline__ void update(const StepArgs& a, const Tensor& t, const void* grad, bool vec, float c, int64_t e0) {
#pragma clang fp contract(off)
    const int64_t left = t.n - e0;
    const size_t at = (size_t)t.blk0 * QB + e0;      // in the moments
    T* p = static_cast<T*>(t.p) + e0;
    float g[8], w[8], m[8], v[8];
    ld8<T>(static_cast<const T*>(grad) + e0, left, vec, g);
    if constexpr (MASTER) ld8<float>(a.master + at, 8, true, w);
    else ld8<T>(p, left, vec, w);
    if constexpr (SMALL) {
        decode8(*reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.m) + at),
                *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + at), a.ms[at / QB], a.vs[at / QB], m, v);
    } else {
        ld8<float>(static_cast<const float*>(a.m) + at, 8, true, m);
        ld8<float>(static_cast<const float*>(a.v) + at, 8, true, v);
    }
    uint32_t top_m = 0, top_v = 0;
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] *= c;
    if (left < 8)   // what lies past the tensor stays zero, whatever c is
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e >= left) g[e] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        m[e] = a.b1 * m[e] + a.omb1 * g[e];
        v[e] = a.b2 * v[e] + a.omb2 * g[e] * g[e];
        r[e] = __builtin_amdgcn_sqrtf(v[e]);
        // lr holds the bias correction c1, rc2 is sqrt(c2)
        w[e] = fmaf(w[e], a.decay, -a.lr * m[e] * __builtin_amdgcn_rcpf(fmaf(r[e], a.rc2, a.eps)));
        if constexpr (SMALL) {
            top_m = max(top_m, __float_as_uint(m[e]) & 0x7fffffffu);
            top_v = max(top_v, __float_as_uint(v[e]) & 0x7fffffffu);
        }
    }
    st8<T>(p, left, vec, w);
    if constexpr (MASTER) {
        if (left < 8)   // (with eps 0: there 0 / 0)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e >= left) w[e] = 0.f;
        st8<float>(a.master + at, 8, true, w);
    }
    if constexpr (SMALL) {
        top_m = max32(top_m);
        top_v = max32(top_v);
        // below the smallest normal number a block counts as zero
        const float sm = top_m < MIN_NORMAL ? 0.f : __uint_as_float(top_m);
        const float sv = top_v < MIN_NORMAL ? 0.f : sqrtf(__uint_as_float(top_v));
        const float im = sm == 0.f ? 0.f : __builtin_amdgcn_rcpf(sm), ir = sv == 0.f ? 0.f : __builtin_amdgcn_rcpf(sv);
        uint32_t km[2] = {0u, 0u}, kv[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = 127.f * __builtin_amdgcn_sqrtf(fabsf(m[e]) * im), y = 255.f * __builtin_amdgcn_sqrtf(r[e] * ir);
            float k = rintf(x), q = rintf(y);
            if (fabsf(x - k) > BORDER) k = rintf(127.f * sqrtf(fabsf(m[e]) / sm));
            if (fabsf(y - q) > BORDER) q = rintf(255.f * sqrtf(sqrtf(v[e]) / sv));
            const int ik = (int)copysignf(k, m[e]), iq = v[e] * ir > 0.f ? max((int)q, 1) : 0;
            km[e >> 2] |= (uint32_t)(ik & 255) << (8 * (e & 3));
            kv[e >> 2] |= (uint32_t)iq << (8 * (e & 3));
        }
        *reinterpret_cast<uint2*>(static_cast<int8_t*>(a.m) + at) = make_uint2(km[0], km[1]);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v) + at) = make_uint2(kv[0], kv[1]);
        if ((lane_id() & 31) == 0) {
            a.ms[at / QB] = sm;
            a.vs[at / QB] = sv;
        }
    } else {
        st8<float>(static_cast<float*>(a.m) + at, 8, true, m);
        st8<float>(static_cast<float*>(a.v) + at, 8, true, v);
    }
}

// The clip factor of all partial sums, by TH threads (all of them get it); out
// non-null: out[0] = G, out[1] = the factor (a NaN stays one)
template <int TH>
__device__ __forceinline__ float clip_factor(const double* __restrict__ part, int n, double max_norm, double* lds, float* out) {
    double s = 0.;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += TH) s += part[i];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    if (lane_id() == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    s = lds[0];
#pragma unroll
    for (int i = 1; i < TH / 64; ++i) s += lds[i];
    const double g = sqrt(s), c = max_norm / (g + 1e-6), f = c > 1. ? 1. : c;
    if (out && threadIdx.x == 0) {
        out[0] = (float)g;
        out[1] = (float)f;
    }
    return (float)f;
}

template <bool SMALL, bool MASTER>
__global__ __launch_bounds__(256) void kda_adamw_kernel(const StepArgs a, const Grads q) {
    const uint32_t wg = q.wg + blockIdx.x;
    const int i = (int)q.owner[wg];
    const Tensor t = q.tensors[i];
    const void* g = q.g[i - q.first];
    const bool vec = ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(t.p)) & 15) == 0;
    float c = 1.f;
    if (a.part) {
        __shared__ double lds[4];
        c = clip_factor<256>(a.part, a.parts, a.max_norm, lds, blockIdx.x == 0 && q.wg == 0 ? a.clip : nullptr);
    } else if (a.clip) {
        c = a.clip[1];
    }
    if (!g) return;
    const int64_t b0 = (int64_t)(wg - t.wg0) * PER_WG, end = min((t.n + QB - 1) / QB * QB, b0 + (int64_t)PER_WG);
    for (int64_t e = b0 + 8 * (int64_t)threadIdx.x; e < end; e += 8 * 256) {   // whole blocks: half waves stay together
        if (t.bf16) update<uint16_t, SMALL, MASTER>(a, t, g, vec, c, e);
        else update<float, SMALL, MASTER>(a, t, g, vec, c, e);
    }
}

// The norm's sums are fp64 from the first square on: the clip factor then is the
// exact one rounded, and does not depend on the order (the conversion and the
// addition cost two more operations a value than fp32 sums, in a pass that waits
// for memory; four pieces a workgroup with their loads in flight together measured the
// same: 2^28 elements with the update 1226 us and 1225).
__global__ __launch_bounds__(256) void kda_grad_norm_kernel(double* __restrict__ part, const Grads q) {
    __shared__ double lds[4];
    const uint32_t wg = q.wg + blockIdx.x;
    const int i = (int)q.owner[wg];
    const Tensor t = q.tensors[i];
    const void* g = q.g[i - q.first];
    double s[4] = {0., 0., 0., 0.};
    if (g) {
        const bool vec = (reinterpret_cast<uintptr_t>(g) & 15) == 0;
        const int64_t b0 = (int64_t)(wg - t.wg0) * PER_WG;
#pragma unroll
        for (int u = 0; u < PER_WG / 2048; ++u) {
            const int64_t e = b0 + 2048 * u + 8 * (int64_t)threadIdx.x, left = t.n - e;
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (left > 0) {
                if (t.bf16) ld8<uint16_t>(static_cast<const uint16_t*>(g) + e, left, vec, x);
                else ld8<float>(static_cast<const float*>(g) + e, left, vec, x);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) s[k & 3] = fma((double)x[k], (double)x[k], s[k & 3]);
        }
    }
    double sum = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    if (lane_id() == 0) lds[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) part[wg] = (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

__global__ __launch_bounds__(1024) void kda_grad_norm_finish_kernel(const double* __restrict__ part, int n, double max_norm,
                                                                    float* __restrict__ out) {
    __shared__ double lds[16];
    clip_factor<1024>(part, n, max_norm, lds, out);
}

// what 8-bit moments stand for, eight a thread
template <typename T>
__global__ __launch_bounds__(256) void kda_adamw_moments_kernel(const int8_t* __restrict__ m, const uint8_t* __restrict__ v,
                                                                const float* __restrict__ ms, const float* __restrict__ vs,
                                                                T* __restrict__ mo, T* __restrict__ vo, size_t n) {
    for (size_t at = 8 * ((size_t)blockIdx.x * 256 + threadIdx.x); at < n; at += 8 * 256 * (size_t)gridDim.x) {
        float x[8], y[8];
        decode8(*reinterpret_cast<const uint2*>(m + at), *reinterpret_cast<const uint2*>(v + at), ms[at / QB], vs[at / QB], x, y);
        st8<T>(mo + at, 8, true, x);
        st8<T>(vo + at, 8, true, y);
    }
}

int check_tensors(const kda_adamw_tensor* t, int count) {
    if (count < 0 || (count > 0 && !t)) return api_fail(KDA_E_INVALID, "count=%d tensors at %p", count, (const void*)t);
    int64_t wgs = 0;
    for (int i = 0; i < count; ++i) {
        if (t[i].dtype != KDA_DTYPE_F32 && t[i].dtype != KDA_DTYPE_BF16)
            return api_fail(KDA_E_UNSUPPORTED, "tensor %d: dtype=%lld: expected 0 (fp32) or 1 (bf16)", i, (long long)t[i].dtype);
        if (t[i].n < 0 || t[i].n > ((int64_t)1 << 36)) return api_fail(KDA_E_INVALID, "tensor %d: n=%lld", i, (long long)t[i].n);
        wgs += (t[i].n + PER_WG - 1) / PER_WG;
        if (t[i].n == 0) continue;
        const uintptr_t es = t[i].dtype == KDA_DTYPE_BF16 ? 2 : 4;
        if (reinterpret_cast<uintptr_t>(t[i].g) % es != 0 || !t[i].p || reinterpret_cast<uintptr_t>(t[i].p) % es != 0)
            return api_fail(KDA_E_INVALID, "tensor %d: p is NULL, or p or g is misaligned", i);
        if (t[i].offset < 0 || t[i].offset % QB != 0 || t[i].offset / QB > 0xffffffffLL)
            return api_fail(KDA_E_INVALID, "tensor %d: offset=%lld: expected a multiple of %d", i, (long long)t[i].offset, QB);
    }
    if (wgs > (1 << 23))   // 256 threads each: below 2^32 in a launch
        return api_fail(KDA_E_UNSUPPORTED, "more than 2^23 * %d elements", PER_WG);
    return KDA_OK;
}

uint32_t workgroups(const kda_adamw_tensor* t, int count) {
    uint32_t n = 0;
    for (int i = 0; i < count; ++i) n += (uint32_t)((t[i].n + PER_WG - 1) / PER_WG);
    return n;
}
const uint32_t* owners(const void* plan, int count) {
    return reinterpret_cast<const uint32_t*>(static_cast<const Tensor*>(plan) + count);
}

// launch(grads, workgroups) for each run of PER_LAUNCH tensors
template <typename F>
hipError_t each_launch(const kda_adamw_tensor* t, int count, const void* plan, F&& launch) {
    Grads q;
    q.tensors = static_cast<const Tensor*>(plan);
    q.owner = owners(plan, count);
    q.wg = 0;
    for (q.first = 0; q.first < count; q.first += PER_LAUNCH) {
        const int n = std::min(PER_LAUNCH, count - q.first);
        for (int i = 0; i < n; ++i) q.g[i] = t[q.first + i].g;
        const uint32_t wg = workgroups(t + q.first, n);
        if (wg > 0) {
            launch(q, dim3(wg));
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        q.wg += wg;
    }
    return hipSuccess;
}

}  // namespace

}  // namespace kda

using namespace kda;

extern "C" {

size_t kda_adamw_plan_size(const kda_adamw_tensor* tensors, int count) {
    if (check_tensors(tensors, count) != KDA_OK) return 0;
    return count * sizeof(Tensor) + workgroups(tensors, count) * sizeof(uint32_t);
}

int kda_adamw_plan(const kda_adamw_tensor* tensors, int count, void* host_plan, size_t bytes) {
    const int rc = check_tensors(tensors, count);
    if (rc != KDA_OK) return rc;
    if (count == 0) return KDA_OK;
    if (!host_plan || reinterpret_cast<uintptr_t>(host_plan) % 8 != 0)
        return api_fail(KDA_E_INVALID, "host_plan is NULL or not 8-byte aligned");
    if (bytes < kda_adamw_plan_size(tensors, count))
        return api_fail(KDA_E_WORKSPACE, "the plan has %zu bytes, needs %zu", bytes, kda_adamw_plan_size(tensors, count));
    Tensor* t = static_cast<Tensor*>(host_plan);
    uint32_t* owner = const_cast<uint32_t*>(owners(host_plan, count));
    uint32_t wg = 0;
    for (int i = 0; i < count; ++i) {
        t[i] = Tensor{tensors[i].p, tensors[i].n, (uint32_t)(tensors[i].offset / QB), wg, tensors[i].dtype};
        for (const uint32_t end = wg + workgroups(tensors + i, 1); wg < end; ++wg) owner[wg] = (uint32_t)i;
    }
    return KDA_OK;
}

size_t kda_adamw_step_workspace_size(const kda_adamw_tensor* tensors, int count) {
    if (check_tensors(tensors, count) != KDA_OK) return 0;
    return workgroups(tensors, count) * sizeof(double);
}

int kda_adamw_step(const kda_adamw_tensor* tensors, int count, const void* plan, int states, void* m, void* v,
                   float* m_scale, float* v_scale, float* master, double max_norm, float* clip, double lr, double beta1,
                   double beta2, double eps, double weight_decay, double correct1, double correct2, void* workspace,
                   size_t ws_bytes, void* stream) {
    const int rc = check_tensors(tensors, count);
    if (rc != KDA_OK) return rc;
    if (states != KDA_ADAMW_F32 && states != KDA_ADAMW_INT8)
        return api_fail(KDA_E_UNSUPPORTED, "states=%d: expected 0 (fp32) or 1 (8 bits)", states);
    if (!(beta1 >= 0. && beta1 < 1. && beta2 >= 0. && beta2 < 1. && eps >= 0. && correct1 > 0. && correct2 > 0.))
        return api_fail(KDA_E_INVALID, "beta1=%g beta2=%g eps=%g correct1=%g correct2=%g", beta1, beta2, eps, correct1,
                        correct2);
    if (!(max_norm >= 0.)) return api_fail(KDA_E_INVALID, "max_norm=%g: expected 0 (no clip) or a positive number", max_norm);
    const size_t parts = workgroups(tensors, count);
    if (max_norm > 0.) {
        if (!clip || reinterpret_cast<uintptr_t>(clip) % 4 != 0) return api_fail(KDA_E_INVALID, "clip is NULL or misaligned");
        if (parts > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 8 != 0))
            return api_fail(KDA_E_INVALID, "workspace is NULL or misaligned");
        if (ws_bytes < parts * sizeof(double))
            return api_fail(KDA_E_WORKSPACE, "workspace has %zu bytes, needs %zu", ws_bytes, parts * sizeof(double));
    }
    if (parts > 0 && (!plan || reinterpret_cast<uintptr_t>(plan) % 8 != 0))
        return api_fail(KDA_E_INVALID, "plan is NULL or not 8-byte aligned");
    const bool small = states == KDA_ADAMW_INT8;
    const uintptr_t all = reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(master);
    if (parts > 0 && (!m || !v || all % 16 != 0)) return api_fail(KDA_E_INVALID, "m, v or master is NULL or not 16-byte aligned");
    if (parts > 0 && small &&
        (!m_scale || !v_scale || (reinterpret_cast<uintptr_t>(m_scale) | reinterpret_cast<uintptr_t>(v_scale)) % 4 != 0))
        return api_fail(KDA_E_INVALID, "m_scale or v_scale is NULL or misaligned");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    StepArgs a;
    a.b1 = (float)beta1; a.omb1 = (float)(1. - beta1);
    a.b2 = (float)beta2; a.omb2 = (float)(1. - beta2);
    a.decay = (float)(1. - lr * weight_decay);
    a.lr = (float)(lr * correct1);
    a.eps = (float)eps;
    a.rc2 = (float)sqrt(correct2);
    a.m = m; a.v = v; a.ms = m_scale; a.vs = v_scale; a.master = master;
    a.clip = nullptr; a.part = nullptr; a.parts = 0; a.max_norm = max_norm;
    if (max_norm > 0.) {
        double* part = static_cast<double*>(workspace);
        hipError_t e = each_launch(tensors, count, plan, [&](const Grads& q, dim3 grid) {
            hipLaunchKernelGGL(kda_grad_norm_kernel, grid, dim3(256), 0, st, part, q);
        });
        if (e != hipSuccess) return api_hip_fail(e, "kda_adamw_step");
        a.clip = clip;
        if (parts > 0 && parts <= SUM_PARTS) {
            a.part = part;
            a.parts = (int)parts;
        } else {
            hipLaunchKernelGGL(kda_grad_norm_finish_kernel, dim3(1), dim3(1024), 0, st, part, (int)parts, max_norm, clip);
            e = hipGetLastError();
            if (e != hipSuccess) return api_hip_fail(e, "kda_adamw_step");
        }
    }
    const hipError_t e = each_launch(tensors, count, plan, [&](const Grads& q, dim3 grid) {
        const dim3 block(256);
        if (small && master) hipLaunchKernelGGL((kda_adamw_kernel<true, true>), grid, block, 0, st, a, q);
        else if (small) hipLaunchKernelGGL((kda_adamw_kernel<true, false>), grid, block, 0, st, a, q);
        else if (master) hipLaunchKernelGGL((kda_adamw_kernel<false, true>), grid, block, 0, st, a, q);
        else hipLaunchKernelGGL((kda_adamw_kernel<false, false>), grid, block, 0, st, a, q);
    });
    return e == hipSuccess ? KDA_OK : api_hip_fail(e, "kda_adamw_step");
}

int kda_adamw_moments(const void* m, const void* v, const float* m_scale, const float* v_scale, void* m_out, void* v_out,
                      int64_t n, int dtype, void* stream) {
    if (dtype != KDA_DTYPE_F32 && dtype != KDA_DTYPE_BF16)
        return api_fail(KDA_E_UNSUPPORTED, "dtype=%d: expected 0 (fp32) or 1 (bf16)", dtype);
    if (n < 0 || n % QB != 0) return api_fail(KDA_E_INVALID, "n=%lld: expected a multiple of %d", (long long)n, QB);
    if (n == 0) return KDA_OK;
    const uintptr_t all = reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(m_out) |
                          reinterpret_cast<uintptr_t>(v_out);
    if (!m || !v || !m_out || !v_out || all % 16 != 0)
        return api_fail(KDA_E_INVALID, "m, v, m_out or v_out is NULL or not 16-byte aligned");
    if (!m_scale || !v_scale || (reinterpret_cast<uintptr_t>(m_scale) | reinterpret_cast<uintptr_t>(v_scale)) % 4 != 0)
        return api_fail(KDA_E_INVALID, "m_scale or v_scale is NULL or misaligned");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)std::min<int64_t>((n / 8 + 255) / 256, 8192)), block(256);
    const int8_t* km = static_cast<const int8_t*>(m);
    const uint8_t* kv = static_cast<const uint8_t*>(v);
    if (dtype == KDA_DTYPE_BF16)
        hipLaunchKernelGGL((kda_adamw_moments_kernel<uint16_t>), grid, block, 0, st, km, kv, m_scale, v_scale,
                           static_cast<uint16_t*>(m_out), static_cast<uint16_t*>(v_out), (size_t)n);
    else
        hipLaunchKernelGGL((kda_adamw_moments_kernel<float>), grid, block, 0, st, km, kv, m_scale, v_scale,
                           static_cast<float*>(m_out), static_cast<float*>(v_out), (size_t)n);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? KDA_OK : api_hip_fail(e, "kda_adamw_moments");
}

}  // extern "C"
