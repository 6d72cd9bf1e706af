// AdamW over many tensors in one launch, with states in 32 or in 8 bits.
//
// m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// States in 8 bits: every 256 consecutive values share a scale, m = code * sm and sqrt(v) = code * sv with e4m3 codes and
// s = largest / 448.  The root is what is stored because it is what the step divides by, and it halves the range that the code has to
// hold.  A root that is not zero never gets the code 0: a later step with a small gradient would divide m by eps alone.  The step itself
// uses m and v before they are rounded.
// Bound by memory: p, g, m, v in, p, m, v out -- 28 bytes a value in full precision, 16 (and two scales in 256 values) with 16-bit weights, a
// full-precision copy of them and states in 8 bits.  21 M fp32 values in 168 tensors 94 us (6.4 TB/s), 85 M with 16-bit weights and 8-bit states
// 233 us (5.9 TB/s), 0.9 M in 28 tensors 8 us.
#include <cuda_fp8.h>
#include <algorithm>
#include "common.cuh"

namespace vig {

constexpr int AW_BLOCK = 256;        // values that share a scale
constexpr int AW_CHUNK = 2048;       // values of a CTA
constexpr int AW_THREADS = 256;
constexpr int AW_MAX = 400;          // tensors of a launch: the table travels in the launch's parameters (at most 32764 bytes) ...
constexpr int AW_FEW = 48;           // ... and a short one in fewer of them

struct AdamTensor {
    void* p;
    const void* g;
    void *m, *v;
    float *master, *ms, *vs;         // ms, vs: scales of 8-bit states, or NULL
    int64_t n;
    uint8_t pt, gt;                  // dtype codes
    uint8_t whole;                   // everything begins on four values
};

struct AdamScalars {
    float keep, b1, c1, b2, c2, rate, root, eps;      // 1 - lr wd, b1, 1 - b1, b2, 1 - b2, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), eps
    const float *grad_scale, *found_inf;
};
template <int MAX> struct AdamTable : AdamScalars {
    int count;
    uint32_t first[MAX];             // the tensors' first chunks, close together: every CTA searches them
    AdamTensor t[MAX];
};
static_assert(sizeof(AdamTable<AW_MAX>) <= 32764, "the parameters of a launch");

__device__ __forceinline__ float load_as(const void* p, int64_t i, int dtype) {
    return dtype == VIG_DTYPE_F32 ? ((const float*)p)[i] : dtype == VIG_DTYPE_BF16 ? __bfloat162float(((const __nv_bfloat16*)p)[i]) : __half2float(((const __half*)p)[i]);
}
__device__ __forceinline__ void store_as(void* p, int64_t i, int dtype, float x) {
    if (dtype == VIG_DTYPE_F32) ((float*)p)[i] = x;
    else if (dtype == VIG_DTYPE_BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(x);
    else ((__half*)p)[i] = __float2half_rn(x);
}

__device__ __forceinline__ float from_e4m3(uint8_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }
__device__ __forceinline__ uint8_t to_e4m3(float x) { return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }

// One value, in two steps: states from the gradient, then the weight; the second returns the root of the new v.  Written so that every path rounds alike.
__device__ __forceinline__ void adam_moments(const AdamScalars& tab, float g, float& m, float& v) {
    m = fmaf(tab.b1, m, __fmul_rn(tab.c1, g));
    v = fmaf(tab.b2, v, __fmul_rn(tab.c2, __fmul_rn(g, g)));
}
// Root and quotient of the MUFU unit, each right to 2^-23 or so of itself: the step is off by that much of itself, the weight by far less.
// The exact forms cost four times the instructions and bound the 8-bit states: 85 M values 270 us with them.  The unit takes a v below the
// smallest normal number for 0, but without eps, or with one as small, m is divided by its root alone: SMALL takes such a v times 2^64.
constexpr float SMALLEST = 1.17549435e-38f;
template <bool SMALL> __device__ __forceinline__ float adam_weight(const AdamScalars& tab, float m, float v, float& p) {
    const bool small = SMALL && v < SMALLEST;
    float root;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"(small ? v * 0x1p64f : v));
    if (small) root *= 0x1p-32f;
    p = fmaf(p, tab.keep, -__fdividef(__fmul_rn(tab.rate, m), fmaf(root, tab.root, tab.eps)));
    return root;
}
// scale of a block from its largest magnitude, and what its values are multiplied by; a scale without a reciprocal makes all codes 0
__device__ __forceinline__ float adam_scale(uint32_t top, float* inv) {
    const float s = __uint_as_float(__reduce_max_sync(0xffffffffu, top)) * (1.f / 448.f);
    *inv = s >= 1.17549435e-38f ? 1.f / s : s - s;
    return s;
}
__device__ __forceinline__ uint32_t bits_of(float x) { return __float_as_uint(x) & 0x7fffffffu; }      // magnitudes order like these, and a NaN comes out on top

// four values of T as one load, and one store
template <typename T> struct Four;
template <> struct Four<float> {
    float4 r;
    __device__ void load(const void* p, int64_t i) { r = *(const float4*)((const float*)p + i); }
    __device__ void get(float* f) const { f[0] = r.x; f[1] = r.y; f[2] = r.z; f[3] = r.w; }
    static __device__ void store(void* p, int64_t i, const float* f) { *(float4*)((float*)p + i) = make_float4(f[0], f[1], f[2], f[3]); }
};
template <typename T> struct Four {
    uint2 r;
    __device__ void load(const void* p, int64_t i) { r = *(const uint2*)((const T*)p + i); }
    __device__ void get(float* f) const {
        const T* e = (const T*)&r;
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = DType<T>::to_f(e[k]);
    }
    static __device__ void store(void* p, int64_t i, const float* f) {
        uint2 r;
        T* e = (T*)&r;
#pragma unroll
        for (int k = 0; k < 4; ++k) e[k] = DType<T>::from_f(f[k]);
        *(uint2*)((T*)p + i) = r;
    }
};
__device__ __forceinline__ void codes_get(uint32_t c, float* f) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float2 v = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> (16 * k)), __NV_E4M3)));
        f[2 * k] = v.x; f[2 * k + 1] = v.y;
    }
}
template <bool ROOT> __device__ __forceinline__ uint32_t codes_put(const float* f, float by) {
    uint32_t c = 0;
    float t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        t[k] = f[k] * by;
        if (ROOT && f[k] > 0.f) t[k] = fmaxf(t[k], 0x1p-9f);           // the smallest code that is not 0
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) c |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(t[2 * k], t[2 * k + 1]), __NV_SATFINITE, __NV_E4M3) << (16 * k);
    return c;
}

// A whole block of 256 values that begin on four: a lane takes two groups of four, and every load of the block is under way before the
// first is used.
template <typename P, typename G, bool EIGHT>
__device__ __forceinline__ void adam_whole(const AdamScalars& tab, const AdamTensor& t, int64_t block, float gs) {
    const int lane = threadIdx.x & 31;
    const int64_t at = block * AW_BLOCK + 4 * lane;
    Four<P> pr[2];
    Four<G> gr[2];
    Four<float> wr[2], mr[2], vr[2];
    uint32_t mc[2], vc[2];
    float sm = 1.f, sv = 1.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t i = at + 128 * j;
        gr[j].load(t.g, i);
        if (EIGHT) {
            mc[j] = *(const uint32_t*)((const uint8_t*)t.m + i);
            vc[j] = *(const uint32_t*)((const uint8_t*)t.v + i);
        } else {
            mr[j].load(t.m, i);
            vr[j].load(t.v, i);
        }
        if (t.master) wr[j].load(t.master, i); else pr[j].load(t.p, i);
    }
    if (EIGHT) { sm = t.ms[block]; sv = t.vs[block]; }
    float m[2][4], v[2][4];
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t i = at + 128 * j;
        float g[4], w[4];
        gr[j].get(g);
        if (t.master) wr[j].get(w); else pr[j].get(w);
        if (EIGHT) { codes_get(mc[j], m[j]); codes_get(vc[j], v[j]); } else { mr[j].get(m[j]); vr[j].get(v[j]); }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (EIGHT) {
                m[j][k] = __fmul_rn(m[j][k], sm);
                const float root = __fmul_rn(v[j][k], sv);
                v[j][k] = __fmul_rn(root, root);
            }
            adam_moments(tab, __fmul_rn(g[k], gs), m[j][k], v[j][k]);
        }
        // one branch for four values: 85 M values with 8-bit states 233 us; 254 with a select in each, 225 without either
        float root[4];
        if (fminf(fminf(v[j][0], v[j][1]), fminf(v[j][2], v[j][3])) < SMALLEST) {
#pragma unroll
            for (int k = 0; k < 4; ++k) root[k] = adam_weight<true>(tab, m[j][k], v[j][k], w[k]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) root[k] = adam_weight<false>(tab, m[j][k], v[j][k], w[k]);
        }
        if (EIGHT) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[j][k] = root[k];
                top_m = max(top_m, bits_of(m[j][k]));
                top_v = max(top_v, bits_of(root[k]));
            }
        }
        if (t.master) Four<float>::store(t.master, i, w);
        Four<P>::store(t.p, i, w);
        if (!EIGHT) { Four<float>::store(t.m, i, m[j]); Four<float>::store(t.v, i, v[j]); }
    }
    if (EIGHT) {
        float im, iv;
        const float nm = adam_scale(top_m, &im), nv = adam_scale(top_v, &iv);
        if (lane == 0) { t.ms[block] = nm; t.vs[block] = nv; }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            *(uint32_t*)((uint8_t*)t.m + at + 128 * j) = codes_put<false>(m[j], im);
            *(uint32_t*)((uint8_t*)t.v + at + 128 * j) = codes_put<true>(v[j], iv);
        }
    }
}

// Any block: the last of a tensor, one that begins anywhere, or fp32 weights with 16-bit gradients; a value at a time (21 M fp32 values 291 us, 91 as whole
// blocks).
__device__ __noinline__ void adam_any(const AdamScalars& tab, const AdamTensor& t, int64_t block, float gs) {
    const int lane = threadIdx.x & 31;
    const int64_t at = block * AW_BLOCK;
    const bool eight = t.ms != nullptr;
    const float sm = eight ? t.ms[block] : 1.f, sv = eight ? t.vs[block] : 1.f;
    float m[8], v[8];
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t i = at + lane + 32 * j;
        m[j] = v[j] = 0.f;
        if (i < t.n) {
            if (eight) {
                m[j] = __fmul_rn(from_e4m3(((const uint8_t*)t.m)[i]), sm);
                const float root = __fmul_rn(from_e4m3(((const uint8_t*)t.v)[i]), sv);
                v[j] = __fmul_rn(root, root);
            } else {
                m[j] = ((const float*)t.m)[i];
                v[j] = ((const float*)t.v)[i];
            }
            float p = t.master ? t.master[i] : load_as(t.p, i, t.pt);
            adam_moments(tab, __fmul_rn(load_as(t.g, i, t.gt), gs), m[j], v[j]);
            const float root = adam_weight<true>(tab, m[j], v[j], p);
            if (t.master) t.master[i] = p;
            store_as(t.p, i, t.pt, p);
            if (eight) {
                v[j] = root;
                top_m = max(top_m, bits_of(m[j]));
                top_v = max(top_v, bits_of(root));
            } else {
                ((float*)t.m)[i] = m[j];
                ((float*)t.v)[i] = v[j];
            }
        }
    }
    if (!eight) return;
    float im, iv;
    const float nm = adam_scale(top_m, &im), nv = adam_scale(top_v, &iv);
    if (lane == 0) { t.ms[block] = nm; t.vs[block] = nv; }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t i = at + lane + 32 * j;
        if (i < t.n) {
            ((uint8_t*)t.m)[i] = to_e4m3(m[j] * im);
            ((uint8_t*)t.v)[i] = to_e4m3(v[j] > 0.f ? fmaxf(v[j] * iv, 0x1p-9f) : v[j] * iv);
        }
    }
}

// A warp takes a block of 256 values, a CTA eight of them.
template <int MAX>
__global__ void __launch_bounds__(AW_THREADS, 4) adamw_kernel(const __grid_constant__ AdamTable<MAX> tab) {
    if (tab.found_inf && *tab.found_inf != 0.f) return;
    int lo = 0, hi = tab.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.first[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const AdamTensor& t = tab.t[lo];
    const float gs = tab.grad_scale ? *tab.grad_scale : 1.f;
    const int64_t block = (int64_t)(blockIdx.x - tab.first[lo]) * (AW_CHUNK / AW_BLOCK) + (threadIdx.x >> 5);
    if (block * AW_BLOCK >= t.n) return;
    if (!t.whole || (block + 1) * AW_BLOCK > t.n || (t.gt != t.pt && t.gt != VIG_DTYPE_F32)) {
        adam_any(tab, t, block, gs);
        return;
    }
#define VIG_AW(P, G) do { if (t.ms) adam_whole<P, G, true>(tab, t, block, gs); else adam_whole<P, G, false>(tab, t, block, gs); } while (0)
    if (t.pt == VIG_DTYPE_F32) VIG_AW(float, float);
    else if (t.pt == VIG_DTYPE_BF16) { if (t.gt == VIG_DTYPE_BF16) VIG_AW(__nv_bfloat16, __nv_bfloat16); else VIG_AW(__nv_bfloat16, float); }
    else { if (t.gt == VIG_DTYPE_F16) VIG_AW(__half, __half); else VIG_AW(__half, float); }
#undef VIG_AW
}

}  // namespace vig

using namespace vig;

extern "C" int vig_adamw_step(int count, void* const* params, const void* const* grads, void* const* exp_avgs, void* const* exp_avg_sqs,
                              float* const* masters, float* const* exp_avg_scales, float* const* exp_avg_sq_scales, const int64_t* numels,
                              const int* param_dtypes, const int* grad_dtypes, int64_t step, double lr, double beta1, double beta2, double eps,
                              double weight_decay, const float* grad_scale, const float* found_inf, void* stream) {
    if (count < 0 || step < 1 || !(lr >= 0.) || !(beta1 >= 0. && beta1 < 1.) || !(beta2 >= 0. && beta2 < 1.) || !(eps >= 0.) || !(weight_decay >= 0.)) return VIG_ERR_ARG;
    if (!count) return VIG_OK;
    if (!params || !grads || !exp_avgs || !exp_avg_sqs || !numels || !param_dtypes || !grad_dtypes) return VIG_ERR_NULL;
    for (int i = 0; i < count; ++i) {
        if (numels[i] < 0) return VIG_ERR_SHAPE;
        if (numels[i] && (!params[i] || !grads[i] || !exp_avgs[i] || !exp_avg_sqs[i])) return VIG_ERR_NULL;
        if (param_dtypes[i] < 0 || param_dtypes[i] > 2 || grad_dtypes[i] < 0 || grad_dtypes[i] > 2) return VIG_ERR_DTYPE;
        if ((exp_avg_scales && exp_avg_scales[i]) != (exp_avg_sq_scales && exp_avg_sq_scales[i])) return VIG_ERR_NULL;
    }
    AdamTable<AW_MAX> tab;
    tab.keep = (float)(1. - lr * weight_decay);
    tab.b1 = (float)beta1; tab.c1 = (float)(1. - beta1); tab.b2 = (float)beta2; tab.c2 = (float)(1. - beta2);
    tab.rate = (float)(lr / (1. - pow(beta1, (double)step)));
    tab.root = (float)(1. / sqrt(1. - pow(beta2, (double)step)));
    tab.eps = (float)eps;
    tab.grad_scale = grad_scale; tab.found_inf = found_inf;
    for (int i = 0; i < count;) {
        int64_t chunks = 0;
        tab.count = 0;
        for (; i < count && tab.count < AW_MAX; ++i) {
            const int64_t more = (numels[i] + AW_CHUNK - 1) / AW_CHUNK;
            if (!more) continue;
            if (more > 0x7fffffff) return VIG_ERR_SHAPE;
            if (chunks + more > 0x7fffffff) break;
            tab.first[tab.count] = (uint32_t)chunks;
            tab.t[tab.count++] = {params[i], grads[i], exp_avgs[i], exp_avg_sqs[i], masters ? masters[i] : nullptr, exp_avg_scales ? exp_avg_scales[i] : nullptr,
                                  exp_avg_sq_scales ? exp_avg_sq_scales[i] : nullptr, numels[i], (uint8_t)param_dtypes[i], (uint8_t)grad_dtypes[i], 0};
            AdamTensor& t = tab.t[tab.count - 1];
            auto on = [](const void* q, int size) { return (uintptr_t)q % (4 * size) == 0; };
            auto size = [](int dtype) { return dtype == VIG_DTYPE_F32 ? 4 : 2; };
            t.whole = on(t.p, size(t.pt)) && on(t.g, size(t.gt)) && on(t.m, t.ms ? 1 : 4) && on(t.v, t.ms ? 1 : 4) && on(t.master, 4);
            chunks += more;
        }
        if (!tab.count) break;
        if (tab.count <= AW_FEW) {
            AdamTable<AW_FEW> few;
            static_cast<AdamScalars&>(few) = tab;
            few.count = tab.count;
            std::copy(tab.first, tab.first + tab.count, few.first);
            std::copy(tab.t, tab.t + tab.count, few.t);
            adamw_kernel<AW_FEW><<<(unsigned)chunks, AW_THREADS, 0, (cudaStream_t)stream>>>(few);
        } else {
            adamw_kernel<AW_MAX><<<(unsigned)chunks, AW_THREADS, 0, (cudaStream_t)stream>>>(tab);
        }
        if (const cudaError_t e = cudaGetLastError()) return (int)e;
    }
    return VIG_OK;
}
