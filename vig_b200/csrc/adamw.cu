// AdamW over many tensors in one launch, with states in 32 or in 8 bits.
//
// m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// States in 8 bits: every 256 consecutive values share a scale, m = code * sm and sqrt(v) = code * sv with e4m3 codes and
// s = largest / 448.  The root is what is stored because it is what the step divides by, and it halves the range that the code has to
// hold.  A root that is not zero never gets the code 0: a later step with a small gradient would divide m by eps alone.  The step itself
// uses m and v before they are rounded.
// Bound by memory: p, g, m, v in, p, m, v out -- 28 bytes a value in full precision, 16 (and two scales in 256 values) with 16-bit weights, a
// full-precision copy of them and states in 8 bits.
#include <cuda_fp8.h>
#include "common.cuh"

namespace vig {

constexpr int AW_BLOCK = 256;        // values that share a scale
constexpr int AW_CHUNK = 2048;       // values of a CTA
constexpr int AW_THREADS = 256;
constexpr int AW_MAX = 400;          // tensors of a launch: the table travels in the launch's parameters (at most 32764 bytes)

struct AdamTensor {
    void* p;
    const void* g;
    void *m, *v;
    float *master, *ms, *vs;         // ms, vs: scales of 8-bit states, or NULL
    int64_t n;
    uint32_t first;                  // its first chunk
    uint16_t pt, gt;                 // dtype codes
};

struct AdamTable {
    AdamTensor t[AW_MAX];
    int count;
    float keep, b1, c1, b2, c2, rate, root, eps;      // 1 - lr wd, b1, 1 - b1, b2, 1 - b2, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), eps
    const float *grad_scale, *found_inf;
};
static_assert(sizeof(AdamTable) <= 32764, "the parameters of a launch");

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

// A warp takes blocks of 256 values, 8 of them a lane.
__global__ void __launch_bounds__(AW_THREADS) adamw_kernel(const __grid_constant__ AdamTable tab) {
    if (tab.found_inf && *tab.found_inf != 0.f) return;
    int lo = 0, hi = tab.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.t[mid].first <= blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const AdamTensor& t = tab.t[lo];
    const int lane = threadIdx.x & 31;
    const float gs = tab.grad_scale ? *tab.grad_scale : 1.f;
    const int64_t block = (int64_t)(blockIdx.x - t.first) * (AW_CHUNK / AW_BLOCK) + (threadIdx.x >> 5);
    const int64_t at = block * AW_BLOCK;
    if (at >= t.n) return;
    const float sm = t.ms ? t.ms[block] : 1.f, sv = t.vs ? t.vs[block] : 1.f;
    float m[8], v[8];
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t i = at + lane + 32 * j;
        m[j] = v[j] = 0.f;
        if (i < t.n) {
            const float g = load_as(t.g, i, t.gt) * gs;
            float root = 0.f;
            if (t.ms) {
                m[j] = from_e4m3(((const uint8_t*)t.m)[i]) * sm;
                root = from_e4m3(((const uint8_t*)t.v)[i]) * sv;
                v[j] = root * root;
            } else {
                m[j] = ((const float*)t.m)[i];
                v[j] = ((const float*)t.v)[i];
            }
            m[j] = fmaf(tab.b1, m[j], tab.c1 * g);
            v[j] = fmaf(tab.b2, v[j], tab.c2 * (g * g));
            root = sqrtf(v[j]);
            float p = t.master ? t.master[i] : load_as(t.p, i, t.pt);
            p = fmaf(p, tab.keep, -(tab.rate * m[j] / fmaf(root, tab.root, tab.eps)));
            if (t.master) t.master[i] = p;
            store_as(t.p, i, t.pt, p);
            if (t.ms) {
                v[j] = root;
                top_m = max(top_m, __float_as_uint(fabsf(m[j])));
                top_v = max(top_v, __float_as_uint(root) & 0x7fffffffu);
            } else {
                ((float*)t.m)[i] = m[j];
                ((float*)t.v)[i] = v[j];
            }
        }
    }
    if (!t.ms) return;
    const float nm = __uint_as_float(__reduce_max_sync(0xffffffffu, top_m)) * (1.f / 448.f);
    const float nv = __uint_as_float(__reduce_max_sync(0xffffffffu, top_v)) * (1.f / 448.f);
    const float im = nm >= 1.17549435e-38f ? 1.f / nm : nm - nm, iv = nv >= 1.17549435e-38f ? 1.f / nv : nv - nv;
    if (lane == 0) { t.ms[block] = nm; t.vs[block] = nv; }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int64_t i = at + lane + 32 * j;
        if (i < t.n) {
            ((uint8_t*)t.m)[i] = to_e4m3(m[j] * im);
            uint8_t c = to_e4m3(v[j] * iv);
            if (c == 0 && v[j] > 0.f) c = 1;
            ((uint8_t*)t.v)[i] = c;
        }
    }
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
    AdamTable tab;
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
            tab.t[tab.count++] = {params[i], grads[i], exp_avgs[i], exp_avg_sqs[i], masters ? masters[i] : nullptr, exp_avg_scales ? exp_avg_scales[i] : nullptr,
                                  exp_avg_sq_scales ? exp_avg_sq_scales[i] : nullptr, numels[i], (uint32_t)chunks, (uint16_t)param_dtypes[i], (uint16_t)grad_dtypes[i]};
            chunks += more;
        }
        if (!tab.count) break;
        adamw_kernel<<<(unsigned)chunks, AW_THREADS, 0, (cudaStream_t)stream>>>(tab);
        if (const cudaError_t e = cudaGetLastError()) return (int)e;
    }
    return VIG_OK;
}
