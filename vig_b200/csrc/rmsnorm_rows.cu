// RMS norm behind a residual add, in the two forms that the block's own kernel (elementwise.cu) does not have: 8-bit rows with scales
// for a product in 8 bits, and a forward with its backward for training.
//
// r = x + residual,  rstd = 1/sqrt(mean(r^2) + eps),  y = r rstd w.
// 8 bits: a row, or each group of 32, 64 or 128 channels of it, has the scale s = max|y| / top (448 for e4m3, 127 for int8) and the codes
// round(y/s); where all of y is zero (or s below the smallest normal number), s and the codes are 0, and a NaN makes s NaN.  y is never rounded to 16 bits on the way.
// Backward, with t = w dy and xh = r rstd:  dr = rstd (t - xh mean(t xh)) + d_r,  dw = sum over rows of dy xh; rstd is computed again from r.
// Bound by memory: x, residual in, r and one byte a value out; backward dy, r, d_r in, dr out.
#include <cuda_fp8.h>
#include "common.cuh"

namespace vig {

constexpr int OUT_SAME = -1;         // y in x's type; else VIG_OUT_E4M3 or VIG_OUT_INT8

struct NormParams {
    const void *x, *res, *w;
    void *y, *r;
    float* scales;
    int64_t ldx, ldr, rows;
    int N, group, w_f32;
    float eps;
};

struct NormBwdParams {
    const void *dy, *r, *w, *dr;
    void *dx, *dw;
    float* partial;                  // [blocks][N]
    int64_t ldy, ldr, lddr, rows;
    int N, w_f32, blocks;
    float eps;
};

template <int OUT> __device__ __forceinline__ float out_top() { return OUT == VIG_OUT_INT8 ? 127.f : 448.f; }

template <int OUT> __device__ __forceinline__ uint8_t code_of(float v) {
    if (OUT == VIG_OUT_INT8) return (uint8_t)(int8_t)__float2int_rn(fminf(fmaxf(v, -127.f), 127.f));
    return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

// scale of a group from the bits of its largest |y| (as integers they order like the values, and a NaN comes out on top), and what
// y is multiplied by
template <int OUT> __device__ __forceinline__ float scale_of(float top, float* inv) {
    float s = top * (1.f / out_top<OUT>());
    if (s < 1.17549435e-38f) s = 0.f;                            // its reciprocal is no number of this type
    *inv = s > 0.f ? 1.f / s : s;
    return s;
}

template <typename T> __device__ __forceinline__ float weight_at(const void* w, int i, int w_f32) {
    return w_f32 ? ((const float*)w)[i] : DType<T>::to_f(((const T*)w)[i]);
}

constexpr int NT = 256;

__device__ __forceinline__ float block_sum(float v, float* sh) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) v += sh[i];
    return v;
}

__device__ __forceinline__ float block_top(float v, float* sh) {
    uint32_t u = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(v)));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = __uint_as_float(u);
    __syncthreads();
    u = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) u = max(u, __float_as_uint(sh[i]));
    return __uint_as_float(u);
}

// Rows of any width and alignment: a CTA takes a row a value at a time, and reads it again for every step.
template <typename T, int OUT>
__global__ void __launch_bounds__(NT) norm_any_kernel(const NormParams p) {
    __shared__ float sh[NT / 32];
    const int tid = threadIdx.x, lane = tid & 31;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.ldx;
        const T* res = p.res ? (const T*)p.res + row * p.ldr : nullptr;
        auto sum = [&](int i) { return DType<T>::to_f(x[i]) + (res ? DType<T>::to_f(res[i]) : 0.f); };
        float ss = 0.f;
        for (int i = tid; i < p.N; i += NT) { const float v = sum(i); ss = fmaf(v, v, ss); }
        const float rstd = 1.f / sqrtf(block_sum(ss, sh) / (float)p.N + p.eps);
        if (OUT == OUT_SAME) {
            for (int i = tid; i < p.N; i += NT) {
                const float v = sum(i);
                ((T*)p.y)[row * p.N + i] = DType<T>::from_f(v * rstd * weight_at<T>(p.w, i, p.w_f32));
                if (p.r) ((T*)p.r)[row * p.N + i] = DType<T>::from_f(v);
            }
        } else if (p.group == p.N) {
            uint32_t top = 0;
            for (int i = tid; i < p.N; i += NT) top = max(top, __float_as_uint(fabsf(sum(i) * rstd * weight_at<T>(p.w, i, p.w_f32))));
            float inv;
            const float s = scale_of<OUT>(block_top(__uint_as_float(top), sh), &inv);
            if (tid == 0) p.scales[row] = s;
            for (int i = tid; i < p.N; i += NT) {
                const float v = sum(i);
                ((uint8_t*)p.y)[row * p.N + i] = code_of<OUT>(v * rstd * weight_at<T>(p.w, i, p.w_f32) * inv);
                if (p.r) ((T*)p.r)[row * p.N + i] = DType<T>::from_f(v);
            }
        } else {
            // a warp takes a group of 32, 64 or 128
            for (int g0 = (tid >> 5) * p.group; g0 < p.N; g0 += NT / 32 * p.group) {
                uint32_t top = 0;
                for (int i = g0 + lane; i < g0 + p.group; i += 32) top = max(top, __float_as_uint(fabsf(sum(i) * rstd * weight_at<T>(p.w, i, p.w_f32))));
                float inv;
                const float s = scale_of<OUT>(__uint_as_float(__reduce_max_sync(0xffffffffu, top)), &inv);
                if (lane == 0) p.scales[row * (p.N / p.group) + g0 / p.group] = s;
                for (int i = g0 + lane; i < g0 + p.group; i += 32) {
                    const float v = sum(i);
                    ((uint8_t*)p.y)[row * p.N + i] = code_of<OUT>(v * rstd * weight_at<T>(p.w, i, p.w_f32) * inv);
                    if (p.r) ((T*)p.r)[row * p.N + i] = DType<T>::from_f(v);
                }
            }
        }
    }
}

// Backward, rows of any width and alignment: a CTA's share of dw stays in its row of the workspace (only the thread that owns a
// channel touches it), and a second launch adds the CTAs' shares in their order, so results do not depend on timing.
template <typename T>
__global__ void __launch_bounds__(NT) norm_bwd_any_kernel(const NormBwdParams p) {
    __shared__ float sh[NT / 32];
    const int tid = threadIdx.x;
    float* part = p.partial + (int64_t)blockIdx.x * p.N;
    for (int i = tid; i < p.N; i += NT) part[i] = 0.f;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* r = (const T*)p.r + row * p.ldr;
        const T* dy = (const T*)p.dy + row * p.ldy;
        const T* dr = p.dr ? (const T*)p.dr + row * p.lddr : nullptr;
        float ss = 0.f, dot = 0.f;
        for (int i = tid; i < p.N; i += NT) {
            const float v = DType<T>::to_f(r[i]);
            ss = fmaf(v, v, ss);
            dot = fmaf(v, DType<T>::to_f(dy[i]) * weight_at<T>(p.w, i, p.w_f32), dot);
        }
        ss = block_sum(ss, sh);
        dot = block_sum(dot, sh);
        const float rstd = 1.f / sqrtf(ss / (float)p.N + p.eps), c = dot / (float)p.N * rstd;
        for (int i = tid; i < p.N; i += NT) {
            const float xh = DType<T>::to_f(r[i]) * rstd, d = DType<T>::to_f(dy[i]);
            part[i] = fmaf(d, xh, part[i]);
            float v = rstd * (d * weight_at<T>(p.w, i, p.w_f32) - xh * c);
            if (dr) v += DType<T>::to_f(dr[i]);
            ((T*)p.dx)[row * p.N + i] = DType<T>::from_f(v);
        }
    }
}

// dw = the CTAs' shares, added in their order: 32 channels x 8 warps
template <typename T>
__global__ void __launch_bounds__(NT) norm_dw_kernel(const NormBwdParams p) {
    __shared__ float sh[NT / 32][32];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (i < p.N)
        for (int b = wid; b < p.blocks; b += NT / 32) s += p.partial[(int64_t)b * p.N + i];
    sh[wid][lane] = s;
    __syncthreads();
    if (wid == 0 && i < p.N) {
#pragma unroll
        for (int k = 1; k < NT / 32; ++k) s += sh[k][lane];
        if (p.w_f32) ((float*)p.dw)[i] = s;
        else ((T*)p.dw)[i] = DType<T>::from_f(s);
    }
}

static int norm_blocks(int64_t rows) {
    const int64_t most = (int64_t)device_sms() * 4;
    return (int)(rows < most ? rows : most);
}

template <typename T, int OUT> int norm_launch(const NormParams& p, cudaStream_t s) {
    const int64_t most = (int64_t)device_sms() * 8;
    norm_any_kernel<T, OUT><<<(unsigned)(p.rows < most ? p.rows : most), NT, 0, s>>>(p);
    return (int)cudaGetLastError();
}

template <typename T> int norm_bwd_launch(const NormBwdParams& p, cudaStream_t s) {
    norm_bwd_any_kernel<T><<<p.blocks, NT, 0, s>>>(p);
    if (const cudaError_t e = cudaGetLastError()) return (int)e;
    norm_dw_kernel<T><<<(p.N + 31) / 32, NT, 0, s>>>(p);
    return (int)cudaGetLastError();
}

template <int OUT> int norm_dispatch(const NormParams& p, int dtype, cudaStream_t s) {
    switch (dtype) {
        case VIG_DTYPE_F32: return norm_launch<float, OUT>(p, s);
        case VIG_DTYPE_BF16: return norm_launch<__nv_bfloat16, OUT>(p, s);
        case VIG_DTYPE_F16: return norm_launch<__half, OUT>(p, s);
    }
    return VIG_ERR_DTYPE;
}

static int norm_check(const void* x, const void* w, const void* y, int64_t rows, int N, int w_dtype, int dtype) {
    if (dtype < VIG_DTYPE_F32 || dtype > VIG_DTYPE_F16 || (w_dtype != dtype && w_dtype != VIG_DTYPE_F32)) return VIG_ERR_DTYPE;
    if (rows < 0 || N <= 0) return VIG_ERR_SHAPE;
    if (rows && (!x || !w || !y)) return VIG_ERR_NULL;
    return VIG_OK;
}

}  // namespace vig

using namespace vig;

extern "C" int vig_add_rmsnorm_8bit_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* w, int w_dtype, void* q, float* scales,
                                        void* residual_out, int64_t rows, int N, int group, float eps, int out_type, int dtype, void* stream) {
    if (const int e = norm_check(x, w, q, rows, N, w_dtype, dtype)) return e;
    if (out_type != VIG_OUT_E4M3 && out_type != VIG_OUT_INT8) return VIG_ERR_ARG;
    if (group == 0) group = N;
    if (group != N && ((group != 32 && group != 64 && group != 128) || N % group)) return VIG_ERR_SHAPE;
    if (!rows) return VIG_OK;
    if (!scales) return VIG_ERR_NULL;
    const NormParams p{x, residual, w, q, residual_out, scales, ldx, ldr, rows, N, group, w_dtype == VIG_DTYPE_F32 && dtype != VIG_DTYPE_F32, eps};
    return out_type == VIG_OUT_E4M3 ? norm_dispatch<VIG_OUT_E4M3>(p, dtype, (cudaStream_t)stream) : norm_dispatch<VIG_OUT_INT8>(p, dtype, (cudaStream_t)stream);
}

extern "C" int vig_add_rmsnorm_train_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* w, int w_dtype, void* y,
                                         void* residual_out, int64_t rows, int N, float eps, int dtype, void* stream) {
    if (const int e = norm_check(x, w, y, rows, N, w_dtype, dtype)) return e;
    if (!rows) return VIG_OK;
    const NormParams p{x, residual, w, y, residual_out, nullptr, ldx, ldr, rows, N, N, w_dtype == VIG_DTYPE_F32 && dtype != VIG_DTYPE_F32, eps};
    return norm_dispatch<OUT_SAME>(p, dtype, (cudaStream_t)stream);
}

extern "C" size_t vig_add_rmsnorm_bwd_workspace_bytes(int64_t rows, int N) {
    return rows > 0 && N > 0 ? (size_t)norm_blocks(rows) * N * sizeof(float) : 0;
}

extern "C" int vig_add_rmsnorm_bwd(const void* dy, int64_t ldy, const void* r, int64_t ldr, const void* w, int w_dtype, const void* d_r, int64_t ld_dr,
                                   void* dx, void* dw, int64_t rows, int N, float eps, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int e = norm_check(r, w, dx, rows, N, w_dtype, dtype)) return e;
    if (!dw || (rows && !dy)) return VIG_ERR_NULL;
    if (!rows) return (int)cudaMemsetAsync(dw, 0, (size_t)N * (w_dtype == VIG_DTYPE_F32 ? 4 : 2), (cudaStream_t)stream);
    if (!workspace || workspace_bytes < vig_add_rmsnorm_bwd_workspace_bytes(rows, N)) return VIG_ERR_WORKSPACE;
    const NormBwdParams p{dy, r, w, d_r, dx, dw, (float*)workspace, ldy, ldr, ld_dr, rows, N, w_dtype == VIG_DTYPE_F32 && dtype != VIG_DTYPE_F32,
                          norm_blocks(rows), eps};
    switch (dtype) {
        case VIG_DTYPE_F32: return norm_bwd_launch<float>(p, (cudaStream_t)stream);
        case VIG_DTYPE_BF16: return norm_bwd_launch<__nv_bfloat16>(p, (cudaStream_t)stream);
        default: return norm_bwd_launch<__half>(p, (cudaStream_t)stream);
    }
}
