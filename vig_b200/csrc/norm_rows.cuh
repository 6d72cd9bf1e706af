// What the kernels over rows of a norm share: a row's threads and their vectors, sums over a row, the workspace of the backward.
#pragma once
#include "common.cuh"

namespace vig {

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

template <typename T> __device__ __forceinline__ void take(Vec16<T>& v, const T* row, int vi, int N, int whole) {
    constexpr int V = DType<T>::VEC;
    if (whole) {
        v.load(row + vi * V);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v.e[i] = vi * V + i < N ? row[vi * V + i] : DType<T>::from_f(0.f);
    }
}
template <typename T> __device__ __forceinline__ void give(const Vec16<T>& v, T* row, int vi, int N, int whole) {
    constexpr int V = DType<T>::VEC;
    if (whole) {
        v.store(row + vi * V);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) if (vi * V + i < N) row[vi * V + i] = v.e[i];
    }
}
template <typename T> __device__ __forceinline__ void weights_of(const void* w, int w_f32, int vi, int N, int whole, float* f) {
    constexpr int V = DType<T>::VEC;
    if (w_f32) {
        Vec16<float> v[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            take<float>(v[i], (const float*)w, vi * (V / 4) + i, N, whole);
            v[i].to_float(f + 4 * i);
        }
    } else {
        Vec16<T> v;
        take<T>(v, (const T*)w, vi, N, whole);
        v.to_float(f);
    }
}

__device__ __forceinline__ float top_of(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }

// a summed and b summed (or, MAX, its largest value by bits) over the TPR threads of a row
template <int TPR, bool MAX> __device__ __forceinline__ void over_row(float& a, float& b, float (*sh)[2], int& buf) {
#pragma unroll
    for (int m = (TPR < 32 ? TPR : 32) / 2; m; m >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, m);
        const float o = __shfl_xor_sync(0xffffffffu, b, m);
        b = MAX ? top_of(b, o) : b + o;
    }
    if (TPR > 32) {
        constexpr int W = TPR / 32;
        float (*s)[2] = sh + buf * W;                            // two buffers in turn, so that one barrier a reduction is enough
        buf ^= 1;
        if ((threadIdx.x & 31) == 0) { s[threadIdx.x >> 5][0] = a; s[threadIdx.x >> 5][1] = b; }
        __syncthreads();
        a = s[0][0]; b = s[0][1];
#pragma unroll
        for (int i = 1; i < W; ++i) { a += s[i][0]; b = MAX ? top_of(b, s[i][1]) : b + s[i][1]; }
    }
}

template <int TPR> constexpr int norm_threads = TPR > 128 ? TPR : 128;

// CTAs of the backward, whose shares of dw the workspace holds: at most four an SM
static int norm_blocks(int64_t rows) {
    const int64_t most = (int64_t)device_sms() * 4;
    return (int)(rows < most ? rows : most);
}

// threads a row of nv vectors: a power of two of which three or four vectors a thread make the row (fewer where a group or a warp wants more)
static int threads_a_row(int nv, int least) {
    int tpr = least;
    while (tpr * 4 < nv) tpr *= 2;
    return tpr;
}

static bool on_16(const void* q, int64_t ld, int size) { return (uintptr_t)q % 16 == 0 && ld * size % 16 == 0; }

// dw = the CTAs' shares, added in a fixed order: 32 channels x 32 warps
constexpr int DW = 32;

}  // namespace vig
