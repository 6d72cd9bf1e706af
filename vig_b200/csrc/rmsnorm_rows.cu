// RMS norm behind a residual add, in the two forms that the block's own kernel (elementwise.cu) does not have: 8-bit rows with scales
// for a product in 8 bits, and a forward with its backward for training.
//
// r = x + residual,  rstd = 1/sqrt(mean(r^2) + eps),  y = r rstd w.
// 8 bits: a row, or each group of 32, 64 or 128 channels of it, has the scale s = max|y| / top (448 for e4m3, 127 for int8) and the codes
// round(y/s); where all of y is zero (or s below the smallest normal number), s and the codes are 0, and a NaN makes s NaN.  y is never rounded to 16 bits on the way.
// Backward, with t = w dy and xh = r rstd:  dr = rstd (t - xh mean(t xh)) + d_r,  dw = sum over rows of dy xh; rstd is computed again from r.
// In 16 bits the backward takes the sum from x and the residual again: r as it was rounded would be one tensor instead of two (8 in all instead
// of 9, backward 68 us instead of 86 in graph replays), but its roundings stand in dw beside dw's own, 2.5e-3 from 64 bits instead of 1.8e-3 in bf16.
// Bound by memory: x, residual in, r and one byte a value out; backward dy, x, residual, d_r in, dr out.  Calls on other inputs and outputs than the
// last: 131072 x 768 bf16 to e4m3 117 us (6.0 TB/s); 262144 x 192 bf16 forward 67 us (6.0 TB/s), backward 89 us (5.7 TB/s); one row of 768 2.6 us, a
// launch.  Rows off 16 bytes are read and written a value at a time: 32768 x 767 87 / 122 / 145 us, 768 35 / 37 / 51; rows wider than a CTA's
// registers (norm_any_kernel, 4096 x 20000) 279 / 307 / 768 us, 0.3 of the bandwidth forward and 0.16 backward.
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
    int whole = 0;                   // rows of all tensors are whole 16-byte vectors on 16 bytes
};

struct NormBwdParams {
    const void *dy, *x, *res, *w, *dr;       // r = x + res (x itself where res is NULL)
    void *dx, *dw;
    float* partial;                  // [blocks][N]
    int64_t ldy, ldx, ldr, lddr, rows;
    int N, w_f32, blocks;
    float eps;
    int whole = 0;
};

template <int OUT> __device__ __forceinline__ float out_top() { return OUT == VIG_OUT_INT8 ? 127.f : 448.f; }

template <int OUT> __device__ __forceinline__ uint8_t code_of(float v) {
    if (OUT == VIG_OUT_INT8) return (uint8_t)(int8_t)__float2int_rn(v);          // 127 at most, by the scale; 0 for a NaN
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

// Rows too wide for the registers of a CTA (more than 16384 values of 16 bits, 8192 of fp32): a CTA takes a row a value at a time, and reads
// it again for every step.
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

// Backward, rows too wide for registers: a CTA's share of dw stays in its row of the workspace (only the thread that owns a
// channel touches it), and a second launch adds the CTAs' shares in their order, so results do not depend on timing.
template <typename T>
__global__ void __launch_bounds__(NT) norm_bwd_any_kernel(const NormBwdParams p) {
    __shared__ float sh[NT / 32];
    const int tid = threadIdx.x;
    float* part = p.partial + (int64_t)blockIdx.x * p.N;
    for (int i = tid; i < p.N; i += NT) part[i] = 0.f;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.ldx;
        const T* res = p.res ? (const T*)p.res + row * p.ldr : nullptr;
        const T* dy = (const T*)p.dy + row * p.ldy;
        const T* dr = p.dr ? (const T*)p.dr + row * p.lddr : nullptr;
        auto sum = [&](int i) { return DType<T>::to_f(x[i]) + (res ? DType<T>::to_f(res[i]) : 0.f); };
        float ss = 0.f, dot = 0.f;
        for (int i = tid; i < p.N; i += NT) {
            const float v = sum(i);
            ss = fmaf(v, v, ss);
            dot = fmaf(v, DType<T>::to_f(dy[i]) * weight_at<T>(p.w, i, p.w_f32), dot);
        }
        ss = block_sum(ss, sh);
        dot = block_sum(dot, sh);
        const float rstd = 1.f / sqrtf(ss / (float)p.N + p.eps), c = dot / (float)p.N * rstd;
        for (int i = tid; i < p.N; i += NT) {
            const float xh = sum(i) * rstd, d = DType<T>::to_f(dy[i]);
            part[i] = fmaf(d, xh, part[i]);
            float v = rstd * (d * weight_at<T>(p.w, i, p.w_f32) - xh * c);
            if (dr) v += DType<T>::to_f(dr[i]);
            ((T*)p.dx)[row * p.N + i] = DType<T>::from_f(v);
        }
    }
}

// dw = the CTAs' shares, added in a fixed order: 32 channels x 32 warps
constexpr int DW = 32;

template <typename T>
__global__ void __launch_bounds__(DW * 32) norm_dw_kernel(const NormBwdParams p) {
    __shared__ float sh[DW][32];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
    pdl_wait();
    float s = 0.f;
    if (i < p.N) {
#pragma unroll 16
        for (int b = wid; b < p.blocks; b += DW) s += p.partial[(int64_t)b * p.N + i];
    }
    sh[wid][lane] = s;
    __syncthreads();
    if (wid == 0 && i < p.N) {
#pragma unroll
        for (int k = 1; k < DW; ++k) s += sh[k][lane];
        if (p.w_f32) ((float*)p.dw)[i] = s;
        else ((T*)p.dw)[i] = DType<T>::from_f(s);
    }
}

// ---------------------------------------------------------------------------------------------------
// TPR threads share a row; a thread holds VPT vectors of 16 bytes of it (vector t + m * TPR) and their weights in registers, and its next
// row is in flight while it works on one.  Everything about a row that needs the other threads -- the sum of squares and max|r w| --
// comes out of one reading and one reduction.  TPR below 32: a warp takes several rows; above: a CTA takes one.  Rows that are no whole
// vectors, or do not begin on 16 bytes, are read and written a value at a time in the same arrangement: the same bits come out.
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

template <int OUT, int V> __device__ __forceinline__ void store_codes(uint8_t* row, int vi, int N, int whole, const float* t, float rstd, float inv) {
    // y first: rstd times the scale's reciprocal may be out of range where neither is
    uint32_t word[V / 4];
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
        if (OUT == VIG_OUT_E4M3) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(t[4 * j] * rstd * inv, t[4 * j + 1] * rstd * inv), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(t[4 * j + 2] * rstd * inv, t[4 * j + 3] * rstd * inv), __NV_SATFINITE, __NV_E4M3);
            word[j] = lo | hi << 16;
        } else {
            word[j] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) word[j] |= (uint32_t)(uint8_t)(int8_t)__float2int_rn(t[4 * j + i] * rstd * inv) << (8 * i);
        }
    }
    uint8_t* q = row + vi * V;
    if (!whole) {
#pragma unroll
        for (int i = 0; i < V; ++i) if (vi * V + i < N) q[i] = (uint8_t)(word[i / 4] >> (8 * (i % 4)));
    } else if constexpr (V == 8) {
        *(uint2*)q = make_uint2(word[0], word[1]);
    } else {
        *(uint32_t*)q = word[0];
    }
}

template <int TPR> constexpr int norm_threads = TPR > 128 ? TPR : 128;

template <typename T, int OUT, int TPR, int VPT>
__global__ void __launch_bounds__(norm_threads<TPR>) norm_rows_kernel(const NormParams p) {
    constexpr int V = DType<T>::VEC, THREADS = norm_threads<TPR>, RPB = THREADS / TPR;            // RPB: rows of a CTA at a time
    static_assert(TPR <= 32 || RPB == 1, "a row's threads are part of a warp, or a CTA");
    __shared__ float sh[2 * (THREADS / 32)][2];
    int buf = 0;
    const int t = threadIdx.x % TPR, nv = (p.N + V - 1) / V, lanes = p.group / V;
    const int64_t hop = (int64_t)gridDim.x * RPB;
    float wf[VPT][V];
#pragma unroll
    for (int m = 0; m < VPT; ++m)
        if (t + m * TPR < nv) weights_of<T>(p.w, p.w_f32, t + m * TPR, p.N, p.whole, wf[m]);
    Vec16<T> xn[VPT], rn[VPT];
    auto fetch = [&](int64_t row) {
        if (row >= p.rows) return;
        const T *x = (const T*)p.x + row * p.ldx, *res = p.res ? (const T*)p.res + row * p.ldr : nullptr;
#pragma unroll
        for (int m = 0; m < VPT; ++m) {
            const int vi = t + m * TPR;
            if (vi < nv) {
                take<T>(xn[m], x, vi, p.N, p.whole);
                if (res) take<T>(rn[m], res, vi, p.N, p.whole);
            }
        }
    };
    int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    fetch(row);
    // a CTA's threads leave together: all of them take part in every reduction
    for (int64_t first = (int64_t)blockIdx.x * RPB; first < p.rows; first += hop, row += hop) {
        const bool in = row < p.rows;
        float v[VPT][V], gt[VPT], ss = 0.f, top = 0.f;
#pragma unroll
        for (int m = 0; m < VPT; ++m) {
            const int vi = t + m * TPR;
            gt[m] = 0.f;
            if (in && vi < nv) {
                xn[m].to_float(v[m]);
                if (p.res) {
                    float rf[V];
                    rn[m].to_float(rf);
#pragma unroll
                    for (int i = 0; i < V; ++i) v[m][i] += rf[i];
                }
                if (p.r) { Vec16<T> o; o.from_float(v[m]); give<T>(o, (T*)p.r + row * p.N, vi, p.N, p.whole); }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    ss = fmaf(v[m][i], v[m][i], ss);
                    v[m][i] *= wf[m][i];
                    if (OUT != OUT_SAME) gt[m] = top_of(gt[m], fabsf(v[m][i]));
                }
                top = top_of(top, gt[m]);
            }
        }
        fetch(row + hop);
        over_row<TPR, true>(ss, top, sh, buf);
        const float rstd = 1.f / sqrtf(ss / (float)p.N + p.eps);
        float inv = 0.f;
        if (OUT != OUT_SAME && p.group == p.N) {
            const float scale = scale_of<OUT>(top * rstd, &inv);
            if (in && t == 0) p.scales[row] = scale;
        }
#pragma unroll
        for (int m = 0; m < VPT; ++m) {
            const int vi = t + m * TPR;
            if (OUT != OUT_SAME && p.group != p.N) {             // group / V neighbouring threads share a group
                float g = gt[m];
                for (int k = lanes / 2; k; k >>= 1) g = top_of(g, __shfl_xor_sync(0xffffffffu, g, k));
                const float scale = scale_of<OUT>(g * rstd, &inv);
                if (in && vi < nv && vi % lanes == 0) p.scales[row * (p.N / p.group) + vi / lanes] = scale;
            }
            if (in && vi < nv) {
                if constexpr (OUT == OUT_SAME) {
#pragma unroll
                    for (int i = 0; i < V; ++i) v[m][i] *= rstd;
                    Vec16<T> o;
                    o.from_float(v[m]);
                    give<T>(o, (T*)p.y + row * p.N, vi, p.N, p.whole);
                } else {
                    store_codes<OUT, V>((uint8_t*)p.y + row * p.N, vi, p.N, p.whole, v[m], rstd, inv);
                }
            }
        }
    }
}

// Backward of the same rows: sum of squares and sum of r w dy in one reduction; a thread's share of dw stays in registers over all of its
// rows.  The next rows are on their way to shared memory meanwhile (262144 x 192 bf16, from the sum: 68 us; 81 without rows ahead, 169 with
// the row ahead in registers).  At the end the CTA's rows of threads are added, and a second launch adds the CTAs' shares in their order.
template <int TPR> constexpr int norm_bwd_threads = TPR > 256 ? TPR : TPR > 32 ? 256 : 128;

// CTAs of an SM, by the values a thread holds: as many as their registers allow without spilling (the same, 24 values: 68 us with 512
// threads an SM, 92 with 768 that spill)
template <int TPR, int VALUES> constexpr int norm_bwd_ctas = TPR > 256 ? 1 : TPR > 32 ? (VALUES <= 16 ? 3 : 2) : VALUES <= 24 ? 4 : 3;
// rows of a thread that are under way or at hand, four tensors each: two where that leaves room for another CTA
template <int TPR, int VPT> constexpr int norm_bwd_row = norm_bwd_threads<TPR> * 4 * VPT * 16;
template <int TPR, int VPT> constexpr int norm_bwd_ahead = 2 * norm_bwd_row<TPR, VPT> <= 112 * 1024 ? 2 : 1;
template <int TPR, int VPT> constexpr int norm_bwd_ring = norm_bwd_ahead<TPR, VPT> * norm_bwd_row<TPR, VPT>;

template <typename T, int TPR, int VPT, bool WHOLE>
__global__ void __launch_bounds__(norm_bwd_threads<TPR>, norm_bwd_ctas<TPR, VPT * DType<T>::VEC>) norm_bwd_rows_kernel(const NormBwdParams p) {
    constexpr int V = DType<T>::VEC, THREADS = norm_bwd_threads<TPR>, RPB = THREADS / TPR, AHEAD = norm_bwd_ahead<TPR, VPT>;
    static_assert(TPR <= 32 || RPB == 1, "a row's threads are part of a warp, or a CTA");
    __shared__ float sh[2 * (THREADS / 32)][2];
    extern __shared__ __align__(16) float share[];               // the ring; at the end [RPB][N]
    int buf = 0;
    const int t = threadIdx.x % TPR, nv = (p.N + V - 1) / V;
    const int64_t hop = (int64_t)gridDim.x * RPB;
    float wf[VPT][V], acc[VPT][V];
#pragma unroll
    for (int m = 0; m < VPT; ++m) {
#pragma unroll
        for (int i = 0; i < V; ++i) acc[m][i] = 0.f;
        if (t + m * TPR < nv) weights_of<T>(p.w, p.w_f32, t + m * TPR, p.N, WHOLE, wf[m]);
    }
    pdl_launch();
    // whole rows come to shared memory, every thread's vectors into slots of its own; others are read where they are
    const uint8_t* const ring = (const uint8_t*)share + threadIdx.x * 16;
    const auto slot = [&](int stage, int n, int m) { return ring + ((stage * 4 + n) * VPT + m) * THREADS * 16; };
    const auto source = [&](int n, int64_t row) {
        return n == 0 ? (const T*)p.x + row * p.ldx : n == 1 ? (const T*)p.dy + row * p.ldy : n == 2 ? (const T*)p.dr + row * p.lddr : (const T*)p.res + row * p.ldr;
    };
    auto bring = [&](int64_t row, int stage) {
        if (WHOLE && row < p.rows) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                if ((n == 2 && !p.dr) || (n == 3 && !p.res)) continue;
                const T* from = source(n, row);
#pragma unroll
                for (int m = 0; m < VPT; ++m)
                    if (t + m * TPR < nv)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(slot(stage, n, m))), "l"(from + (t + m * TPR) * V) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) bring(row + k * hop, k);
    int stage = 0;
    for (int64_t first = (int64_t)blockIdx.x * RPB; first < p.rows; first += hop, row += hop, stage = stage + 1 < AHEAD ? stage + 1 : 0) {
        const bool in = row < p.rows;
        asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
        const auto get = [&](int n, int m, float* f) {
            Vec16<T> v;
            if (WHOLE) v.load((const T*)slot(stage, n, m));
            else take<T>(v, source(n, row), t + m * TPR, p.N, 0);
            v.to_float(f);
        };
        const auto sum = [&](int m, float* f) {
            get(0, m, f);
            if (p.res) {
                float o[V];
                get(3, m, o);
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] += o[i];
            }
        };
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int m = 0; m < VPT; ++m) {
            if (in && t + m * TPR < nv) {
                float rf[V], df[V];
                sum(m, rf);
                get(1, m, df);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    ss = fmaf(rf[i], rf[i], ss);
                    dot = fmaf(rf[i], df[i] * wf[m][i], dot);
                }
            }
        }
        over_row<TPR, false>(ss, dot, sh, buf);
        const float rstd = 1.f / sqrtf(ss / (float)p.N + p.eps), c = -dot / (float)p.N * rstd * rstd;
#pragma unroll
        for (int m = 0; m < VPT; ++m) {
            const int vi = t + m * TPR;
            if (in && vi < nv) {
                float rf[V], df[V], o[V];
                sum(m, rf);
                get(1, m, df);
                if (p.dr) {
                    get(2, m, o);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) o[i] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float xh = rf[i] * rstd;
                    acc[m][i] = fmaf(df[i], xh, acc[m][i]);
                    o[i] = fmaf(df[i] * wf[m][i], rstd, fmaf(xh, c, o[i]));         // rstd (t - xh mean(t xh)) + d_r
                }
                Vec16<T> v;
                v.from_float(o);
                give<T>(v, (T*)p.dx + row * p.N, vi, p.N, WHOLE);
            }
        }
        bring(row + AHEAD * hop, stage);
    }
    if (RPB > 1) __syncthreads();                                // the ring's room is taken for the CTA's shares of dw
    float* part = p.partial + (int64_t)blockIdx.x * p.N;
#pragma unroll
    for (int m = 0; m < VPT; ++m) {
        const int vi = t + m * TPR;
        if (vi < nv) {
            float* to = RPB > 1 ? share + (threadIdx.x / TPR) * p.N : part;
#pragma unroll
            for (int i = 0; i < V / 4; ++i) give<float>(*(const Vec16<float>*)(acc[m] + 4 * i), to, vi * (V / 4) + i, p.N, WHOLE);
        }
    }
    if (RPB > 1) {
        __syncthreads();
        for (int i = threadIdx.x; i < p.N; i += THREADS) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < RPB; ++k) v += share[k * p.N + i];
            part[i] = v;
        }
    }
}

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

template <typename T, int OUT, int TPR> int norm_rows_launch(const NormParams& p, int nv, cudaStream_t s) {
    constexpr int THREADS = norm_threads<TPR>, RPB = THREADS / TPR;
    const int vpt = (nv + TPR - 1) / TPR;
    const int64_t need = (p.rows + RPB - 1) / RPB, most = (int64_t)device_sms() * (2048 / THREADS);
    const unsigned grid = (unsigned)(need < most ? need : most);
    switch (vpt) {
        case 1: norm_rows_kernel<T, OUT, TPR, 1><<<grid, THREADS, 0, s>>>(p); break;
        case 2: norm_rows_kernel<T, OUT, TPR, 2><<<grid, THREADS, 0, s>>>(p); break;
        case 3: norm_rows_kernel<T, OUT, TPR, 3><<<grid, THREADS, 0, s>>>(p); break;
        default: norm_rows_kernel<T, OUT, TPR, 4><<<grid, THREADS, 0, s>>>(p); break;
    }
    return (int)cudaGetLastError();
}

template <typename T, int OUT> int norm_launch(NormParams p, cudaStream_t s) {
    constexpr int V = DType<T>::VEC;
    const int size = (int)sizeof(T);
    p.whole = p.N % V == 0 && on_16(p.x, p.ldx, size) && (!p.res || on_16(p.res, p.ldr, size)) && on_16(p.w, 0, 1) && on_16(p.y, 0, 1) && (!p.r || on_16(p.r, 0, 1));
    const int nv = (p.N + V - 1) / V;
    switch (threads_a_row(nv, p.group != p.N && p.group / V > 8 ? p.group / V : 8)) {
        case 8: return norm_rows_launch<T, OUT, 8>(p, nv, s);
        case 16: return norm_rows_launch<T, OUT, 16>(p, nv, s);
        case 32: return norm_rows_launch<T, OUT, 32>(p, nv, s);
        case 64: case 128: return norm_rows_launch<T, OUT, 128>(p, nv, s);
        case 256: return norm_rows_launch<T, OUT, 256>(p, nv, s);
        case 512: return norm_rows_launch<T, OUT, 512>(p, nv, s);
    }
    const int64_t most = (int64_t)device_sms() * 8;
    norm_any_kernel<T, OUT><<<(unsigned)(p.rows < most ? p.rows : most), NT, 0, s>>>(p);
    return (int)cudaGetLastError();
}

template <typename T, int TPR, int VPT> int norm_bwd_rows(NormBwdParams& p, cudaStream_t s) {
    constexpr int THREADS = norm_bwd_threads<TPR>, RPB = THREADS / TPR;
    constexpr int smem = norm_bwd_ring<TPR, VPT>;                // more than RPB rows of N values in fp32
    constexpr int ctas = norm_bwd_ctas<TPR, VPT * DType<T>::VEC>, fit = 227 * 1024 / (smem + 2048);
    const int64_t need = (p.rows + RPB - 1) / RPB, room = (int64_t)device_sms() * (ctas < fit ? ctas : fit);
    p.blocks = (int)(need < room ? need : room);
    static_assert(smem >= RPB * TPR * VPT * DType<T>::VEC * 4, "the shares of dw find room where the ring was");
    void (*const kernel)(NormBwdParams) = p.whole ? norm_bwd_rows_kernel<T, TPR, VPT, true> : norm_bwd_rows_kernel<T, TPR, VPT, false>;
    if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return (int)e;
    kernel<<<p.blocks, THREADS, smem, s>>>(p);
    return (int)cudaGetLastError();
}

template <typename T, int TPR> int norm_bwd_rows_launch(NormBwdParams& p, int nv, cudaStream_t s) {
    switch ((nv + TPR - 1) / TPR) {
        case 1: return norm_bwd_rows<T, TPR, 1>(p, s);
        case 2: return norm_bwd_rows<T, TPR, 2>(p, s);
        case 3: return norm_bwd_rows<T, TPR, 3>(p, s);
        default: return norm_bwd_rows<T, TPR, 4>(p, s);
    }
}

template <typename T> int norm_bwd_launch(NormBwdParams p, cudaStream_t s) {
    constexpr int V = DType<T>::VEC;
    const int size = (int)sizeof(T);
    p.whole = p.N % V == 0 && on_16(p.x, p.ldx, size) && (!p.res || on_16(p.res, p.ldr, size)) && on_16(p.dy, p.ldy, size) && (!p.dr || on_16(p.dr, p.lddr, size)) && on_16(p.w, 0, 1) && on_16(p.dx, 0, 1) &&
                         on_16(p.partial, 0, 1);
    const int nv = (p.N + V - 1) / V, tpr = threads_a_row(nv, 8);
    int e;
    if (tpr <= 512) {
        switch (tpr) {
            case 8: e = norm_bwd_rows_launch<T, 8>(p, nv, s); break;
            case 16: e = norm_bwd_rows_launch<T, 16>(p, nv, s); break;
            case 32: e = norm_bwd_rows_launch<T, 32>(p, nv, s); break;
            case 512: e = norm_bwd_rows_launch<T, 512>(p, nv, s); break;
            default: e = norm_bwd_rows_launch<T, 256>(p, nv, s); break;
        }
    } else {
        norm_bwd_any_kernel<T><<<p.blocks, NT, 0, s>>>(p);
        e = (int)cudaGetLastError();
    }
    if (e) return e;
    return (int)launch_next(norm_dw_kernel<T>, dim3((p.N + 31) / 32), dim3(DW * 32), 0, s, p);
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
    if (rows < 0 || N <= 0 || N >= (1 << 30)) return VIG_ERR_SHAPE;
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

extern "C" int vig_add_rmsnorm_bwd(const void* dy, int64_t ldy, const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* w, int w_dtype, const void* d_r, int64_t ld_dr,
                                   void* dx, void* dw, int64_t rows, int N, float eps, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int e = norm_check(x, w, dx, rows, N, w_dtype, dtype)) return e;
    if (!dw || (rows && !dy)) return VIG_ERR_NULL;
    if (!rows) return (int)cudaMemsetAsync(dw, 0, (size_t)N * (w_dtype == VIG_DTYPE_F32 ? 4 : 2), (cudaStream_t)stream);
    if (!workspace || workspace_bytes < vig_add_rmsnorm_bwd_workspace_bytes(rows, N)) return VIG_ERR_WORKSPACE;
    const NormBwdParams p{dy, x, residual, w, d_r, dx, dw, (float*)workspace, ldy, ldx, ldr, ld_dr, rows, N, w_dtype == VIG_DTYPE_F32 && dtype != VIG_DTYPE_F32,
                          norm_blocks(rows), eps};
    switch (dtype) {
        case VIG_DTYPE_F32: return norm_bwd_launch<float>(p, (cudaStream_t)stream);
        case VIG_DTYPE_BF16: return norm_bwd_launch<__nv_bfloat16>(p, (cudaStream_t)stream);
        default: return norm_bwd_launch<__half>(p, (cudaStream_t)stream);
    }
}
