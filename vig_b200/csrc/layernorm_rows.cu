// Layer norm behind a residual add, for training: forward, and backward with the reductions of the weight's and the bias's gradients.
//
// r = x + residual,  xh = (r - mean(r)) / sqrt(var(r) + eps),  y = xh w + bias.  With t = w dy:
//   dr = rstd (t - mean(t) - xh mean(t xh)) + d_r,   dw = sum over rows of dy xh,   dbias = sum over rows of dy.
// The variance is the mean of (r - mean)^2 with the row in registers, a second reduction: the mean of r^2 less the squared mean loses all digits where
// the mean is large beside the deviation.  Mean and deviation are computed again in the backward, from x and the residual (in 16 bits the rounded sum
// would put its rounding into dw).  Bound by memory: x, residual in, y, r out; backward dy, x, residual, d_r in, dr out.
// 200704 x 96 bf16: forward 37 us (4.2 TB/s), backward 41 (4.7 TB/s).
#include "norm_rows.cuh"

namespace vig {

struct LayerParams {
    const void *x, *res, *w, *bias;
    void *y, *r;
    int64_t ldx, ldr, rows;
    int N, w_f32;
    float eps;
    int whole = 0;                   // rows of all tensors are whole 16-byte vectors on 16 bytes
};

struct LayerBwdParams {
    const void *dy, *x, *res, *w, *dr;
    void *dx, *dw, *dbias;
    float* partial;                  // [block][dw, dbias][N]
    int64_t ldy, ldx, ldr, lddr, rows;
    int N, w_f32, blocks;
    float eps;
    int whole = 0;
};

// Rows too wide for the registers of a CTA: a value at a time, read again for every step.
template <typename T> __global__ void __launch_bounds__(NT) layer_any_kernel(const LayerParams p) {
    __shared__ float sh[NT / 32];
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.ldx;
        const T* res = p.res ? (const T*)p.res + row * p.ldr : nullptr;
        auto sum = [&](int i) { return DType<T>::to_f(x[i]) + (res ? DType<T>::to_f(res[i]) : 0.f); };
        float s = 0.f, ss = 0.f;
        for (int i = threadIdx.x; i < p.N; i += NT) s += sum(i);
        const float mean = block_sum(s, sh) / (float)p.N;
        for (int i = threadIdx.x; i < p.N; i += NT) { const float v = sum(i) - mean; ss = fmaf(v, v, ss); }
        const float rstd = 1.f / sqrtf(block_sum(ss, sh) / (float)p.N + p.eps);
        for (int i = threadIdx.x; i < p.N; i += NT) {
            const float v = sum(i);
            ((T*)p.y)[row * p.N + i] = DType<T>::from_f(fmaf((v - mean) * rstd, weight_at<T>(p.w, i, p.w_f32), p.bias ? weight_at<T>(p.bias, i, p.w_f32) : 0.f));
            if (p.r) ((T*)p.r)[row * p.N + i] = DType<T>::from_f(v);
        }
    }
}

template <typename T> __global__ void __launch_bounds__(NT) layer_bwd_any_kernel(const LayerBwdParams p) {
    __shared__ float sh[NT / 32];
    float *pw = p.partial + (int64_t)blockIdx.x * 2 * p.N, *pb = pw + p.N;
    for (int i = threadIdx.x; i < p.N; i += NT) pw[i] = pb[i] = 0.f;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.ldx;
        const T* res = p.res ? (const T*)p.res + row * p.ldr : nullptr;
        const T* dy = (const T*)p.dy + row * p.ldy;
        const T* dr = p.dr ? (const T*)p.dr + row * p.lddr : nullptr;
        auto sum = [&](int i) { return DType<T>::to_f(x[i]) + (res ? DType<T>::to_f(res[i]) : 0.f); };
        auto back = [&](int i) { return DType<T>::to_f(dy[i]) * weight_at<T>(p.w, i, p.w_f32); };
        float s = 0.f, st = 0.f, ss = 0.f, dot = 0.f;
        for (int i = threadIdx.x; i < p.N; i += NT) { s += sum(i); st += back(i); }
        const float mean = block_sum(s, sh) / (float)p.N, mean_t = block_sum(st, sh) / (float)p.N;
        for (int i = threadIdx.x; i < p.N; i += NT) { const float v = sum(i) - mean; ss = fmaf(v, v, ss); dot = fmaf(v, back(i), dot); }
        const float rstd = 1.f / sqrtf(block_sum(ss, sh) / (float)p.N + p.eps), c = block_sum(dot, sh) / (float)p.N * rstd;
        for (int i = threadIdx.x; i < p.N; i += NT) {
            const float xh = (sum(i) - mean) * rstd, d = DType<T>::to_f(dy[i]);
            pw[i] = fmaf(d, xh, pw[i]);
            pb[i] += d;
            float v = rstd * (back(i) - mean_t - xh * c);
            if (dr) v += DType<T>::to_f(dr[i]);
            ((T*)p.dx)[row * p.N + i] = DType<T>::from_f(v);
        }
    }
}

template <typename T> __global__ void __launch_bounds__(DW * 32) layer_dw_kernel(const LayerBwdParams p) {
    __shared__ float sh[DW][32];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;       // dw, and behind it dbias
    pdl_wait();
    float s = 0.f;
    if (i < 2 * p.N) {
#pragma unroll 16
        for (int b = wid; b < p.blocks; b += DW) s += p.partial[(int64_t)b * 2 * p.N + i];
    }
    sh[wid][lane] = s;
    __syncthreads();
    if (wid == 0 && i < 2 * p.N) {
#pragma unroll
        for (int k = 1; k < DW; ++k) s += sh[k][lane];
        void* to = i < p.N ? p.dw : p.dbias;
        const int at = i < p.N ? i : i - p.N;
        if (!to) return;
        if (p.w_f32) ((float*)to)[at] = s;
        else ((T*)to)[at] = DType<T>::from_f(s);
    }
}

// a summed over the TPR threads of a row
template <int TPR> __device__ __forceinline__ void over_row(float& a, float (*sh)[2], int& buf) {
#pragma unroll
    for (int m = (TPR < 32 ? TPR : 32) / 2; m; m >>= 1) a += __shfl_xor_sync(0xffffffffu, a, m);
    if (TPR > 32) {
        constexpr int W = TPR / 32;
        float (*s)[2] = sh + buf * W;
        buf ^= 1;
        if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5][0] = a;
        __syncthreads();
        a = s[0][0];
#pragma unroll
        for (int i = 1; i < W; ++i) a += s[i][0];
    }
}

// TPR threads share a row, VPT vectors of 16 bytes each, as in the RMS norm's kernels.
template <typename T, int TPR, int VPT> __global__ void __launch_bounds__(norm_threads<TPR>) layer_rows_kernel(const LayerParams p) {
    constexpr int V = DType<T>::VEC, THREADS = norm_threads<TPR>, RPB = THREADS / TPR;
    static_assert(TPR <= 32 || RPB == 1, "a row's threads are part of a warp, or a CTA");
    __shared__ float sh[2 * (THREADS / 32)][2];
    int buf = 0;
    const int t = threadIdx.x % TPR, nv = (p.N + V - 1) / V;
    const int64_t hop = (int64_t)gridDim.x * RPB;
    float wf[VPT][V], bf[VPT][V];
#pragma unroll
    for (int m = 0; m < VPT; ++m) {
        if (t + m * TPR < nv) {
            weights_of<T>(p.w, p.w_f32, t + m * TPR, p.N, p.whole, wf[m]);
            if (p.bias) weights_of<T>(p.bias, p.w_f32, t + m * TPR, p.N, p.whole, bf[m]);
        }
        if (!p.bias) {
#pragma unroll
            for (int i = 0; i < V; ++i) bf[m][i] = 0.f;
        }
    }
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
        float v[VPT][V], s = 0.f, ss = 0.f;
#pragma unroll
        for (int m = 0; m < VPT; ++m) {
            const int vi = t + m * TPR;
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
                for (int i = 0; i < V; ++i) s += v[m][i];                // values behind the row's end are zeros
            }
        }
        fetch(row + hop);
        over_row<TPR>(s, sh, buf);
        const float mean = s / (float)p.N;
#pragma unroll
        for (int m = 0; m < VPT; ++m) {
            const int vi = t + m * TPR;
            if (in && vi < nv) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    v[m][i] = p.whole || vi * V + i < p.N ? v[m][i] - mean : 0.f;
                    ss = fmaf(v[m][i], v[m][i], ss);
                }
            }
        }
        over_row<TPR>(ss, sh, buf);
        const float rstd = 1.f / sqrtf(ss / (float)p.N + p.eps);
#pragma unroll
        for (int m = 0; m < VPT; ++m) {
            const int vi = t + m * TPR;
            if (in && vi < nv) {
#pragma unroll
                for (int i = 0; i < V; ++i) v[m][i] = fmaf(v[m][i] * rstd, wf[m][i], bf[m][i]);
                Vec16<T> o;
                o.from_float(v[m]);
                give<T>(o, (T*)p.y + row * p.N, vi, p.N, p.whole);
            }
        }
    }
}

// Backward of the same rows.  A thread's shares of dw and dbias stay in registers over all of its rows; the next rows are on their way to shared memory
// meanwhile.  At the end the CTA's rows of threads are added, and a second launch adds the CTAs' shares in their order.
template <int TPR> constexpr int layer_bwd_threads = TPR > 256 ? TPR : TPR > 32 ? 256 : 128;
template <int TPR, int VALUES> constexpr int layer_bwd_ctas = TPR > 256 ? 1 : TPR > 32 ? 2 : VALUES <= 16 ? 4 : 3;
template <int TPR, int VPT> constexpr int layer_bwd_row = layer_bwd_threads<TPR> * 4 * VPT * 16;
template <int TPR, int VPT> constexpr int layer_bwd_ahead = 2 * layer_bwd_row<TPR, VPT> <= 112 * 1024 ? 2 : 1;
template <int TPR, int VPT> constexpr int layer_bwd_ring = layer_bwd_ahead<TPR, VPT> * layer_bwd_row<TPR, VPT>;

template <typename T, int TPR, int VPT, bool WHOLE>
__global__ void __launch_bounds__(layer_bwd_threads<TPR>, layer_bwd_ctas<TPR, VPT * DType<T>::VEC>) layer_bwd_rows_kernel(const LayerBwdParams p) {
    constexpr int V = DType<T>::VEC, THREADS = layer_bwd_threads<TPR>, RPB = THREADS / TPR, AHEAD = layer_bwd_ahead<TPR, VPT>;
    static_assert(TPR <= 32 || RPB == 1, "a row's threads are part of a warp, or a CTA");
    __shared__ float sh[2 * (THREADS / 32)][2];
    extern __shared__ __align__(16) float share[];               // the ring; at the end [RPB][N]
    int buf = 0;
    const int t = threadIdx.x % TPR, nv = (p.N + V - 1) / V;
    const int64_t hop = (int64_t)gridDim.x * RPB;
    float wf[VPT][V], dw[VPT][V], db[VPT][V];
#pragma unroll
    for (int m = 0; m < VPT; ++m) {
#pragma unroll
        for (int i = 0; i < V; ++i) dw[m][i] = db[m][i] = 0.f;
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
        float s = 0.f, st = 0.f, ss = 0.f, dot = 0.f;
#pragma unroll
        for (int m = 0; m < VPT; ++m) {
            if (in && t + m * TPR < nv) {
                float rf[V], df[V];
                sum(m, rf);
                get(1, m, df);
#pragma unroll
                for (int i = 0; i < V; ++i) { s += rf[i]; st = fmaf(df[i], wf[m][i], st); }
            }
        }
        over_row<TPR, false>(s, st, sh, buf);
        const float mean = s / (float)p.N;
#pragma unroll
        for (int m = 0; m < VPT; ++m) {
            const int vi = t + m * TPR;
            if (in && vi < nv) {
                float rf[V], df[V];
                sum(m, rf);
                get(1, m, df);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float v = WHOLE || vi * V + i < p.N ? rf[i] - mean : 0.f;
                    ss = fmaf(v, v, ss);
                    dot = fmaf(v, df[i] * wf[m][i], dot);
                }
            }
        }
        over_row<TPR, false>(ss, dot, sh, buf);
        const float rstd = 1.f / sqrtf(ss / (float)p.N + p.eps), c0 = -st / (float)p.N * rstd, c1 = -dot / (float)p.N * rstd * rstd;
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
                    const float xh = (rf[i] - mean) * rstd;
                    dw[m][i] = fmaf(df[i], xh, dw[m][i]);
                    db[m][i] += df[i];
                    o[i] += fmaf(df[i] * wf[m][i], rstd, fmaf(xh, c1, c0));        // rstd (t - mean(t) - xh mean(t xh)) + d_r
                }
                Vec16<T> v;
                v.from_float(o);
                give<T>(v, (T*)p.dx + row * p.N, vi, p.N, WHOLE);
            }
        }
        bring(row + AHEAD * hop, stage);
    }
    float* part = p.partial + (int64_t)blockIdx.x * 2 * p.N;
#pragma unroll
    for (int which = 0; which < 2; ++which, part += p.N) {
        if (RPB > 1) __syncthreads();                            // the ring's room is taken for the CTA's shares
#pragma unroll
        for (int m = 0; m < VPT; ++m) {
            const int vi = t + m * TPR;
            if (vi < nv) {
                float* to = RPB > 1 ? share + (threadIdx.x / TPR) * p.N : part;
#pragma unroll
                for (int i = 0; i < V / 4; ++i) give<float>(*(const Vec16<float>*)((which ? db : dw)[m] + 4 * i), to, vi * (V / 4) + i, p.N, WHOLE);
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
}

template <typename T, int TPR> int layer_rows_launch(const LayerParams& p, int nv, cudaStream_t s) {
    constexpr int THREADS = norm_threads<TPR>, RPB = THREADS / TPR;
    const int64_t need = (p.rows + RPB - 1) / RPB, most = (int64_t)device_sms() * (2048 / THREADS);
    const unsigned grid = (unsigned)(need < most ? need : most);
    switch ((nv + TPR - 1) / TPR) {
        case 1: layer_rows_kernel<T, TPR, 1><<<grid, THREADS, 0, s>>>(p); break;
        case 2: layer_rows_kernel<T, TPR, 2><<<grid, THREADS, 0, s>>>(p); break;
        case 3: layer_rows_kernel<T, TPR, 3><<<grid, THREADS, 0, s>>>(p); break;
        default: layer_rows_kernel<T, TPR, 4><<<grid, THREADS, 0, s>>>(p); break;
    }
    return (int)cudaGetLastError();
}

template <typename T> int layer_launch(LayerParams p, cudaStream_t s) {
    constexpr int V = DType<T>::VEC;
    const int size = (int)sizeof(T), nv = (p.N + V - 1) / V;
    p.whole = p.N % V == 0 && on_16(p.x, p.ldx, size) && (!p.res || on_16(p.res, p.ldr, size)) && on_16(p.w, 0, 1) && on_16(p.bias, 0, 1) && on_16(p.y, 0, 1) && on_16(p.r, 0, 1);
    switch (threads_a_row(nv, 4)) {
        case 4: return layer_rows_launch<T, 4>(p, nv, s);
        case 8: return layer_rows_launch<T, 8>(p, nv, s);
        case 16: return layer_rows_launch<T, 16>(p, nv, s);
        case 32: return layer_rows_launch<T, 32>(p, nv, s);
        case 64: case 128: return layer_rows_launch<T, 128>(p, nv, s);
        case 256: return layer_rows_launch<T, 256>(p, nv, s);
        case 512: return layer_rows_launch<T, 512>(p, nv, s);
    }
    const int64_t most = (int64_t)device_sms() * 8;
    layer_any_kernel<T><<<(unsigned)(p.rows < most ? p.rows : most), NT, 0, s>>>(p);
    return (int)cudaGetLastError();
}

template <typename T, int TPR, int VPT> int layer_bwd_rows(LayerBwdParams& p, cudaStream_t s) {
    constexpr int THREADS = layer_bwd_threads<TPR>, RPB = THREADS / TPR;
    constexpr int smem = layer_bwd_ring<TPR, VPT>;
    constexpr int ctas = layer_bwd_ctas<TPR, VPT * DType<T>::VEC>, fit = 227 * 1024 / (smem + 2048);
    const int64_t need = (p.rows + RPB - 1) / RPB, room = (int64_t)device_sms() * (ctas < fit ? ctas : fit);
    p.blocks = (int)(need < room ? need : room);
    static_assert(smem >= RPB * TPR * VPT * DType<T>::VEC * 4, "the shares of dw find room where the ring was");
    void (*const kernel)(LayerBwdParams) = p.whole ? layer_bwd_rows_kernel<T, TPR, VPT, true> : layer_bwd_rows_kernel<T, TPR, VPT, false>;
    if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return (int)e;
    kernel<<<p.blocks, THREADS, smem, s>>>(p);
    return (int)cudaGetLastError();
}

template <typename T, int TPR> int layer_bwd_rows_launch(LayerBwdParams& p, int nv, cudaStream_t s) {
    switch ((nv + TPR - 1) / TPR) {
        case 1: return layer_bwd_rows<T, TPR, 1>(p, s);
        case 2: return layer_bwd_rows<T, TPR, 2>(p, s);
        case 3: return layer_bwd_rows<T, TPR, 3>(p, s);
        default: return layer_bwd_rows<T, TPR, 4>(p, s);
    }
}

template <typename T> int layer_bwd_launch(LayerBwdParams p, cudaStream_t s) {
    constexpr int V = DType<T>::VEC;
    const int size = (int)sizeof(T);
    p.whole = p.N % V == 0 && on_16(p.x, p.ldx, size) && (!p.res || on_16(p.res, p.ldr, size)) && on_16(p.dy, p.ldy, size) && (!p.dr || on_16(p.dr, p.lddr, size)) && on_16(p.w, 0, 1) &&
              on_16(p.dx, 0, 1) && on_16(p.partial, 0, 1);
    const int nv = (p.N + V - 1) / V;
    int e;
    switch (threads_a_row(nv, 4)) {
        case 4: e = layer_bwd_rows_launch<T, 4>(p, nv, s); break;
        case 8: e = layer_bwd_rows_launch<T, 8>(p, nv, s); break;
        case 16: e = layer_bwd_rows_launch<T, 16>(p, nv, s); break;
        case 32: e = layer_bwd_rows_launch<T, 32>(p, nv, s); break;
        case 64: case 128: case 256: e = layer_bwd_rows_launch<T, 256>(p, nv, s); break;
        case 512: e = layer_bwd_rows_launch<T, 512>(p, nv, s); break;
        default:
            layer_bwd_any_kernel<T><<<p.blocks, NT, 0, s>>>(p);
            e = (int)cudaGetLastError();
    }
    if (e) return e;
    return (int)launch_next(layer_dw_kernel<T>, dim3((2 * p.N + 31) / 32), dim3(DW * 32), 0, s, p);
}

static int layer_check(const void* x, const void* w, const void* y, int64_t rows, int N, int w_dtype, int dtype) {
    if (dtype < VIG_DTYPE_F32 || dtype > VIG_DTYPE_F16 || (w_dtype != dtype && w_dtype != VIG_DTYPE_F32)) return VIG_ERR_DTYPE;
    if (rows < 0 || N <= 0 || N >= (1 << 30)) return VIG_ERR_SHAPE;
    if (rows && (!x || !w || !y)) return VIG_ERR_NULL;
    return VIG_OK;
}

}  // namespace vig

using namespace vig;

extern "C" int vig_add_layernorm_train_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* w, const void* bias, int w_dtype, void* y,
                                           void* residual_out, int64_t rows, int N, float eps, int dtype, void* stream) {
    if (const int e = layer_check(x, w, y, rows, N, w_dtype, dtype)) return e;
    if (!rows) return VIG_OK;
    const LayerParams p{x, residual, w, bias, y, residual_out, ldx, ldr, rows, N, w_dtype == VIG_DTYPE_F32 && dtype != VIG_DTYPE_F32, eps};
    switch (dtype) {
        case VIG_DTYPE_F32: return layer_launch<float>(p, (cudaStream_t)stream);
        case VIG_DTYPE_BF16: return layer_launch<__nv_bfloat16>(p, (cudaStream_t)stream);
        default: return layer_launch<__half>(p, (cudaStream_t)stream);
    }
}

extern "C" size_t vig_add_layernorm_bwd_workspace_bytes(int64_t rows, int N) {
    return rows > 0 && N > 0 ? (size_t)norm_blocks(rows) * 2 * N * sizeof(float) : 0;
}

extern "C" int vig_add_layernorm_bwd(const void* dy, int64_t ldy, const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* w, int w_dtype,
                                     const void* d_r, int64_t ld_dr, void* dx, void* dw, void* d_bias, int64_t rows, int N, float eps, int dtype, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    if (const int e = layer_check(x, w, dx, rows, N, w_dtype, dtype)) return e;
    if (!dw || (rows && !dy)) return VIG_ERR_NULL;
    const cudaStream_t s = (cudaStream_t)stream;
    if (!rows) {
        const size_t bytes = (size_t)N * (w_dtype == VIG_DTYPE_F32 ? 4 : 2);
        if (const cudaError_t e = cudaMemsetAsync(dw, 0, bytes, s)) return (int)e;
        return d_bias ? (int)cudaMemsetAsync(d_bias, 0, bytes, s) : VIG_OK;
    }
    if (!workspace || workspace_bytes < vig_add_layernorm_bwd_workspace_bytes(rows, N)) return VIG_ERR_WORKSPACE;
    const LayerBwdParams p{dy, x, residual, w, d_r, dx, dw, d_bias, (float*)workspace, ldy, ldx, ldr, ld_dr, rows, N, w_dtype == VIG_DTYPE_F32 && dtype != VIG_DTYPE_F32,
                           norm_blocks(rows), eps};
    switch (dtype) {
        case VIG_DTYPE_F32: return layer_bwd_launch<float>(p, s);
        case VIG_DTYPE_BF16: return layer_bwd_launch<__nv_bfloat16>(p, s);
        default: return layer_bwd_launch<__half>(p, s);
    }
}
