// Short causal convolution, a channel at a time: pre_t = bias + sum_k w_k x_{t-K+1+k}, y = silu(pre) or pre.
// Backward: dpre = dy act'(pre) with pre computed again,  dx_t = sum_k w_k dpre_{t+K-1-k},  dw_k = sum_t dpre_t x_{t-K+1+k},  dbias = sum_t dpre_t.
//
// Bound by memory: x in, y out; backward x and dy in, dx out.  A thread walks a run of tokens of a few neighbouring channels and keeps the
// window in registers, so that each value is read once and, at the border of two runs, K - 1 times more out of the cache.
#include "common.cuh"

namespace vig {
namespace {

constexpr int MAX_K = 8;

struct ConvParams {
    const void *x, *w, *bias, *state, *dy, *d_out;               // d_out: gradient of the state handed on
    void *y, *state_out, *dx, *d_state, *dw, *dbias;
    float* partial;                                              // backward: [block][K + 1][D]
    const int32_t* lengths;
    int64_t s_x[2], s_y[2], s_st[2], s_out[2], s_dy[2];
    int B, L, D, w_f32, w_whole, silu, run, runs, blocks;
};

__device__ __forceinline__ int length_of(const ConvParams& p, int b) { return p.lengths ? min(max(p.lengths[b], 0), p.L) : p.L; }

template <typename T, int V> struct Piece {
    T e[V];
    __device__ void load(const T* q) {
        if constexpr (V * sizeof(T) == 16) { const uint4 w = *(const uint4*)q; memcpy(e, &w, 16); }
        else if constexpr (V * sizeof(T) == 8) { const uint2 w = *(const uint2*)q; memcpy(e, &w, 8); }
        else {
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] = q[i];
        }
    }
    __device__ void store(T* q) const {
        if constexpr (V * sizeof(T) == 16) { uint4 w; memcpy(&w, e, 16); *(uint4*)q = w; }
        else if constexpr (V * sizeof(T) == 8) { uint2 w; memcpy(&w, e, 8); *(uint2*)q = w; }
        else {
#pragma unroll
            for (int i = 0; i < V; ++i) q[i] = e[i];
        }
    }
    __device__ void zero() {
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = DType<T>::from_f(0.f);
    }
};

template <typename T> __device__ __forceinline__ float weight(const void* w, int64_t i, int f32) { return f32 ? ((const float*)w)[i] : DType<T>::to_f(((const T*)w)[i]); }

// the taps and biases of V neighbouring channels: whole pieces of 16 bytes where the channels are, since they lie one behind the other
template <typename T, typename W, int K, int V> __device__ __forceinline__ void taps_of(const W* w, const W* bias, int d, int whole, float (*f)[V], float* b) {
    W e[V * K], c[V];
    constexpr bool PIECES = V * (int)sizeof(W) % 16 == 0;
    if (PIECES && whole) {
        const uint4* from = (const uint4*)(w + (int64_t)d * K);
#pragma unroll
        for (int i = 0; i < V * K * (int)sizeof(W) / 16; ++i) { const uint4 v = __ldg(from + i); memcpy((char*)e + 16 * i, &v, 16); }
        if (bias) {
#pragma unroll
            for (int i = 0; i < V * (int)sizeof(W) / 16; ++i) { const uint4 v = __ldg((const uint4*)(bias + d) + i); memcpy((char*)c + 16 * i, &v, 16); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V * K; ++i) e[i] = w[(int64_t)d * K + i];
        if (bias) {
#pragma unroll
            for (int v = 0; v < V; ++v) c[v] = bias[d + v];
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        b[v] = bias ? DType<W>::to_f(c[v]) : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) f[k][v] = DType<W>::to_f(e[v * K + k]);
    }
}
template <typename T, int K, int V> __device__ __forceinline__ void taps(const ConvParams& p, int d, float (*f)[V], float* b) {
    if (p.w_f32) taps_of<T, float, K, V>((const float*)p.w, (const float*)p.bias, d, p.w_whole, f, b);
    else taps_of<T, T, K, V>((const T*)p.w, (const T*)p.bias, d, p.w_whole, f, b);
}

// token t of channels d..d+V-1: out of the state in front of the first, zeros from the end on
template <typename T, int K, int V> __device__ __forceinline__ Piece<T, V> token(const ConvParams& p, int b, int64_t t, int len, int d) {
    Piece<T, V> v;
    if (t >= 0) {
        if (t < len) v.load((const T*)p.x + b * p.s_x[0] + t * p.s_x[1] + d);
        else v.zero();
    } else if (p.state && t >= -(K - 1)) {
        v.load((const T*)p.state + b * p.s_st[0] + (t + K - 1) * p.s_st[1] + d);
    } else {
        v.zero();
    }
    return v;
}

constexpr int AHEAD = 8;                                         // tokens that a thread has under way

template <typename T, int K, int V> __global__ void __launch_bounds__(256) conv_fwd_kernel(const ConvParams p) {
    const int nv = p.D / V;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)p.B * p.runs * nv;
    if (i >= all) return;
    const int d = (int)(i % nv) * V, r = (int)(i / nv % p.runs), b = (int)(i / nv / p.runs), len = length_of(p, b);
    const int64_t t0 = (int64_t)r * p.run, t1 = min((int64_t)p.L, t0 + p.run);
    float w[K][V], bias[V], win[K][V];                           // win[k]: token t - K + 1 + k
    taps<T, K, V>(p, d, w, bias);
#pragma unroll
    for (int k = 1; k < K; ++k) {
        const Piece<T, V> x = token<T, K, V>(p, b, t0 - K + k, len, d);
#pragma unroll
        for (int v = 0; v < V; ++v) win[k][v] = DType<T>::to_f(x.e[v]);
    }
    T* const y = (T*)p.y + b * p.s_y[0] + d;
    for (int64_t t = t0; t < t1; t += AHEAD) {
        Piece<T, V> x[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (t + j < min(t1, (int64_t)len)) x[j].load((const T*)p.x + b * p.s_x[0] + (t + j) * p.s_x[1] + d);
            else x[j].zero();
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (t + j >= t1) break;
            Piece<T, V> out;
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int k = 0; k + 1 < K; ++k) win[k][v] = win[k + 1][v];
                win[K - 1][v] = DType<T>::to_f(x[j].e[v]);
                float s = bias[v];
#pragma unroll
                for (int k = 0; k < K; ++k) s = fmaf(w[k][v], win[k][v], s);
                if (p.silu) s *= sigmoidf_(s);
                out.e[v] = DType<T>::from_f(t + j < len ? s : 0.f);
            }
            out.store(y + (t + j) * p.s_y[1]);
        }
    }
    if (p.state_out && r == p.runs - 1) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) token<T, K, V>(p, b, (int64_t)len - (K - 1) + k, len, d).store((T*)p.state_out + b * p.s_out[0] + k * p.s_out[1] + d);
    }
}

// A block takes 32 V channels and walks runs of tokens, eight at a time; its threads' shares of dw and dbias stay in registers, are added in shared memory
// and left for conv_sum_kernel.  Where a gradient of the state is wanted, a sequence's first run begins K - 1 tokens ahead of it.
template <typename T, int K, int V> __global__ void __launch_bounds__(256) conv_bwd_kernel(const ConvParams p) {
    __shared__ float sh[8][32 * V];
    const int lane = threadIdx.x, row = threadIdx.y, nv = p.D / V;
    const int vec = blockIdx.x * 32 + lane;
    const bool in = vec < nv;
    const int d = (in ? vec : 0) * V;
    float w[K][V], bias[V], dw[K][V], db[V];
    taps<T, K, V>(p, d, w, bias);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        db[v] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) dw[k][v] = 0.f;
    }
    const int64_t all = (int64_t)p.B * p.runs;
    for (int64_t i = (int64_t)blockIdx.y * 8 + row; i < all && in; i += (int64_t)gridDim.y * 8) {
        const int r = (int)(i % p.runs), b = (int)(i / p.runs), len = length_of(p, b);
        const int64_t first = (int64_t)r * p.run, t1 = min((int64_t)p.L, first + p.run), t0 = r == 0 && p.d_state ? -(K - 1) : first;
        float win[K][V], dp[K][V];                               // dp[k]: dpre of token t - K + 1 + k
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const Piece<T, V> x = token<T, K, V>(p, b, t0 - K + k, len, d);
#pragma unroll
            for (int v = 0; v < V; ++v) { win[k][v] = DType<T>::to_f(x.e[v]); dp[k][v] = 0.f; }
        }
        for (int64_t t = t0; t < t1 + K - 1; t += 4) {
            Piece<T, V> xs[4], ds[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                xs[j] = token<T, K, V>(p, b, t + j, len, d);
                if (t + j >= 0 && t + j < len) ds[j].load((const T*)p.dy + b * p.s_dy[0] + (t + j) * p.s_dy[1] + d);
                else ds[j].zero();
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t tj = t + j, to = tj - (K - 1);     // the window of token `to` is complete with tj
                if (tj >= t1 + K - 1) break;
                const bool own = tj >= first && tj < t1;         // whose share of dw is this run's
                Piece<T, V> out;
#pragma unroll
                for (int v = 0; v < V; ++v) {
#pragma unroll
                    for (int k = 0; k + 1 < K; ++k) { win[k][v] = win[k + 1][v]; dp[k][v] = dp[k + 1][v]; }
                    win[K - 1][v] = DType<T>::to_f(xs[j].e[v]);
                    float g = DType<T>::to_f(ds[j].e[v]);
                    if (p.silu) {
                        float s = bias[v];
#pragma unroll
                        for (int k = 0; k < K; ++k) s = fmaf(w[k][v], win[k][v], s);
                        const float sg = sigmoidf_(s);
                        g = tj >= 0 && tj < len ? g * sg * fmaf(s, 1.f - sg, 1.f) : 0.f;
                    }
                    dp[K - 1][v] = g;
                    if (own) {
                        db[v] += g;
#pragma unroll
                        for (int k = 0; k < K; ++k) dw[k][v] = fmaf(g, win[k][v], dw[k][v]);
                    }
                    float o = 0.f;
#pragma unroll
                    for (int k = 0; k < K; ++k) o = fmaf(w[K - 1 - k][v], dp[k][v], o);
                    // what the state handed on gives back: its row k is token len - (K - 1) + k
                    if (p.d_out && to >= len - (K - 1) && to < len) o += DType<T>::to_f(((const T*)p.d_out)[((int64_t)b * (K - 1) + (to - len + K - 1)) * p.D + d + v]);
                    out.e[v] = DType<T>::from_f(to < len ? o : 0.f);
                }
                if (to >= t0) {
                    if (to >= 0) out.store((T*)p.dx + ((int64_t)b * p.L + to) * p.D + d);
                    else out.store((T*)p.d_state + ((int64_t)b * (K - 1) + to + K - 1) * p.D + d);
                }
            }
        }
    }
    // shares of the block's eight rows of threads
#pragma unroll
    for (int k = 0; k <= K; ++k) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) sh[row][lane * V + v] = k < K ? dw[k < K ? k : 0][v] : db[v];
        __syncthreads();
        const int c = row * 32 + lane;
        if (c < 32 * V && blockIdx.x * 32 * V + c < p.D) {
            float s = 0.f;
#pragma unroll
            for (int r = 0; r < 8; ++r) s += sh[r][c];
            p.partial[((int64_t)blockIdx.y * (K + 1) + k) * p.D + blockIdx.x * 32 * V + c] = s;
        }
    }
}

// the blocks' shares in their order; 32 channels x 8 warps, a warp adds every eighth share
template <typename T, int K> __global__ void __launch_bounds__(256) conv_sum_kernel(const ConvParams p) {
    __shared__ float sh[8][32];
    const int lane = threadIdx.x, row = threadIdx.y, d = blockIdx.x * 32 + lane, k = blockIdx.y;
    pdl_wait();
    float s = 0.f;
    if (d < p.D) for (int i = row; i < p.blocks; i += 8) s += p.partial[((int64_t)i * (K + 1) + k) * p.D + d];
    sh[row][lane] = s;
    __syncthreads();
    if (row == 0 && d < p.D) {
#pragma unroll
        for (int r = 1; r < 8; ++r) s += sh[r][lane];
        void* to = k < K ? p.dw : p.dbias;
        const int64_t at = k < K ? (int64_t)d * K + k : d;
        if (!to) return;
        if (p.w_f32) ((float*)to)[at] = s;
        else ((T*)to)[at] = DType<T>::from_f(s);
    }
}

template <typename T, int K> __global__ void __launch_bounds__(128) conv_step_kernel(const ConvParams p) {
    const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (i >= (int64_t)p.B * p.D) return;
    const int d = (int)(i % p.D), b = (int)(i / p.D);
    T* const st = (T*)p.state_out + b * p.s_out[0] + d;
    T row[K];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) row[k] = st[k * p.s_out[1]];
    row[K - 1] = ((const T*)p.x)[b * p.s_x[0] + d];
    float s = p.bias ? weight<T>(p.bias, d, p.w_f32) : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) s = fmaf(weight<T>(p.w, (int64_t)d * K + k, p.w_f32), DType<T>::to_f(row[k]), s);
    if (p.silu) s *= sigmoidf_(s);
    ((T*)p.y)[b * p.s_y[0] + d] = DType<T>::from_f(s);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) st[k * p.s_out[1]] = row[k + 1];
}

bool aligned(const void* q, const int64_t* s, int count, int bytes, int size) {
    if (!q) return true;
    if ((uintptr_t)q % bytes) return false;
    for (int i = 0; i < count; ++i) if (s[i] * size % bytes) return false;
    return true;
}

template <typename T, int K> int fwd_launch(ConvParams& p, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int size = (int)sizeof(T);
    const bool whole = p.D % V == 0 && aligned(p.x, p.s_x, 2, 16, size) && aligned(p.y, p.s_y, 2, 16, size) && aligned(p.state, p.s_st, 2, 16, size) &&
                       aligned(p.state_out, p.s_out, 2, 16, size);
    const int64_t nv = whole ? p.D / V : p.D;
    // runs of 32 tokens, or shorter ones down to 8 where that would be less than 512 threads an SM
    p.run = 32;
    while (p.run > AHEAD && (int64_t)p.B * ((p.L + p.run - 1) / p.run) * nv < (int64_t)device_sms() * 512) p.run /= 2;
    p.runs = p.L ? (p.L + p.run - 1) / p.run : 1;
    const int64_t grid = ((int64_t)p.B * p.runs * nv + 255) / 256;
    if (grid >= (1ll << 31)) return VIG_ERR_SHAPE;
    if (whole) conv_fwd_kernel<T, K, V><<<(unsigned)grid, 256, 0, s>>>(p);
    else conv_fwd_kernel<T, K, 1><<<(unsigned)grid, 256, 0, s>>>(p);
    return (int)cudaGetLastError();
}

// blocks of the backward along the tokens, whose shares the workspace holds
int bwd_blocks(int64_t B, int64_t L, int D) {
    const int64_t most = ((int64_t)device_sms() * 6 + (D + 127) / 128 - 1) / ((D + 127) / 128), runs = B * (L / 8 + 1);
    return (int)(runs < most ? runs : most);
}

template <typename T, int K> int bwd_launch(ConvParams& p, cudaStream_t s) {
    constexpr int V = 4;
    const int size = (int)sizeof(T), bytes = V * size;
    const int64_t rows[1] = {p.D};
    const bool whole = p.D % V == 0 && aligned(p.x, p.s_x, 2, bytes, size) && aligned(p.dy, p.s_dy, 2, bytes, size) && aligned(p.state, p.s_st, 2, bytes, size) &&
                       aligned(p.dx, rows, 1, bytes, size) && aligned(p.d_state, rows, 1, bytes, size);
    const int width = whole ? 32 * V : 32, cols = (p.D + width - 1) / width;
    p.run = 64;
    while (p.run > 8 && (int64_t)p.B * ((p.L + p.run - 1) / p.run) < 8ll * p.blocks) p.run /= 2;
    p.runs = p.L ? (p.L + p.run - 1) / p.run : 1;
    const dim3 grid(cols, p.blocks), block(32, 8);
    if (whole) conv_bwd_kernel<T, K, V><<<grid, block, 0, s>>>(p);
    else conv_bwd_kernel<T, K, 1><<<grid, block, 0, s>>>(p);
    if (const cudaError_t e = cudaGetLastError()) return (int)e;
    return (int)launch_next(conv_sum_kernel<T, K>, dim3((p.D + 31) / 32, K + 1), block, 0, s, p);
}

template <typename T, int K> int step_launch(ConvParams& p, cudaStream_t s) {
    conv_step_kernel<T, K><<<(unsigned)(((int64_t)p.B * p.D + 127) / 128), 128, 0, s>>>(p);
    return (int)cudaGetLastError();
}

enum { FWD, BWD, STEP };
template <int WHAT, typename T, int K> int launch(ConvParams& p, cudaStream_t s) {
    if constexpr (WHAT == FWD) return fwd_launch<T, K>(p, s);
    else if constexpr (WHAT == BWD) return bwd_launch<T, K>(p, s);
    else return step_launch<T, K>(p, s);
}
template <int WHAT, typename T> int by_taps(ConvParams& p, int K, cudaStream_t s) {
    switch (K) {
        case 1: return launch<WHAT, T, 1>(p, s);
        case 2: return launch<WHAT, T, 2>(p, s);
        case 3: return launch<WHAT, T, 3>(p, s);
        case 4: return launch<WHAT, T, 4>(p, s);
        case 5: return launch<WHAT, T, 5>(p, s);
        case 6: return launch<WHAT, T, 6>(p, s);
        case 7: return launch<WHAT, T, 7>(p, s);
        default: return launch<WHAT, T, 8>(p, s);
    }
}
template <int WHAT> int by_type(ConvParams& p, int K, int dtype, cudaStream_t s) {
    switch (dtype) {
        case VIG_DTYPE_F32: return by_taps<WHAT, float>(p, K, s);
        case VIG_DTYPE_BF16: return by_taps<WHAT, __nv_bfloat16>(p, K, s);
        default: return by_taps<WHAT, __half>(p, K, s);
    }
}

int check(int B, int L, int D, int K, int w_dtype, int dtype) {
    if (dtype < VIG_DTYPE_F32 || dtype > VIG_DTYPE_F16 || (w_dtype != dtype && w_dtype != VIG_DTYPE_F32)) return VIG_ERR_DTYPE;
    if (B < 0 || L < 0 || D < 0 || K < 1 || K > MAX_K || (int64_t)B * D >= (1ll << 31) || D >= (1 << 28) || L >= (1 << 30)) return VIG_ERR_SHAPE;
    return VIG_OK;
}
void strides(int64_t* to, const int64_t* from, int64_t rows, int64_t D) { to[0] = from ? from[0] : rows * D; to[1] = from ? from[1] : D; }

}  // namespace
}  // namespace vig

using namespace vig;

extern "C" int vig_causal_conv_fwd(const void* x, const void* w, int w_dtype, const void* bias, const void* state, void* y, void* state_out, const int32_t* lengths,
                                   int B, int L, int D, int K, const int64_t* strides_x, const int64_t* strides_y, const int64_t* strides_state,
                                   const int64_t* strides_state_out, int silu, int dtype, void* stream) {
    if (const int e = check(B, L, D, K, w_dtype, dtype)) return e;
    if (!B || !D || (!L && (!state_out || K == 1))) return VIG_OK;
    if (!w || (L && (!x || !y))) return VIG_ERR_NULL;
    ConvParams p{};
    p.x = x; p.w = w; p.bias = bias; p.state = K > 1 ? state : nullptr; p.y = y; p.state_out = K > 1 ? state_out : nullptr; p.lengths = lengths;
    strides(p.s_x, strides_x, L, D); strides(p.s_y, strides_y, L, D); strides(p.s_st, strides_state, K - 1, D); strides(p.s_out, strides_state_out, K - 1, D);
    p.B = B; p.L = L; p.D = D; p.w_f32 = w_dtype == VIG_DTYPE_F32; p.w_whole = ((uintptr_t)w | (uintptr_t)bias) % 16 == 0; p.silu = silu;
    return by_type<FWD>(p, K, dtype, (cudaStream_t)stream);
}

extern "C" size_t vig_causal_conv_bwd_workspace_bytes(int B, int L, int D, int K) {
    return B > 0 && L >= 0 && D > 0 && K > 0 ? (size_t)bwd_blocks(B, L, D) * (K + 1) * D * sizeof(float) : 0;
}

extern "C" int vig_causal_conv_bwd(const void* x, const void* w, int w_dtype, const void* bias, const void* state, const void* d_y, const void* d_state_out,
                                   const int32_t* lengths, void* d_x, void* d_w, void* d_bias, void* d_state, int B, int L, int D, int K, const int64_t* strides_x,
                                   const int64_t* strides_state, const int64_t* strides_dy, int silu, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int e = check(B, L, D, K, w_dtype, dtype)) return e;
    if (!B || !D) return VIG_OK;
    if (!w || !d_w || (L && (!x || !d_y || !d_x))) return VIG_ERR_NULL;
    if (!workspace || workspace_bytes < vig_causal_conv_bwd_workspace_bytes(B, L, D, K)) return VIG_ERR_WORKSPACE;
    ConvParams p{};
    p.x = x; p.w = w; p.bias = bias; p.state = K > 1 ? state : nullptr; p.dy = d_y; p.d_out = K > 1 ? d_state_out : nullptr; p.lengths = lengths;
    p.dx = d_x; p.dw = d_w; p.dbias = d_bias; p.d_state = K > 1 ? d_state : nullptr; p.partial = (float*)workspace;
    strides(p.s_x, strides_x, L, D); strides(p.s_st, strides_state, K - 1, D); strides(p.s_dy, strides_dy, L, D);
    p.B = B; p.L = L; p.D = D; p.w_f32 = w_dtype == VIG_DTYPE_F32; p.w_whole = ((uintptr_t)w | (uintptr_t)bias) % 16 == 0; p.silu = silu;
    p.blocks = bwd_blocks(B, L, D);
    return by_type<BWD>(p, K, dtype, (cudaStream_t)stream);
}

extern "C" int vig_causal_conv_step(const void* x, int64_t ldx, void* state, const int64_t* strides_state, const void* w, int w_dtype, const void* bias, void* y, int64_t ldy,
                                    int B, int D, int K, int silu, int dtype, void* stream) {
    if (const int e = check(B, 1, D, K, w_dtype, dtype)) return e;
    if (!B || !D) return VIG_OK;
    if (!x || !w || !y || (K > 1 && !state)) return VIG_ERR_NULL;
    ConvParams p{};
    p.x = x; p.w = w; p.bias = bias; p.y = y; p.state_out = state;
    p.s_x[0] = ldx; p.s_y[0] = ldy;
    strides(p.s_out, strides_state, K - 1, D);
    p.B = B; p.L = 1; p.D = D; p.w_f32 = w_dtype == VIG_DTYPE_F32; p.silu = silu;
    return by_type<STEP>(p, K, dtype, (cudaStream_t)stream);
}
