// Short causal convolution, a channel at a time: pre_t = bias + sum_k w_k x_{t-K+1+k}, y = silu(pre) or pre.
// Backward: dpre = dy act'(pre) with pre computed again,  dx_t = sum_k w_k dpre_{t+K-1-k},  dw_k = sum_t dpre_t x_{t-K+1+k},  dbias = sum_t dpre_t.
//
// Bound by memory: x in, y out; backward x and dy in, dx out.  A thread walks a run of tokens of a few neighbouring channels and keeps the
// window in registers, so that each value is read once and, at the border of two runs, K - 1 times more out of the cache.  16 x 4096 x 768 bf16, 4 taps: forward
// 50 us (4.0 TB/s; 25 instructions a value, issue slots at 71 %), backward 136 (2.2 TB/s; 51 instructions a value, issue slots at 57 % with 16 warps an SM; at the 128
// registers that these allow, 4 taps of 4 channels in 16 bits spill 120 bytes).
#include <type_traits>
#include "tc_common.cuh"

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
        else if constexpr (V * sizeof(T) == 4) { const uint32_t w = *(const uint32_t*)q; memcpy(e, &w, 4); }
        else {
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] = q[i];
        }
    }
    __device__ void store(T* q) const {
        if constexpr (V * sizeof(T) == 16) { uint4 w; memcpy(&w, e, 16); *(uint4*)q = w; }
        else if constexpr (V * sizeof(T) == 8) { uint2 w; memcpy(&w, e, 8); *(uint2*)q = w; }
        else if constexpr (V * sizeof(T) == 4) { uint32_t w; memcpy(&w, e, 4); *(uint32_t*)q = w; }
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

// the taps and biases of V neighbouring channels: those in fp32 in whole pieces of 16 bytes, since they lie one behind the other; those in 16 bits, whose V biases
// are 8 bytes, one at a time
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

__device__ __forceinline__ float sigmoid_of(float x) { return tc::rcp(1.f + tc::ex2(-x * tc::LOG2E)); }

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

// Tokens come in blocks of U: the window X holds the K - 1 before a block and the block itself, so that every index is known to the compiler and nothing is moved
// but K - 1 values a block.  Blocks to come are on their way to shared memory, STAGES of them, every thread's values into slots of its own: registers
// would hold one and leave room for half the threads (16384 x 768 38 us, training 16 x 4096 x 768 362).  Single values of 16 bits, which no asynchronous copy
// takes, go through registers.
constexpr int STAGES = 4;

template <typename T, int V, int U, int ROWS, int THREADS> struct Ahead {
    static constexpr int BYTES = V * (int)sizeof(T);
    static constexpr bool ASYNC = BYTES >= 4;
    static constexpr int ROOM = ASYNC ? STAGES * ROWS * U * THREADS * BYTES : 0;
    char* slots;                                                 // the thread's
    __device__ __forceinline__ char* slot(int stage, int row, int j) const { return slots + ((stage * ROWS + row) * U + j) * THREADS * BYTES; }
    __device__ __forceinline__ void bring(int stage, int row, int j, const T* from, bool there) const {
        if constexpr (ASYNC) {
            const uint32_t to = (uint32_t)__cvta_generic_to_shared(slot(stage, row, j));
            const int bytes = there ? BYTES : 0;                 // the rest of the slot becomes zeros
            if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
            else if constexpr (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
            else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
        }
    }
    __device__ __forceinline__ void done() const { asm volatile("cp.async.commit_group;" ::: "memory"); }
    __device__ __forceinline__ void wait() const { asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory"); }
    __device__ __forceinline__ void take(int stage, int row, int j, const T* from, bool there, float* f) const {
        Piece<T, V> v;
        if constexpr (ASYNC) v.load((const T*)slot(stage, row, j));
        else if (there) v.load(from);
        else v.zero();
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = DType<T>::to_f(v.e[e]);
    }
};

template <typename T, int K, int V, int U> __global__ void __launch_bounds__(256) conv_fwd_kernel(const ConvParams p) {
    extern __shared__ __align__(16) char ring[];
    const Ahead<T, V, U, 1, 256> ahead{ring + threadIdx.x * V * (int)sizeof(T)};
    const int nv = p.D / V;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)p.B * p.runs * nv;
    if (i >= all) return;
    const int d = (int)(i % nv) * V, r = (int)(i / nv % p.runs), b = (int)(i / nv / p.runs), len = length_of(p, b);
    const int t0 = r * p.run, t1 = min(p.L, t0 + p.run), stop = min(t1, len);
    const T* const x = (const T*)p.x + b * p.s_x[0] + d;
    T* const y = (T*)p.y + b * p.s_y[0] + d;
    const int64_t sx = p.s_x[1], sy = p.s_y[1];
    auto bring = [&](int t, int stage) {
#pragma unroll
        for (int j = 0; j < U; ++j) ahead.bring(stage, 0, j, t + j < stop ? x + (t + j) * sx : x, t + j < stop);
        ahead.done();
    };
#pragma unroll
    for (int k = 0; k < STAGES; ++k) bring(t0 + k * U, k);
    float w[K][V], bias[V], X[K - 1 + U][V];
    taps<T, K, V>(p, d, w, bias);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        const Piece<T, V> v = token<T, K, V>(p, b, (int64_t)t0 - (K - 1) + k, len, d);
#pragma unroll
        for (int e = 0; e < V; ++e) X[k][e] = DType<T>::to_f(v.e[e]);
    }
    int stage = 0;
    for (int t = t0; t < t1; t += U, stage = stage + 1 < STAGES ? stage + 1 : 0) {
        ahead.wait();
#pragma unroll
        for (int j = 0; j < U; ++j) ahead.take(stage, 0, j, x + (t + j) * sx, t + j < stop, X[K - 1 + j]);
        bring(t + STAGES * U, stage);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (t + j >= t1) break;
            Piece<T, V> out;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float s = bias[e];
#pragma unroll
                for (int k = 0; k < K; ++k) s = fmaf(w[k][e], X[j + k][e], s);
                if (p.silu) s *= sigmoid_of(s);
                out.e[e] = DType<T>::from_f(t + j < len ? s : 0.f);
            }
            out.store(y + (t + j) * sy);
        }
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) X[k][e] = X[U + k][e];
    }
    if (p.state_out && r == p.runs - 1) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) token<T, K, V>(p, b, (int64_t)len - (K - 1) + k, len, d).store((T*)p.state_out + b * p.s_out[0] + k * p.s_out[1] + d);
    }
}

// A block of threads takes 32 V channels and walks runs of tokens, ROWS at a time; its threads' shares of dw and dbias stay in registers, are added in shared memory
// and left for conv_sum_kernel.  Where a gradient of the state is wanted, a sequence's first run begins K - 1 tokens ahead of it.  A run's last tokens
// want dpre of the K - 1 behind it; blocks of U tokens all inside run and sequence go without the questions that this and the ends ask.
constexpr int ROWS = 8;

template <typename T, int K, int V, int U> __global__ void __launch_bounds__(32 * ROWS, 2) conv_bwd_kernel(const ConvParams p) {
    extern __shared__ __align__(16) char ring[];                 // at the end [ROWS][32 V] shares
    const Ahead<T, V, U, 2, 32 * ROWS> ahead{ring + (threadIdx.y * 32 + threadIdx.x) * V * (int)sizeof(T)};
    const int lane = threadIdx.x, row = threadIdx.y, nv = p.D / V;
    const int vec = blockIdx.x * 32 + lane;
    const bool in = vec < nv;
    const int d = (in ? vec : 0) * V;
    float w[K][V], bias[V], dw[K][V], db[V];
    taps<T, K, V>(p, d, w, bias);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        db[e] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) dw[k][e] = 0.f;
    }
    const int64_t all = (int64_t)p.B * p.runs;
    for (int64_t i = (int64_t)blockIdx.y * ROWS + row; i < all && in; i += (int64_t)gridDim.y * ROWS) {
        const int r = (int)(i % p.runs), b = (int)(i / p.runs), len = length_of(p, b);
        const int first = r * p.run, t1 = min(p.L, first + p.run), t0 = r == 0 && p.d_state ? -(K - 1) : first, end = t1 + K - 1;
        const int stop = min(t1, len), calm = stop - (p.d_out ? K - 1 : 0);   // tokens of the run that count; up to where a block asks nothing
        const T *const x = (const T*)p.x + b * p.s_x[0] + d, *const dy = (const T*)p.dy + b * p.s_dy[0] + d;
        const T* const st = p.state ? (const T*)p.state + b * p.s_st[0] + d : nullptr;
        T* const dx = (T*)p.dx + (int64_t)b * p.L * p.D + d;
        const int64_t sx = p.s_x[1], sd = p.s_dy[1], ss = p.s_st[1];
        float X[K - 1 + U][V], P[K - 1 + U][V];                  // tokens; their dpre
        // where token t is, and whether it is there at all
        auto place = [&](int t, bool& there) {
            there = t < 0 ? st && t >= -(K - 1) : t < len;
            return !there ? x : t < 0 ? st + (t + K - 1) * ss : x + t * sx;
        };
        auto bring = [&](int t, int stage) {
#pragma unroll
            for (int j = 0; j < U; ++j) {
                bool there;
                const T* from = place(t + j, there);
                there = there && t + j < end;
                ahead.bring(stage, 0, j, there ? from : x, there);
                const bool inside = t + j >= 0 && t + j < len && t + j < end;
                ahead.bring(stage, 1, j, inside ? dy + (t + j) * sd : dy, inside);
            }
            ahead.done();
        };
#pragma unroll
        for (int k = 0; k < STAGES; ++k) bring(t0 + k * U, k);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            const Piece<T, V> v = token<T, K, V>(p, b, (int64_t)t0 - (K - 1) + k, len, d);
#pragma unroll
            for (int e = 0; e < V; ++e) { X[k][e] = DType<T>::to_f(v.e[e]); P[k][e] = 0.f; }
        }
        auto block = [&](int t, auto quiet) {
            constexpr bool Q = decltype(quiet)::value;
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int tj = t + j;
                    float s = bias[e];
#pragma unroll
                    for (int k = 0; k < K; ++k) s = fmaf(w[k][e], X[j + k][e], s);
                    const float sg = sigmoid_of(s), own = P[K - 1 + j][e], act = own * sg * fmaf(s, 1.f - sg, 1.f);
                    float g = p.silu ? act : own;
                    if (!Q && (tj < 0 || tj >= len)) g = 0.f;
                    P[K - 1 + j][e] = g;
                    if (Q || (tj >= first && tj < stop)) {       // whose share of dw is this run's
                        db[e] += g;
#pragma unroll
                        for (int k = 0; k < K; ++k) dw[k][e] = fmaf(g, X[j + k][e], dw[k][e]);
                    }
                }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int to = t + j - (K - 1);                  // the window of token `to` is complete with t + j
                if (to < t0 || (!Q && to >= t1)) continue;
                Piece<T, V> out;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float o = 0.f;
#pragma unroll
                    for (int k = 0; k < K; ++k) o = fmaf(w[K - 1 - k][e], P[j + k][e], o);
                    if (!Q) {
                        // what the state handed on gives back: its row k is token len - (K - 1) + k
                        if (p.d_out && to >= len - (K - 1) && to < len) o += DType<T>::to_f(((const T*)p.d_out)[((int64_t)b * (K - 1) + (to - len + K - 1)) * p.D + d + e]);
                        if (to >= len) o = 0.f;
                    }
                    out.e[e] = DType<T>::from_f(o);
                }
                if (Q || to >= 0) out.store(dx + (int64_t)to * p.D);
                else out.store((T*)p.d_state + ((int64_t)b * (K - 1) + to + K - 1) * p.D + d);
            }
        };
        int stage = 0;
        for (int t = t0; t < end; t += U, stage = stage + 1 < STAGES ? stage + 1 : 0) {
            ahead.wait();
#pragma unroll
            for (int j = 0; j < U; ++j) {
                bool there = true;
                const T* from = Ahead<T, V, U, 2, 32 * ROWS>::ASYNC ? x : place(t + j, there);
                ahead.take(stage, 0, j, from, there, X[K - 1 + j]);
                ahead.take(stage, 1, j, dy + (t + j) * sd, t + j >= 0 && t + j < len, P[K - 1 + j]);
            }
            bring(t + STAGES * U, stage);
            if (t >= K - 1 && t + U <= calm) block(t, std::true_type{});
            else block(t, std::false_type{});
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) { X[k][e] = X[U + k][e]; P[k][e] = P[U + k][e]; }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    // shares of the block's rows of threads
    float (*const sh)[32 * V] = (float (*)[32 * V])ring;
#pragma unroll
    for (int k = 0; k <= K; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) sh[row][lane * V + e] = k < K ? dw[k < K ? k : 0][e] : db[e];
        __syncthreads();
        for (int c = row * 32 + lane; c < 32 * V && blockIdx.x * 32 * V + c < p.D; c += 32 * ROWS) {
            float s = 0.f;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) s += sh[r][c];
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
    if (p.silu) s *= sigmoid_of(s);
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

// tokens of a run where a sequence has about `runs` of them: whole blocks, two at least
template <int U> int run_of(int L, int64_t runs) {
    const int64_t run = runs > 0 ? (L + runs - 1) / runs : L;
    return (int)(run <= 2 * U ? 2 * U : (run + U - 1) / U * U);
}

template <typename T, int K> int fwd_launch(ConvParams& p, cudaStream_t s) {
    constexpr int V = 4, U = 4;
    const int size = (int)sizeof(T), bytes = V * size;
    const bool whole = p.D % V == 0 && aligned(p.x, p.s_x, 2, bytes, size) && aligned(p.y, p.s_y, 2, bytes, size) && aligned(p.state, p.s_st, 2, bytes, size) &&
                       aligned(p.state_out, p.s_out, 2, bytes, size);
    const int64_t nv = whole ? p.D / V : p.D;
    // runs as long as they may be where every thread that finds room has one: each begins with taps, a window and a wait
    p.run = run_of<U>(p.L, (int64_t)device_sms() * 768 / (p.B * nv));
    p.runs = p.L ? (p.L + p.run - 1) / p.run : 1;
    const int64_t grid = ((int64_t)p.B * p.runs * nv + 255) / 256;
    if (grid >= (1ll << 31)) return VIG_ERR_SHAPE;
    const auto kernel = whole ? conv_fwd_kernel<T, K, V, U> : conv_fwd_kernel<T, K, 1, U>;
    const int smem = whole ? Ahead<T, V, U, 1, 256>::ROOM : Ahead<T, 1, U, 1, 256>::ROOM;
    if (const cudaError_t e = tc::ensure_smem_attr((const void*)kernel, smem)) return (int)e;
    kernel<<<(unsigned)grid, 256, smem, s>>>(p);
    return (int)cudaGetLastError();
}

// blocks of the backward along the tokens, whose shares the workspace holds
int bwd_blocks(int64_t B, int64_t L, int D) {
    const int64_t cols = (D + 127) / 128, most = ((int64_t)device_sms() * 4 + cols - 1) / cols, runs = B * (L / 8 + 1);
    return (int)(runs < most ? runs : most);
}

template <typename T, int K> int bwd_launch(ConvParams& p, cudaStream_t s) {
    constexpr int V = K <= 4 ? 4 : 2, U = 4;
    const int size = (int)sizeof(T), bytes = V * size;
    const int64_t rows[1] = {p.D};
    const bool whole = p.D % V == 0 && aligned(p.x, p.s_x, 2, bytes, size) && aligned(p.dy, p.s_dy, 2, bytes, size) && aligned(p.state, p.s_st, 2, bytes, size) &&
                       aligned(p.dx, rows, 1, bytes, size) && aligned(p.d_state, rows, 1, bytes, size);
    const int width = whole ? 32 * V : 32, cols = (p.D + width - 1) / width;
    p.run = run_of<U>(p.L, (int64_t)ROWS * p.blocks / p.B);
    p.runs = p.L ? (p.L + p.run - 1) / p.run : 1;
    const dim3 grid(cols, p.blocks), block(32, ROWS);
    const auto kernel = whole ? conv_bwd_kernel<T, K, V, U> : conv_bwd_kernel<T, K, 1, U>;
    constexpr int shares = ROWS * 32 * 4;                        // a channel's
    const int smem = whole ? max(Ahead<T, V, U, 2, 32 * ROWS>::ROOM, V * shares) : max(Ahead<T, 1, U, 2, 32 * ROWS>::ROOM, shares);
    if (const cudaError_t e = tc::ensure_smem_attr((const void*)kernel, smem)) return (int)e;
    kernel<<<grid, block, smem, s>>>(p);
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
