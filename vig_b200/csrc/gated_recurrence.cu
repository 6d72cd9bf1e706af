// Gated linear recurrence with one state per channel, h_t = a_t h_{t-1} + x_t, along either direction of a sequence: forward, all
// gradients, and the one-token form (the same call with L = 1 and the state updated in place).
//
// a_t = exp(g_t) from log-gates, or sigmoid(z_t)^(1/n) = exp(logsigmoid(z_t)/n) from raw logits z with n = gate_logit_normalizer.
// Gradients: u_t = a_t (dh_t + u_{t+1}), the same recurrence from the other end;  dx_t = dh_t + u_{t+1},  dg_t = u_t h_{t-1},
// dz_t = dg_t (1 - sigmoid(z_t)) / n,  dh_{-1} = u_0.  States, decays and sums are fp32; h is rounded once, to x's type.  The h_{t-1} of
// the gate gradients: fp32 calls read h.  In 16 bits the forward of a training step leaves the fp32 state in front of every eight tokens
// (counted from the end of its scan, half a byte a value), and the backward reads x and walks each eight of them again: h as it was rounded
// costs the gate gradient a third of its precision (2.3e-3 from 64 bits in bf16 instead of 1.7e-3, fp16 2.9e-4 instead of 2.1e-4).
// Bound by memory where sequences are many (3 tensors forward: x, g in, h out; 5 backward: g, dh, h or x in, dx, dg out), and by the MUFU unit
// beside it: a raw logit is two of its instructions (three backward) and seven multiply-adds, half of its rate at the copy bandwidth.  Calls on other
// inputs and outputs than the last, 16 x 4096 x 768 bf16 from raw logits: forward 62 us (4.9 TB/s), 66 with states, backward 111 us (4.8 TB/s), 74 and 121
// in a loop of seconds, where the power limit takes a tenth of the clock; 16 x 2048 x 768 fp32 54 and 87 us (5.6 and 5.8 TB/s); 1 x 16384 x 768 bf16, 48
// strips on 384 CTAs, 29 and 47 us.
// Three forms, by the rule in rec_launch: rows of 16-byte pieces through shared memory (rec_tile_kernel), rows of any alignment through
// registers (rec_strip_kernel), few tokens a thread at a time (rec_few_kernel).
#include <string.h>
#include <type_traits>
#include "tc_common.cuh"

namespace vig {

struct RecParams {
    const void *x, *g;              // backward: x is dh
    const void* h_in;               // backward: the forward's h; with `walk` its x
    float* states;                  // [B][(L - 1) / 8][D]: state in front of eight tokens, the scan's last eight (but none in front of its first)
    int keep, walk;                 // forward: write them; backward: h_{t-1} from them and x instead of from h
    const float* s0;                // state that enters the scan: the initial state; backward: d(final)
    const float* h0;                // backward: the forward's initial state
    void* out;                      // h; backward: dx
    void* out_g;                    // backward: dg
    float* s_end;                   // final state; backward: d(initial state)
    int64_t sx[2], sg[2], sh[2], so[2], sog[2];   // (b, l) element strides
    int64_t ld_s0, ld_end;
    int B, L, D;
    float inv_norm;                 // > 0: g holds raw logits
    int from_end;                   // the scan at hand starts at token L-1
    int32_t* status;
    // Eight tokens that share a state are counted in the order of the backward: tokens 8 j to 8 j + 7 from the end of the forward's scan.
    __host__ __device__ int64_t groups() const { return (L - 1) / 8; }
};
constexpr int GROUP = 8;

// The exponential of base two of the MUFU unit, without the scaling that denormal arguments and results would take (decays that small make
// no difference to a sum in fp32).
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
constexpr float LOG2E = 1.4426950408889634f;

// two values at a time where there are two
template <int V> __device__ __forceinline__ void fma_v(float* d, const float* a, const float* b, const float* c) {
    if constexpr (V == 2)
        asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
            : "=f"(d[0]), "=f"(d[1]) : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]), "f"(c[0]), "f"(c[1]));
    else
        d[0] = fmaf(a[0], b[0], c[0]);
}
template <int V> __device__ __forceinline__ void add_v(float* d, const float* a, const float* b) {
    if constexpr (V == 2)
        asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
            : "=f"(d[0]), "=f"(d[1]) : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]));
    else
        d[0] = a[0] + b[0];
}
template <int V> __device__ __forceinline__ void mul_v(float* d, const float* a, const float* b) {
    if constexpr (V == 2)
        asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
            : "=f"(d[0]), "=f"(d[1]) : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]));
    else
        d[0] = a[0] * b[0];
}

// log2(1 + e) = e P(e) for e of 0 to 1, P fitted to the least relative error: 1.4e-6 with 7 terms (16-bit types), 2e-7 with 9 (fp32).  Relative,
// because a long memory is a small e: the logarithm of the MUFU unit is right to 2^-22 absolute, which at a logit of 9 is 1e-3 of the rate at
// which the state decays.  It takes as long (the unit is as busy as the multiply-adds: 16 x 4096 x 768 bf16 61 / 95 us with it, 60 / 96 with P, replays, backward from h).
template <typename T, int W> __device__ __forceinline__ void log2_1p(float* y, const float* e) {
    constexpr int N = sizeof(T) == 4 ? 9 : 7;
    const float c[N] = {1.44269323f, -0.721159458f, 0.477668375f, -0.339089006f, 0.215284511f, -0.0957975239f, 0.0204011761f};
    const float d[9] = {1.44269502f, -0.721340179f, 0.480692953f, -0.358408481f, 0.275641412f, -0.197118953f, 0.112856172f, -0.0425670482f, 0.00754917832f};
    float q[W];
#pragma unroll
    for (int w = 0; w < W; ++w) q[w] = sizeof(T) == 4 ? d[N - 1] : c[N - 1];
#pragma unroll
    for (int k = N - 2; k >= 0; --k) {
        const float ck[2] = {sizeof(T) == 4 ? d[k] : c[k], sizeof(T) == 4 ? d[k] : c[k]};
        fma_v<W>(q, q, e, ck);
    }
    mul_v<W>(y, q, e);
}

// Decays of V tokens' values g, and with REST also d logsigmoid(z) / dz = sigmoid(-z): one MUFU instruction for a log-gate (fp32: the exact
// function), two for a raw logit and one for REST.
template <typename T, bool LOGITS, bool REST, int V> __device__ __forceinline__ void decays(const float* g, float inv_norm, float* a, float* rest) {
    if constexpr (!LOGITS) {
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] = sizeof(T) == 4 ? expf(g[v]) : ex2(g[v] * LOG2E);
    } else {
        constexpr int W = V > 1 ? 2 : 1;
        const float l2e[2] = {LOG2E, LOG2E}, minus[2] = {-1.f, -1.f}, inv[2] = {inv_norm, inv_norm};
#pragma unroll
        for (int v = 0; v < V; v += W) {
            float z[W], e[W], t[W];
            mul_v<W>(z, g + v, l2e);
#pragma unroll
            for (int w = 0; w < W; ++w) { e[w] = ex2(-fabsf(z[w])); t[w] = fminf(z[w], 0.f); }
            log2_1p<T, W>(e, e);
            fma_v<W>(t, e, minus, t);                            // log2 of the sigmoid: min(z, 0) - log2(1 + 2^-|z|)
            mul_v<W>(e, t, inv);
#pragma unroll
            for (int w = 0; w < W; ++w) a[v + w] = ex2(e[w]);
            if (REST) {
                fma_v<W>(t, z, minus, t);
#pragma unroll
                for (int w = 0; w < W; ++w) rest[v + w] = ex2(fminf(t[w], 0.f));         // (a logit of -inf: -inf + inf, for 0)
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------
// Few tokens: a thread owns V channels (one, or 16 bytes of them; the backward of 16 bits 4, for it holds eight tokens' decays and states) and
// walks their tokens, the loads of up to four or eight tokens under way together.
template <typename T, bool BWD> constexpr int few_v = (BWD && sizeof(T) == 2 ? 4 : 16) / (int)sizeof(T);
template <typename T, int V> struct Few {
    alignas(V * sizeof(T)) T e[V];
    __device__ void load(const T* p) {
        if constexpr (V * sizeof(T) == 16) *(uint4*)e = *(const uint4*)p;
        else if constexpr (V > 1) *(uint32_t*)e = *(const uint32_t*)p;
        else e[0] = *p;
    }
    __device__ void get(float* f) const {
#pragma unroll
        for (int v = 0; v < V; ++v) f[v] = DType<T>::to_f(e[v]);
    }
    static __device__ void store(T* p, const float* f) {
        Few o;
#pragma unroll
        for (int v = 0; v < V; ++v) o.e[v] = DType<T>::from_f(f[v]);
        if constexpr (V * sizeof(T) == 16) *(uint4*)p = *(const uint4*)o.e;
        else if constexpr (V > 1) *(uint32_t*)p = *(const uint32_t*)o.e;
        else *p = o.e[0];
    }
};
template <int V> __device__ __forceinline__ void state_in(float* s, const float* p) {
    if constexpr (V == 2) {
        *(float2*)s = *(const float2*)p;
    } else if constexpr (V > 1) {
#pragma unroll
        for (int v = 0; v < V; v += 4) *(float4*)(s + v) = *(const float4*)(p + v);
    } else {
        s[0] = *p;
    }
}
template <int V> __device__ __forceinline__ void state_out(float* p, const float* s) {
    if constexpr (V == 2) {
        *(float2*)p = *(const float2*)s;
    } else if constexpr (V > 1) {
#pragma unroll
        for (int v = 0; v < V; v += 4) *(float4*)(p + v) = *(const float4*)(s + v);
    } else {
        *p = s[0];
    }
}

template <typename T, bool LOGITS, bool BWD, bool KEEP, int V>
__global__ void __launch_bounds__(128) rec_few_kernel(const RecParams p) {
    constexpr bool WALKS = BWD && sizeof(T) == 2;
    constexpr int U = WALKS ? GROUP : 4;
    const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
    const int per = p.D / V;
    if (i >= (int64_t)p.B * per) return;
    const int b = (int)(i / per), d = (int)(i % per) * V;
    const T* x = (const T*)p.x + b * p.sx[0] + d;
    const T* g = (const T*)p.g + b * p.sg[0] + d;
    const T* hin = BWD ? (const T*)p.h_in + b * p.sh[0] + d : nullptr;
    T* out = (T*)p.out + b * p.so[0] + d;
    T* outg = BWD ? (T*)p.out_g + b * p.sog[0] + d : nullptr;
    auto at = [&](int k) { return (int64_t)(p.from_end ? p.L - 1 - k : k); };
    alignas(4 * V) float s[V];
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = 0.f;
    if (p.s0) state_in<V>(s, p.s0 + b * p.ld_s0 + d);
    const int next = WALKS && p.walk ? 0 : 1;      // token of h_in that belongs to a token
    for (int k0 = 0; k0 < p.L; k0 += U) {
        Few<T, V> xr[U], gr[U], hr[BWD ? U : 1];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k0 + u < p.L) {
                xr[u].load(x + at(k0 + u) * p.sx[1]);
                gr[u].load(g + at(k0 + u) * p.sg[1]);
                if (BWD && k0 + u + next < p.L) hr[u].load(hin + at(k0 + u + next) * p.sh[1]);
            }
        }
        if constexpr (WALKS) {
            const int left = p.L - k0;
            float a[U][V], rest[U][V], before[U][V], h[V];
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = 0.f;
            if (left > U && p.walk) state_in<V>(h, p.states + ((int64_t)b * p.groups() + k0 / U) * p.D + d);
            else if (left <= U && p.h0) state_in<V>(h, p.h0 + (int64_t)b * p.D + d);
#pragma unroll
            for (int u = U - 1; u >= 0; --u) {
                if (u >= left) continue;
                float gf[V], hf[V];
                gr[u].get(gf);
                decays<T, LOGITS, BWD, V>(gf, p.inv_norm, a[u], rest[u]);
                hr[u].get(hf);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    before[u][v] = p.walk || u + 1 == left ? h[v] : hf[v];
                    h[v] = fmaf(a[u][v], h[v], hf[v]);                     // (used where hf is x)
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u >= left) break;
                float xf[V], og[V];
                xr[u].get(xf);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    xf[v] += s[v];
                    s[v] = a[u][v] * xf[v];
                    og[v] = s[v] * before[u][v];
                    if (LOGITS) og[v] *= p.inv_norm * rest[u][v];
                }
                Few<T, V>::store(out + at(k0 + u) * p.so[1], xf);
                Few<T, V>::store(outg + at(k0 + u) * p.sog[1], og);
            }
        } else {
            const int due = (p.L - 1 - k0) % GROUP;        // the token that leaves its state
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (k0 + u >= p.L) break;
                float xf[V], gf[V], a[V], rest[V];
                xr[u].get(xf);
                gr[u].get(gf);
                decays<T, LOGITS, BWD, V>(gf, p.inv_norm, a, rest);
                if (!BWD) {
#pragma unroll
                    for (int v = 0; v < V; ++v) s[v] = fmaf(a[v], s[v], xf[v]);
                    Few<T, V>::store(out + at(k0 + u) * p.so[1], s);
                    if (KEEP && u == due && k0 + u + 1 < p.L) state_out<V>(p.states + ((int64_t)b * p.groups() + (p.L - 1 - k0) / GROUP - 1) * p.D + d, s);
                } else {
                    float hb[V], og[V];
                    if (k0 + u + 1 < p.L) {
                        hr[u].get(hb);
                    } else {
#pragma unroll
                        for (int v = 0; v < V; ++v) hb[v] = 0.f;
                        if (p.h0) state_in<V>(hb, p.h0 + (int64_t)b * p.D + d);
                    }
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        xf[v] += s[v];
                        s[v] = a[v] * xf[v];
                        og[v] = s[v] * hb[v];
                        if (LOGITS) og[v] *= p.inv_norm * rest[v];
                    }
                    Few<T, V>::store(out + at(k0 + u) * p.so[1], xf);
                    Few<T, V>::store(outg + at(k0 + u) * p.sog[1], og);
                }
            }
        }
    }
    if (p.s_end) state_out<V>(p.s_end + b * p.ld_end + d, s);
}


// ---------------------------------------------------------------------------------------------------
// Rows of any alignment.  A cluster of CTAs owns a strip of 32 channels of one sequence and walks it in steps of (CTAs x 8 warps x RUN)
// tokens.  A warp's lanes are channels, a thread holds RUN consecutive tokens of its channel in registers.  In a step every
// thread scans its tokens from a zero state, which gives the product of their decays and their own contribution; these pairs meet in shared
// memory, the CTAs' totals in the shared memory of every CTA of the cluster (stores that its mbarrier counts: a cluster barrier would
// also wait for the outputs of the step before).  Each thread then joins the pairs ahead of it to the state that the step began with and
// walks its tokens again from there, in the order of the definition.  The next step's tokens are requested before the first meeting.
// Every value is read and written once.  No state is rounded, no order depends on timing.
// (Decays may exceed one, as long as their product over a step's tokens stays below 3.4e38.)
template <typename T, int V> struct Raw;
template <> struct Raw<float, 1> {
    using type = float;
    static __device__ void get(float r, float* f) { f[0] = r; }
    static __device__ float put(const float* f) { return f[0]; }
};
template <typename T> struct Raw<T, 1> {
    using type = T;
    static __device__ void get(T r, float* f) { f[0] = DType<T>::to_f(r); }
    static __device__ T put(const float* f) { return DType<T>::from_f(f[0]); }
};
template <> struct Raw<__nv_bfloat16, 2> {
    using type = __nv_bfloat162;
    static __device__ void get(type r, float* f) { const float2 v = __bfloat1622float2(r); f[0] = v.x; f[1] = v.y; }
    static __device__ type put(const float* f) { return __floats2bfloat162_rn(f[0], f[1]); }
};
template <> struct Raw<__half, 2> {
    using type = __half2;
    static __device__ void get(type r, float* f) { const float2 v = __half22float2(r); f[0] = v.x; f[1] = v.y; }
    static __device__ type put(const float* f) { return __floats2half2_rn(f[0], f[1]); }
};

constexpr int RW = 8;                 // warps of a CTA, and of one below
constexpr int TW = 4;
constexpr int RC = 8;                 // CTAs of a cluster of this kernel, at most

// The product of decays of a stretch of tokens, kept finite: 0 times it stays 0.  (Were a decay NaN, the stretch's contribution is NaN.)
__device__ __forceinline__ float finite(float a) { return fminf(a, 3.4028235e38f); }

// A stretch's product of decays can be 0 in fp32 where none of them is, and an infinite state would become NaN over it.  A CTA that met one (which
// costs a maximum a step to know) tells its cluster, and when all are done the warps go over such channels again, 32 tokens to a scan in which a product of
// 0 without a decay of 0 is -0 and leaves an infinite state as it is.  What is not finite is written, the rest keeps its bits.  (16 x 4096 x 768 bf16
// with an infinity in one channel of each sequence 0.32 ms, in all 2.9.  Telling the zeros apart in every join instead: 62 / 111 -> 66 / 125 us without any.)
constexpr float INFINITE = __builtin_huge_valf();
__device__ __forceinline__ float times(float a, float b) {
    const float c = finite(a * b);
    return c == 0.f ? (__float_as_uint(a) == 0 || __float_as_uint(b) == 0 ? 0.f : -0.f) : c;
}
__device__ __forceinline__ float behind(float a, float s, float h) {
    return __float_as_uint(a) == 0x80000000u && fabsf(s) == INFINITE ? s + h : fmaf(a, s, h);
}
__device__ __forceinline__ void mark(uint32_t* word, uint32_t ctas) {
    const uint32_t at = tc::smem_u32(word);
    for (uint32_t r = 0; r < ctas; ++r) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::map_rank(at, r)), "r"(1u) : "memory");
}
template <typename T, bool LOGITS, bool BWD, bool KEEP> __device__ __noinline__ void rec_again(const RecParams& p, int b, int d, float s) {
    constexpr uint32_t ALL = 0xffffffffu;
    const int lane = threadIdx.x & 31;
    const bool walk = BWD && sizeof(T) == 2 && p.walk;
    auto at = [&](const void* q, const int64_t* st, int k) { return (T*)q + b * st[0] + (int64_t)(p.from_end ? p.L - 1 - k : k) * st[1] + d; };
    auto get = [&](const void* q, const int64_t* st, int k) { return k < p.L ? DType<T>::to_f(*at(q, st, k)) : 0.f; };
    float xn = get(p.x, p.sx, lane), gn = get(p.g, p.sg, lane), hn = BWD ? get(p.h_in, p.sh, lane + (walk ? 0 : 1)) : 0.f;
    for (int k0 = 0; k0 < p.L; k0 += 32) {
        const int k = k0 + lane;
        const bool in = k < p.L;
        const float x = xn, g = gn, hin = hn;
        if (k0 + 32 < p.L) {
            xn = get(p.x, p.sx, k + 32);
            gn = get(p.g, p.sg, k + 32);
            if (BWD) hn = get(p.h_in, p.sh, k + 32 + (walk ? 0 : 1));
        }
        float a, rest = 1.f;
        decays<T, LOGITS, BWD, 1>(&g, p.inv_norm, &a, &rest);
        if (!in) a = 1.f;
        float A = a, H = BWD ? a * x : x;
#pragma unroll
        for (int off = 1; off < 32; off *= 2) {
            const float oa = __shfl_up_sync(ALL, A, off), oh = __shfl_up_sync(ALL, H, off);
            if (lane >= off) {
                H = behind(A, oh, H);
                A = times(A, oa);
            }
        }
        const float state = behind(A, s, H);
        float before = __shfl_up_sync(ALL, state, 1);
        if (lane == 0) before = s;
        s = __shfl_sync(ALL, state, 31);
        auto odd = [](float value) { return !(fabsf(value) <= 3.4028235e38f); };
        if (!BWD) {
            if (in && odd(state)) {
                *at(p.out, p.so, k) = DType<T>::from_f(state);
                const int later = p.L - 1 - k;
                if (KEEP && later && later % GROUP == 0) p.states[((int64_t)b * p.groups() + later / GROUP - 1) * p.D + d] = state;
            }
        } else {
            float hb = hin;
            if (walk) {
                const int left = p.L - (k & ~(GROUP - 1));
                float h = left > GROUP ? p.states[((int64_t)b * p.groups() + k / GROUP) * p.D + d] : left > 0 && p.h0 ? p.h0[(int64_t)b * p.D + d] : 0.f;
#pragma unroll
                for (int i = GROUP - 1; i >= 0; --i) {
                    if ((lane & (GROUP - 1)) == i) hb = h;
                    h = fmaf(__shfl_sync(ALL, a, i, GROUP), h, __shfl_sync(ALL, hin, i, GROUP));
                }
            } else if (k == p.L - 1) {
                hb = p.h0 ? p.h0[(int64_t)b * p.D + d] : 0.f;
            }
            const float dx = x + before;
            if (in && odd(dx)) {
                *at(p.out, p.so, k) = DType<T>::from_f(dx);
                *at(p.out_g, p.sog, k) = DType<T>::from_f(LOGITS ? state * hb * p.inv_norm * rest : state * hb);
            }
        }
    }
    if (p.s_end && lane == 0 && !(fabsf(s) <= 3.4028235e38f)) p.s_end[b * p.ld_end + d] = s;
}

template <typename T, bool LOGITS, bool BWD, bool KEEP, int RUN>
__global__ void __launch_bounds__(RW * 32, 2) rec_strip_kernel(const __grid_constant__ RecParams p) {
    constexpr int V = 1;
    using R = typename Raw<T, V>::type;
    struct alignas(8 * V) Pair { float a[V], h[V]; };                 // product of decays and contribution of a stretch of tokens
    __shared__ Pair own[2][RW][32];                // of each warp's tokens
    __shared__ Pair all[2][RC][32];                // of each CTA's
    __shared__ uint64_t landed[2];                 // counts the bytes of `all`
    __shared__ float begun[32];                    // the state that entered, and whether one was infinite: for a CTA that walks again
    __shared__ uint32_t met[32];
    const uint32_t rank = tc::cluster_rank(), ctas = tc::cluster_size(), bar = tc::smem_u32(landed);
    if (ctas > 1) {
        if (threadIdx.x == 0) {
            tc::mbar_init(bar, 1);
            tc::mbar_init(bar + 8, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
    }
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int strips = (p.D + 32 * V - 1) / (32 * V);
    const int strip = blockIdx.x / ctas, b = strip / strips, d = (strip % strips) * 32 * V + lane * V;
    const bool live = d < p.D;
    // tokens are numbered as the scan meets them: k-th token at base + k * step bytes
    struct Walk { char* base; int step; };
    auto walk = [&](const void* q, const int64_t* st) {
        const int64_t last = p.from_end ? (int64_t)(p.L - 1) * st[1] : 0;
        return Walk{(char*)((T*)q + b * st[0] + last + d), (int)((p.from_end ? -st[1] : st[1]) * (int64_t)sizeof(T))};
    };
    const Walk x = walk(p.x, p.sx), g = walk(p.g, p.sg), out = walk(p.out, p.so), hin = BWD ? walk(p.h_in, p.sh) : x, outg = BWD ? walk(p.out_g, p.sog) : x;
    auto to = [](const Walk& w, int k) { return w.base + (int64_t)k * w.step; };
    auto cell = [](char* at, const Walk& w, int i) { return (R*)(at + (int64_t)i * w.step); };
    const int per = (int)ctas * RW * RUN;          // tokens of a step
    float carry[V], first[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        carry[v] = live && p.s0 ? p.s0[b * p.ld_s0 + d + v] : 0.f;
        first[v] = BWD && live && p.h0 ? p.h0[(int64_t)b * p.D + d + v] : 0.f;
    }
    constexpr bool WALKS = BWD && sizeof(T) == 2;
    static_assert(!BWD || RUN == GROUP, "a thread's tokens share a state");
    float* const kept = KEEP || (WALKS && p.walk) ? p.states + (int64_t)b * p.groups() * p.D + d : nullptr;
    const int keeps = (p.L - 1) % GROUP;           // KEEP: which of eight tokens leave their state
    const int next = WALKS && p.walk ? 0 : 1;      // token of h_in that belongs to a token
    if (wid == 0) { begun[lane] = carry[0]; met[lane] = 0; }
    float most = 0.f;                              // the largest magnitude of a state or a contribution
    R xn[RUN], gn[RUN], hn[BWD ? RUN : 1];
    float sn[V] = {};
    auto fetch = [&](int k0) {
        if (!live) return;
        char *px = to(x, k0), *pg = to(g, k0), *ph = to(hin, k0);
        if (WALKS && p.walk && k0 + RUN < p.L) sn[0] = kept[(int64_t)(k0 / GROUP) * p.D];
        if (k0 + RUN < p.L) {
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                xn[i] = *cell(px, x, i);
                gn[i] = *cell(pg, g, i);
                if (BWD) hn[i] = *cell(ph, hin, i + next);
            }
        } else {
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                if (k0 + i < p.L) { xn[i] = *cell(px, x, i); gn[i] = *cell(pg, g, i); }
                if (BWD && k0 + i + next < p.L) hn[i] = *cell(ph, hin, i + next);
            }
        }
    };
    const int mine = ((int)rank * RW + wid) * RUN;
    fetch(mine);
    uint32_t phase = 0;
    for (int base = 0, buf = 0; base < p.L; base += per, buf ^= 1) {
        if (ctas > 1 && threadIdx.x == 0) tc::mbar_expect_tx(bar + 8 * buf, ctas * 32 * (uint32_t)sizeof(Pair));
        const int k0 = base + mine, left = live ? p.L - k0 : 0;        // tokens behind the last one leave the state as it is
        float a[RUN][V], rest[BWD && LOGITS ? RUN : 1][V], A[V], H[V], before[BWD ? RUN : 1][V];
        R xr[RUN];
#pragma unroll
        for (int v = 0; v < V; ++v) { A[v] = 1.f; H[v] = 0.f; }
        auto local = [&](auto whole) {
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                float gf[V], xf[V];
                Raw<T, V>::get(gn[i], gf);
                Raw<T, V>::get(xn[i], xf);
                decays<T, LOGITS, BWD, V>(gf, p.inv_norm, a[i], rest[BWD && LOGITS ? i : 0]);
                if (!decltype(whole)::value && i >= left) {
#pragma unroll
                    for (int v = 0; v < V; ++v) { a[i][v] = 1.f; xf[v] = 0.f; }
                }
                xr[i] = xn[i];
                if (BWD) {
                    Raw<T, V>::get(hn[i], before[i]);
#pragma unroll
                    for (int v = 0; v < V; ++v) H[v] += xf[v];
                    mul_v<V>(H, a[i], H);
                } else {
                    fma_v<V>(H, a[i], H, xf);
                }
                mul_v<V>(A, A, a[i]);
            }
        };
        if (left >= RUN) local(std::true_type()); else local(std::false_type());
        if constexpr (BWD) {
            // the states ahead of the tokens in the forward's order
            if (WALKS && p.walk) {
                float h = left > RUN ? sn[0] : first[0];
#pragma unroll
                for (int i = RUN - 1; i >= 0; --i) {
                    if (i < left) {
                        const float xi = before[i][0];
                        before[i][0] = h;
                        h = fmaf(a[i][0], h, xi);
                    }
                }
            } else if (left <= RUN) {
#pragma unroll
                for (int i = 0; i < RUN; ++i) if (i + 1 == left) before[i][0] = first[0];
            }
        }
        if (base + per < p.L) fetch(k0 + per);
        Pair me;
#pragma unroll
        for (int v = 0; v < V; ++v) { me.a[v] = finite(A[v]); me.h[v] = H[v]; }
        own[buf][wid][lane] = me;
        // I run, and have read the state that enters: waited for before a CTA's memory is written, and so before the final state is, which may lie there
        if (ctas > 1 && base == 0) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        __syncthreads();
        float s[V];
        if (ctas > 1) {
            // joined: the tokens of the CTA ahead of this warp's; and all of them
            float pa[V], ph[V];
#pragma unroll
            for (int v = 0; v < V; ++v) { me.a[v] = 1.f; me.h[v] = 0.f; }
#pragma unroll
            for (int w = 0; w < RW; ++w) {
                const Pair e = own[buf][w][lane];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (w == wid) { pa[v] = me.a[v]; ph[v] = me.h[v]; }
                    me.h[v] = fmaf(e.a[v], me.h[v], e.h[v]);
                    me.a[v] = finite(me.a[v] * e.a[v]);
                }
            }
            if (base == 0) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
            for (uint32_t other = wid; other < ctas; other += RW) {
                const uint32_t at = tc::map_rank(tc::smem_u32(&all[buf][rank][lane]), other), count = tc::map_rank(bar + 8 * buf, other);
                asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];"
                             ::"r"(at), "r"(__float_as_uint(me.a[0])), "r"(__float_as_uint(me.h[0])), "r"(count) : "memory");
            }
            int tries = 0;
            while (!tc::mbar_try_wait_parked(bar + 8 * buf, (phase >> buf) & 1, 1000000)) {
                if (++tries > 2000) {                                  // about a second or two: say so, and finish with what is there
                    if (p.status && lane == 0) atomicOr(p.status, 1);
                    break;
                }
            }
            phase ^= 1u << buf;
#pragma unroll
            for (int v = 0; v < V; ++v) s[v] = carry[v];
#pragma unroll 4
            for (uint32_t r = 0; r < ctas; ++r) {
                const Pair e = all[buf][r][lane];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (r == rank) s[v] = carry[v];
                    carry[v] = fmaf(e.a[v], carry[v], e.h[v]);
                }
            }
#pragma unroll
            for (int v = 0; v < V; ++v) s[v] = fmaf(pa[v], s[v], ph[v]);
        } else {
#pragma unroll
            for (int w = 0; w < RW; ++w) {
                const Pair e = own[buf][w][lane];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (w == wid) s[v] = carry[v];
                    carry[v] = fmaf(e.a[v], carry[v], e.h[v]);
                }
            }
        }
        most = fmaxf(most, fmaxf(fabsf(s[0]), fabsf(H[0])));
        char *po = to(out, k0), *pog = to(outg, k0);
        auto outputs = [&](auto whole) {
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                if (!decltype(whole)::value && i >= left) break;
                float xf[V], o[V];
                Raw<T, V>::get(xr[i], xf);
                if (!BWD) {
                    fma_v<V>(s, a[i], s, xf);
                    *cell(po, out, i) = Raw<T, V>::put(s);
                    if (KEEP && i % GROUP == keeps && (decltype(whole)::value || i + 1 < left)) kept[(int64_t)((p.L - 1 - k0 - i) / GROUP - 1) * p.D] = s[0];
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) o[v] = xf[v] + s[v];
                    mul_v<V>(s, a[i], o);
                    *cell(po, out, i) = Raw<T, V>::put(o);
                    mul_v<V>(o, s, before[i]);
                    if (LOGITS) {
#pragma unroll
                        for (int v = 0; v < V; ++v) o[v] *= p.inv_norm * rest[i][v];
                    }
                    *cell(pog, outg, i) = Raw<T, V>::put(o);
                }
            }
        };
        if (left > RUN) outputs(std::true_type()); else outputs(std::false_type());
        // the state behind the last token, as that token's output was rounded from it
        if (p.s_end && left > 0 && left <= RUN) {
#pragma unroll
            for (int v = 0; v < V; ++v) p.s_end[b * p.ld_end + d + v] = s[v];
        }
    }
    // no CTA leaves while another may still write to it (one that gave up waiting; marks), and what another has written is there
    if (most == INFINITE) mark(met + lane, ctas);
    if (ctas == 1) __syncthreads();
    if (ctas > 1) {
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }
    for (int c = wid * (int)ctas + (int)rank; c < 32; c += RW * (int)ctas) if (met[c]) rec_again<T, LOGITS, BWD, KEEP>(p, b, d - lane + c, begun[c]);
}

// ---------------------------------------------------------------------------------------------------
// The same walk for rows of whole 16-byte pieces, which come to shared memory by asynchronous copies, two steps ahead.  A chunk is RUN tokens of
// 4 bytes a lane (V channels) times LPC lanes; a warp holds 32 / LPC chunks side by side (its lanes, LPC by LPC) and brings their rows
// itself.  No registers wait for memory.  Narrow strips (LPC 16 or 8) are the finer pieces of work where 32 lanes a strip would leave SMs idle;
// the pairs of a warp's own chunks meet by shuffles.  What it measured on the way, forward, raw bf16 logits (us):
//   loads a step ahead in registers, pairs over a barrier           16 x 4096 x 768   92     1 x 16384 x 768   41
//   rows in shared memory, three CTAs of eight warps an SM                            75                       26
//   decays of the next step under the outputs of this one                             67                       28
//   the state handed from warp to warp, no barrier                                    62                       28
//   four CTAs of four warps an SM, requests under the exchange                        62 (backward 103 -> 91)  24
//   (graph replays on the same buffers; backward from h.  States and x in its place: 91 -> 108)
// Also tried: every warp adding up all pairs behind flags instead of the hand-over (the warps then keep step: 71), 32 tokens a thread
// (1 x 16384 x 768 26), prefetch hints on the copies (no difference).
__device__ __forceinline__ void copy_16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }

template <bool BWD> constexpr int tile_run = BWD ? 8 : 16;
constexpr int tile_stages = 3;
// bytes of a chunk of one tensor, with the shift that keeps the chunks of a warp in different banks
template <int LPC, int RUN> constexpr int tile_chunk = RUN * LPC * 4 + (LPC < 32 ? LPC * 4 : 0);
template <bool BWD, int LPC> constexpr int tile_warp = (BWD ? 3 : 2) * (32 / LPC) * tile_chunk<LPC, tile_run<BWD>>;      // of a warp and stage
template <bool BWD, int LPC> constexpr int tile_smem = TW * tile_stages * tile_warp<BWD, LPC>;
// ... and of what its warps, or its cluster's CTAs, tell one another (a pair is 8 bytes a channel)
template <int LPC, int V> int tile_words(int ctas) { return ctas == 1 ? TW * LPC * V * 4 : 2 * (TW + ctas) * LPC * V * 8; }

template <typename T, bool LOGITS, bool BWD, bool KEEP, int LPC>
__global__ void __launch_bounds__(TW * 32, 4) rec_tile_kernel(const __grid_constant__ RecParams p) {
    constexpr int V = 4 / (int)sizeof(T), RUN = tile_run<BWD>, NC = 32 / LPC, ROW = LPC * 4, PIECES = ROW / 16, NT = BWD ? 3 : 2;
    constexpr int CHUNK = tile_chunk<LPC, RUN>;
    using R = typename Raw<T, V>::type;
    struct alignas(8 * V) Pair { float a[V], h[V]; };
    extern __shared__ __align__(128) uint8_t tiles[];
    __shared__ float begun[LPC * V];               // the state that entered, and whether one was infinite: for a CTA that walks again
    __shared__ uint32_t met[LPC * V];
    __shared__ uint64_t landed[TW];                // one CTA: one a warp, its mail is there; several: 0 and 1 count the bytes of `all`
    const uint32_t rank = tc::cluster_rank(), ctas = tc::cluster_size(), bar = tc::smem_u32(landed);
    // behind the tiles, one CTA: the state ahead of each warp's tokens, from the warp before; several: the pair of each warp's tokens and of each
    // CTA's, for this step and the one before
    float (*mail)[LPC][V] = (float (*)[LPC][V])(tiles + tile_smem<BWD, LPC>);
    Pair (*own)[TW][LPC] = (Pair (*)[TW][LPC])(tiles + tile_smem<BWD, LPC>), *all = (Pair*)(own + 2);
    if (threadIdx.x < TW) tc::mbar_init(bar + 8 * threadIdx.x, 1);
    if (threadIdx.x < LPC * V) met[threadIdx.x] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, q = lane / LPC, l = lane % LPC;
    const int strips = (p.D + LPC * V - 1) / (LPC * V);
    const int strip = blockIdx.x / ctas, b = strip / strips, d0 = (strip % strips) * LPC * V, d = d0 + l * V;
    const bool live = d < p.D;
    const int per = (int)ctas * TW * NC * RUN;     // tokens of a step
    const int first_of_warp = ((int)rank * TW + wid) * NC * RUN, mine = first_of_warp + q * RUN;
    // ---- the warp's copies: piece `pc` of rows r0, r0 + 32 / PIECES, ... of its NC * RUN rows
    const int pc = lane % PIECES, r0 = lane / PIECES;
    const uint32_t ring = tc::smem_u32(tiles) + wid * tile_stages * tile_warp<BWD, LPC>;
    struct Walk { const char* base; int step; };   // tokens are numbered as the scan meets them: the k-th at base + k * step bytes
    auto walk = [&](const void* at, const int64_t* st, int channel) {
        const int64_t last = p.from_end ? (int64_t)(p.L - 1) * st[1] : 0;
        return Walk{(const char*)((const T*)at + b * st[0] + last + channel), (int)((p.from_end ? -st[1] : st[1]) * (int64_t)sizeof(T))};
    };
    const bool piece = d0 + pc * (16 / (int)sizeof(T)) < p.D;
    const int pd = piece ? d0 + pc * (16 / (int)sizeof(T)) : 0;
    const Walk src[3] = {walk(p.x, p.sx, pd), walk(p.g, p.sg, pd), BWD ? walk(p.h_in, p.sh, pd) : Walk{}};
    constexpr bool WALKS = BWD && sizeof(T) == 2;
    static_assert(!BWD || RUN == GROUP, "a thread's tokens share a state");
    const int next = WALKS && p.walk ? 0 : 1;      // token of h_in that belongs to a token
    const uint32_t slot = ring + (r0 / RUN) * CHUNK + (r0 % RUN) * ROW + pc * 16;
    constexpr int HOP = 32 / PIECES, AHEAD = HOP / RUN * CHUNK + HOP % RUN * ROW;      // rows from one copy of a lane to its next, and how far that is
    static_assert(HOP % RUN == 0 || RUN % HOP == 0, "a lane's rows are evenly spaced, or lie in one chunk");
    auto bring = [&](int base, int stage) {
        const int k0 = base + first_of_warp;
        if (k0 + NC * RUN + (BWD ? next : 0) <= p.L) {
            if (piece) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const char* from = src[n].base + (int64_t)(k0 + r0 + (n == 2 ? next : 0)) * src[n].step;
#pragma unroll
                    for (int r = 0; r < NC * RUN / HOP; ++r)
                        copy_16(slot + stage * tile_warp<BWD, LPC> + n * NC * CHUNK + (HOP >= RUN ? r * AHEAD : r / (RUN / HOP) * CHUNK + r % (RUN / HOP) * AHEAD),
                                from + (int64_t)(r * HOP) * src[n].step);
                }
            }
        } else if (piece && k0 < p.L) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                for (int r = 0; r < NC * RUN / HOP; ++r) {
                    const int row = r * HOP + r0, k = k0 + row + (n == 2 ? next : 0);
                    if (k < p.L)
                        copy_16(ring + pc * 16 + stage * tile_warp<BWD, LPC> + n * NC * CHUNK + (row / RUN) * CHUNK + (row % RUN) * ROW, src[n].base + (int64_t)k * src[n].step);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int st = 0; st < tile_stages; ++st) bring(st * per, st);
    const Walk out = walk(p.out, p.so, d), outg = BWD ? walk(p.out_g, p.sog, d) : out;
    float carry[V], first[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        carry[v] = live && p.s0 ? p.s0[b * p.ld_s0 + d + v] : 0.f;
        first[v] = BWD && live && p.h0 ? p.h0[(int64_t)b * p.D + d + v] : 0.f;
    }
    float* const kept = KEEP || (WALKS && p.walk) ? p.states + (int64_t)b * p.groups() * p.D + d : nullptr;
    const int keeps = (p.L - 1) % GROUP;           // KEEP: which of eight tokens leave their state
    float sn[V] = {};                              // state in front of the thread's tokens, a step ahead
    auto state_of = [&](int k0) {
        if (WALKS && p.walk && live && k0 + RUN < p.L) {
            const float* from = kept + (int64_t)(k0 / GROUP) * p.D;
            if constexpr (V == 2) *(float2*)sn = *(const float2*)from;
            else sn[0] = *from;
        }
    };
    state_of(mine);
    if (threadIdx.x < LPC) {
#pragma unroll
        for (int v = 0; v < V; ++v) begun[l * V + v] = carry[v];
    }
    float most[V] = {};                            // the largest magnitude of a state or a contribution
    uint32_t phase = 0;
    float a[RUN][V], rest[BWD && LOGITS ? RUN : 1][V], A[V], H[V], s[V];
    uint8_t* const mine_of_ring = tiles + wid * tile_stages * tile_warp<BWD, LPC> + q * CHUNK + l * 4;
    auto place = [&](int stage, int n, int i) { return (uint32_t*)(mine_of_ring + stage * tile_warp<BWD, LPC> + n * NC * CHUNK + i * ROW); };
    auto cell = [&](int stage, int n, int i) {
        const uint32_t word = *place(stage, n, i);
        R r;
        memcpy(&r, &word, 4);
        return r;
    };
    // token i of a step: its decay, and the chunk's pair up to it
    auto enter = [&](int stage, int i, bool in) {
        float gf[V], xf[V];
        Raw<T, V>::get(cell(stage, 1, i), gf);
        Raw<T, V>::get(cell(stage, 0, i), xf);
        decays<T, LOGITS, BWD, V>(gf, p.inv_norm, a[i], rest[BWD && LOGITS ? i : 0]);
        if (!in) {
#pragma unroll
            for (int v = 0; v < V; ++v) { a[i][v] = 1.f; xf[v] = 0.f; }
        }
        if (BWD) {
            add_v<V>(H, H, xf);
            mul_v<V>(H, a[i], H);
        } else {
            fma_v<V>(H, a[i], H, xf);
        }
        mul_v<V>(A, A, a[i]);
    };
    // 16 bits: the states ahead of the tokens in the forward's order, in the places of what has been used of them (the gate, and h or x)
    auto before = [&](int stage, int i, int v) { return place(stage, v ? 1 : 2, i); };
    auto states = [&](int stage, int left) {
        float h[V], f[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = left > RUN ? sn[v] : first[v];
        if (p.walk && left >= RUN) {
            R xs[RUN];
#pragma unroll
            for (int i = RUN - 1; i >= 0; --i) xs[i] = cell(stage, 2, i);
#pragma unroll
            for (int i = RUN - 1; i >= 0; --i) {
                Raw<T, V>::get(xs[i], f);
#pragma unroll
                for (int v = 0; v < V; ++v) *before(stage, i, v) = __float_as_uint(h[v]);
                fma_v<V>(h, a[i], h, f);
            }
        } else {
#pragma unroll
            for (int i = RUN - 1; i >= 0; --i) {
                if (i >= left) continue;
                Raw<T, V>::get(cell(stage, 2, i), f);
                const bool known = p.walk || i + 1 == left;
#pragma unroll
                for (int v = 0; v < V; ++v) *before(stage, i, v) = __float_as_uint(known ? h[v] : f[v]);
                fma_v<V>(h, a[i], h, f);
            }
        }
    };
    // token i of a step: its outputs from the state ahead of it
    auto leave = [&](int stage, int i, char* po, char* pog, bool last, float* keep) {
        float xf[V], o[V];
        Raw<T, V>::get(cell(stage, 0, i), xf);
        if (!BWD) {
            fma_v<V>(s, a[i], s, xf);
            *(R*)(po + (int64_t)i * out.step) = Raw<T, V>::put(s);
            if (KEEP && i % GROUP == keeps && !last) {
                float* to = keep - (int64_t)(i / GROUP) * p.D;
                if constexpr (V == 2) *(float2*)to = make_float2(s[0], s[1]);
                else *to = s[0];
            }
        } else {
            float hf[V];
            if constexpr (WALKS) {
#pragma unroll
                for (int v = 0; v < V; ++v) hf[v] = __uint_as_float(*before(stage, i, v));
            } else {
                Raw<T, V>::get(cell(stage, 2, i), hf);
                if (last) {
#pragma unroll
                    for (int v = 0; v < V; ++v) hf[v] = first[v];
                }
            }
            add_v<V>(o, xf, s);
            mul_v<V>(s, a[i], o);
            *(R*)(po + (int64_t)i * out.step) = Raw<T, V>::put(o);
            mul_v<V>(o, s, hf);
            if (LOGITS) {
                const float inv[2] = {p.inv_norm, p.inv_norm};
                mul_v<V>(o, o, inv);
                mul_v<V>(o, o, rest[i]);
            }
            *(R*)(pog + (int64_t)i * outg.step) = Raw<T, V>::put(o);
        }
    };
    auto begin = [&]() {
#pragma unroll
        for (int v = 0; v < V; ++v) { A[v] = 1.f; H[v] = 0.f; }
    };
    asm volatile("cp.async.wait_group %0;" ::"n"(tile_stages - 1) : "memory");
    __syncwarp();
    begin();
#pragma unroll
    for (int i = 0; i < RUN; ++i) enter(0, i, live && mine + i < p.L);
    for (int base = 0, buf = 0, stage = 0; base < p.L; base += per, buf ^= 1) {
        if (ctas > 1 && threadIdx.x == 0) tc::mbar_expect_tx(bar + 8 * buf, ctas * LPC * (uint32_t)sizeof(Pair));
        const int k0 = base + mine, left = live ? p.L - k0 : 0;        // tokens behind the last one leave the state as it is
        // chunks of the warp ahead of mine: (ea, eh); the lanes of the last chunk then hold the warp's pair
        float ea[V], eh[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { A[v] = finite(A[v]); ea[v] = 1.f; eh[v] = 0.f; }
#pragma unroll
        for (int off = LPC; off < 32; off *= 2) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float oa = __shfl_up_sync(0xffffffffu, A[v], off), oh = __shfl_up_sync(0xffffffffu, H[v], off);
                if (lane >= off) {
                    H[v] = fmaf(A[v], oh, H[v]);
                    A[v] = finite(A[v] * oa);
                    if (NC == 2) { ea[v] = oa; eh[v] = oh; }
                }
            }
        }
        if (NC > 2) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float oa = __shfl_up_sync(0xffffffffu, A[v], LPC), oh = __shfl_up_sync(0xffffffffu, H[v], LPC);
                if (lane >= LPC) { ea[v] = oa; eh[v] = oh; }
            }
        }
        auto wait = [&](uint32_t what, uint32_t parity) {
            int tries = 0;
            while (!tc::mbar_try_wait_parked(what, parity, 1000000)) {
                if (++tries > 2000) {                                  // about a second or two: say so, and finish with what is there
                    if (p.status && lane == 0) atomicOr(p.status, 1);
                    break;
                }
            }
        };
        if (ctas > 1) {
            Pair me;
            if (lane >= 32 - LPC) {
#pragma unroll
                for (int v = 0; v < V; ++v) { me.a[v] = A[v]; me.h[v] = H[v]; }
                own[buf][wid][l] = me;
            }
            // I run, and have read the state that enters: waited for before a CTA's memory is written, and so before the final state is, which may lie there
            if (base == 0) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
            __syncthreads();
            // joined: the tokens of the CTA ahead of this warp's; and all of them
            float pa[V], ph[V];
#pragma unroll
            for (int v = 0; v < V; ++v) { me.a[v] = 1.f; me.h[v] = 0.f; }
#pragma unroll
            for (int w = 0; w < TW; ++w) {
                const Pair e = own[buf][w][l];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (w == wid) { pa[v] = me.a[v]; ph[v] = me.h[v]; }
                    me.h[v] = fmaf(e.a[v], me.h[v], e.h[v]);
                    me.a[v] = finite(me.a[v] * e.a[v]);
                }
            }
            if (base == 0) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
            if (lane < LPC)
                for (uint32_t other = wid; other < ctas; other += TW) {
                    const uint32_t at = tc::map_rank(tc::smem_u32(all + (buf * ctas + rank) * LPC + l), other), count = tc::map_rank(bar + 8 * buf, other);
                    if constexpr (V == 2)
                        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                                     ::"r"(at), "r"(__float_as_uint(me.a[0])), "r"(__float_as_uint(me.a[1])), "r"(__float_as_uint(me.h[0])), "r"(__float_as_uint(me.h[1])), "r"(count) : "memory");
                    else
                        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];"
                                     ::"r"(at), "r"(__float_as_uint(me.a[0])), "r"(__float_as_uint(me.h[0])), "r"(count) : "memory");
                }
            if (base) bring(base + (tile_stages - 1) * per, stage ? stage - 1 : tile_stages - 1);      // what the step before has read, while totals are under way
            if constexpr (WALKS) states(stage, left);
            wait(bar + 8 * buf, (phase >> buf) & 1);
            phase ^= 1u << buf;
#pragma unroll
            for (int v = 0; v < V; ++v) s[v] = carry[v];
#pragma unroll 4
            for (uint32_t r = 0; r < ctas; ++r) {
                const Pair e = all[(buf * ctas + r) * LPC + l];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (r == rank) s[v] = carry[v];
                    carry[v] = fmaf(e.a[v], carry[v], e.h[v]);
                }
            }
#pragma unroll
            for (int v = 0; v < V; ++v) s[v] = fmaf(pa[v], s[v], ph[v]);
        } else {
            // from warp to warp, round and round: no barrier, so the warps stay apart and one's arithmetic runs under another's waiting
            if constexpr (WALKS) states(stage, left);
            if (base || wid) {
                wait(bar + 8 * wid, (phase >> 2) & 1);
                phase ^= 4;
#pragma unroll
                for (int v = 0; v < V; ++v) s[v] = mail[wid][l][v];
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) s[v] = carry[v];
            }
            if (base + (wid == TW - 1 ? per : 0) < p.L) {
                const int to = (wid + 1) % TW;
                if (lane >= 32 - LPC) {
#pragma unroll
                    for (int v = 0; v < V; ++v) mail[to][l][v] = fmaf(A[v], s[v], H[v]);
                }
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar + 8 * to) : "memory");
            }
        }
        if (LPC < 32) fma_v<V>(s, ea, s, eh);
#pragma unroll
        for (int v = 0; v < V; ++v) most[v] = fmaxf(most[v], fmaxf(fabsf(s[v]), fabsf(H[v])));
        char *po = (char*)out.base + (int64_t)k0 * out.step, *pog = (char*)outg.base + (int64_t)k0 * outg.step;
        float* const keep = kept + (int64_t)((p.L - 1 - k0 - keeps) / GROUP - 1) * p.D;         // where the first token to leave its state does
        state_of(k0 + per);
        const int ahead = stage + 1 < tile_stages ? stage + 1 : 0;
        const bool more = base + per < p.L;
        asm volatile("cp.async.wait_group %0;" ::"n"(tile_stages - 2) : "memory");
        __syncwarp();
        begin();
        if (left - per >= RUN) {
            // a token's decay is used for the last time, and in its place comes that of the next step: the MUFU unit works under the
            // multiply-adds and stores (one after the other, the warps of an SM fall into step and leave it idle)
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                leave(stage, i, po, pog, false, keep);
                enter(ahead, i, true);
            }
        } else {
#pragma unroll
            for (int i = 0; i < RUN; ++i)
                if (i < left) leave(stage, i, po, pog, i + 1 == left, keep);
            if (more) {
#pragma unroll
                for (int i = 0; i < RUN; ++i) enter(ahead, i, i < left - per);
            }
        }
        // the state behind the last token, as that token's output was rounded from it
        if (p.s_end && left > 0 && left <= RUN) {
#pragma unroll
            for (int v = 0; v < V; ++v) p.s_end[b * p.ld_end + d + v] = s[v];
        }
        __syncwarp();
        if (ctas == 1) bring(base + tile_stages * per, stage);
        stage = ahead;
    }
    // no CTA leaves while another may still write to it (one that gave up waiting; marks), and what another has written is there
#pragma unroll
    for (int v = 0; v < V; ++v) if (most[v] == INFINITE) mark(met + l * V + v, ctas);
    if (ctas == 1) __syncthreads();
    if (ctas > 1) {
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }
    for (int c = wid * (int)ctas + (int)rank; c < LPC * V; c += TW * (int)ctas) if (met[c]) rec_again<T, LOGITS, BWD, KEEP>(p, b, d0 + c, begun[c]);
}

static cudaError_t rec_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute& attr, void (*kernel)(RecParams), int64_t strips, int c, int warps, size_t smem, cudaStream_t s) {
    cfg = {};
    cfg.gridDim = dim3((unsigned)(strips * c)); cfg.blockDim = dim3(warps * 32); cfg.stream = s; cfg.dynamicSmemBytes = smem;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = c; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (smem > 24 * 1024)                          // with what is static, more than a kernel has unasked
        if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) return e;
    return c > 8 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) : cudaSuccess;
}

static int rec_clusters(void (*kernel)(RecParams), const RecParams& p, int64_t strips, int c, int warps, size_t smem, cudaStream_t s) {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    if (const cudaError_t e = rec_config(cfg, attr, kernel, strips, c, warps, smem, s)) return (int)e;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}

// Whether this device places clusters of 16 of a kernel: more than is promised, so it is asked once.
template <typename T, bool LOGITS, bool BWD, bool KEEP, int LPC> bool places_16() {
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    int k = known[dev].load(std::memory_order_relaxed);
    if (!k) {
        cudaLaunchConfig_t cfg;
        cudaLaunchAttribute attr;
        int n = 0;
        auto kernel = rec_tile_kernel<T, LOGITS, BWD, KEEP, LPC>;
        const bool yes = rec_config(cfg, attr, kernel, 1, 16, TW, tile_smem<BWD, LPC> + tile_words<LPC, 4 / (int)sizeof(T)>(16), nullptr) == cudaSuccess && cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess && n > 0;
        if (!yes) cudaGetLastError();
        known[dev].store(k = yes ? 1 : 2, std::memory_order_relaxed);
    }
    return k == 1;
}

// CTAs of a cluster, a power of two up to 8 (others are placed badly: three took longer than four): the fewest that make `want` of them in
// all, no more than the sequence has steps for
static int rec_ctas(int64_t strips, int L, int step, int64_t want) {
    int c = 1;
    while (c < 8 && c * strips < want && c * (int64_t)step < L) c *= 2;
    return c;
}

template <typename T, bool LOGITS, bool BWD, bool KEEP>
int rec_strips(const RecParams& p, cudaStream_t s) {
    constexpr int RUN = BWD ? 8 : 16;
    const int64_t strips = (int64_t)p.B * ((p.D + 31) / 32);
    return rec_clusters(rec_strip_kernel<T, LOGITS, BWD, KEEP, RUN>, p, strips, rec_ctas(strips, p.L, RW * RUN, device_sms()), RW, 0, s);
}

template <typename T, bool LOGITS, bool BWD, bool KEEP, int LPC>
int rec_tiles(const RecParams& p, int64_t strips, int c, cudaStream_t s) {
    return rec_clusters(rec_tile_kernel<T, LOGITS, BWD, KEEP, LPC>, p, strips, c, TW, tile_smem<BWD, LPC> + tile_words<LPC, 4 / (int)sizeof(T)>(c), s);
}

// Whether a step over all three or five tensors is a 32-bit number of bytes
inline bool short_steps(const RecParams& p, bool bwd) {
    const int64_t most = (1ll << 29) - 1;
    auto fits = [&](const int64_t* st) { return st[1] <= most && st[1] >= -most; };
    return fits(p.sx) && fits(p.sg) && fits(p.so) && (!bwd || (fits(p.sh) && fits(p.sog)));
}

// Whether all rows are 16-byte pieces
template <typename T> bool in_pieces(const RecParams& p, bool bwd) {
    auto fits = [&](const void* q, const int64_t* st) { return (uintptr_t)q % 16 == 0 && (p.B == 1 || st[0] * sizeof(T) % 16 == 0) && (p.L == 1 || st[1] * sizeof(T) % 16 == 0); };
    return p.D * sizeof(T) % 16 == 0 && fits(p.x, p.sx) && fits(p.g, p.sg) && fits(p.out, p.so) && (!bwd || (fits(p.h_in, p.sh) && fits(p.out_g, p.sog)));
}

template <typename T, bool LOGITS, bool BWD, bool KEEP = false>
int rec_launch(const RecParams& p, cudaStream_t s) {
    const bool pieces = in_pieces<T>(p, BWD);
    // A strip's CTA is made for 64 tokens and more: below 16 a thread that walks them is as fast (8 x 768 channels, 15 tokens: 3.7 us, 16 in strips
    // 4.8), and below 48 where the strips are more than find room at once (256 x 1024 channels, 16 tokens: 29 us in strips, 9 this way).
    const int64_t wide = (int64_t)p.B * ((p.D * (int64_t)sizeof(T) + 127) / 128);
    if (p.L < (wide >= 4 * device_sms() ? 48 : 16) || !short_steps(p, BWD)) {
        // several channels a thread once there are threads enough for every SM
        constexpr int V = few_v<T, BWD>;
        const int64_t n = (int64_t)p.B * p.D;
        auto state = [](const float* q, int64_t ld) { return (uintptr_t)q % 16 == 0 && ld % 4 == 0; };
        if (pieces && n / V >= 256ll * device_sms() && state(p.s0, p.ld_s0) && state(p.s_end, p.ld_end) && state(p.h0, 0))
            rec_few_kernel<T, LOGITS, BWD, KEEP, V><<<(unsigned)((n / V + 127) / 128), 128, 0, s>>>(p);
        else
            rec_few_kernel<T, LOGITS, BWD, KEEP, 1><<<(unsigned)((n + 127) / 128), 128, 0, s>>>(p);
        return (int)cudaGetLastError();
    }
    if (!pieces) return rec_strips<T, LOGITS, BWD, KEEP>(p, s);
    // Width of the strips and CTAs of a cluster.  Four CTAs find room on an SM.  Best is the widest strip of which there are enough by
    // themselves, 6/10 of the room (a cluster's meetings cost: 16 x 4096 x 768 bf16, forward, 64 us with 32 channels and one CTA, 72 with 64 and
    // two); else the widest that reaches that in clusters (4 x 4096 x 384, forward: 16.7 us with 32 channels and eight CTAs, 18.5 with 16 and
    // four); else the narrowest (1 x 16384 x 768, forward / backward: 29 / 47 us with 16 channels, 35 / 61 with 32).  The backward takes
    // narrower strips by themselves from 45/100 (16 x 2048 x 768: 61 us with 32 channels, 67 with 64 and two CTAs, 84 with one; 24 x 4096 x 768: 143, 158
    // and 175).  In fp32 its two tensors' half rows cost once many are under way (12 x 4096 x 768: 202 us with 16 channels, 153 with 32 and two
    // CTAs): whole rows of 128 bytes from 35/100 of the room.
    const int64_t room = 4 * device_sms(), joined = room * 60 / 100, alone = BWD ? room * 45 / 100 : joined;
    const int64_t whole_rows = BWD && sizeof(T) == 4 ? room * 35 / 100 : joined;
    auto strips = [&](int lpc) { const int w = lpc * (4 / (int)sizeof(T)); return (int64_t)p.B * ((p.D + w - 1) / w); };
    auto ctas = [&](int lpc) { return rec_ctas(strips(lpc), p.L, TW * (32 / lpc) * tile_run<BWD>, joined); };
    int lpc = 0, c = 1;
    if (strips(32) >= whole_rows) { lpc = 32; c = ctas(32); }
    // a few more than find room at once would make a second round of their own: in halves (56 x 1024 x 768, 672 strips of 64 channels: backward 105
    // us, 94 with 32; 50 x 2048 x 768, 600 strips: forward 102, 93)
    if (strips(32) > room && strips(32) * 10 <= room * (BWD ? 15 : 11)) { lpc = 16; c = 1; }
    for (int w = 16; w >= 8 && !lpc; w /= 2) if (strips(w) >= alone) lpc = w;
    for (int w = 32; w >= 8 && !lpc; w /= 2) if (strips(w) * ctas(w) >= joined) { lpc = w; c = ctas(w); }
    if (!lpc) {
        lpc = 8;
        c = ctas(8);
        // twice as many where they still find room at once (1 x 65536 x 192: 53 / 100 us with eight, 41 / 73 with sixteen)
        if (c == 8 && 16 * strips(8) <= room && 8ll * TW * 4 * tile_run<BWD> < p.L && places_16<T, LOGITS, BWD, KEEP, 8>()) c = 16;
    }
    switch (lpc) {
        case 32: return rec_tiles<T, LOGITS, BWD, KEEP, 32>(p, strips(32), c, s);
        case 16: return rec_tiles<T, LOGITS, BWD, KEEP, 16>(p, strips(16), c, s);
        default: return rec_tiles<T, LOGITS, BWD, KEEP, 8>(p, strips(8), c, s);
    }
}

template <bool BWD> int rec_dispatch(const RecParams& p, int dtype, cudaStream_t s) {
    if constexpr (!BWD) if (p.keep) {
        if (dtype == VIG_DTYPE_BF16) return p.inv_norm > 0.f ? rec_launch<__nv_bfloat16, true, false, true>(p, s) : rec_launch<__nv_bfloat16, false, false, true>(p, s);
        return p.inv_norm > 0.f ? rec_launch<__half, true, false, true>(p, s) : rec_launch<__half, false, false, true>(p, s);
    }
    switch (dtype) {
        case VIG_DTYPE_F32: return p.inv_norm > 0.f ? rec_launch<float, true, BWD>(p, s) : rec_launch<float, false, BWD>(p, s);
        case VIG_DTYPE_BF16: return p.inv_norm > 0.f ? rec_launch<__nv_bfloat16, true, BWD>(p, s) : rec_launch<__nv_bfloat16, false, BWD>(p, s);
        case VIG_DTYPE_F16: return p.inv_norm > 0.f ? rec_launch<__half, true, BWD>(p, s) : rec_launch<__half, false, BWD>(p, s);
    }
    return VIG_ERR_DTYPE;
}

// what every call is asked; token numbers are 32-bit with room for a step behind the last one
static int rec_check(int B, int L, int D, float norm, int dtype) {
    if (dtype < VIG_DTYPE_F32 || dtype > VIG_DTYPE_F16) return VIG_ERR_DTYPE;
    if (B < 0 || L < 0 || L >= (1 << 30) || D < 0 || D >= (1 << 28) || (int64_t)B * D >= (1ll << 31)) return VIG_ERR_SHAPE;
    if (norm != 0.f && !(norm >= 1e-30f && norm <= 1e30f)) return VIG_ERR_ARG;
    return VIG_OK;
}

// no token: the state that enters is the state that leaves
static int rec_empty(const float* s0, int64_t ld0, float* s_end, int64_t ld_end, int B, int D, cudaStream_t s) {
    const int64_t n = (int64_t)B * D;
    if (!s_end || !n) return VIG_OK;
    RecParams p{};
    p.s0 = s0; p.ld_s0 = ld0; p.s_end = s_end; p.ld_end = ld_end; p.B = B; p.D = D;
    rec_few_kernel<float, false, false, false, 1><<<(unsigned)((n + 127) / 128), 128, 0, s>>>(p);
    return (int)cudaGetLastError();
}

static void two(int64_t* dst, const int64_t* src, int L, int D) {
    dst[0] = src ? src[0] : (int64_t)L * D;
    dst[1] = src ? src[1] : D;
}

}  // namespace vig

using namespace vig;

extern "C" size_t vig_gated_recurrence_states_bytes(int B, int L, int D) {
    return B > 0 && L > GROUP && D > 0 ? (size_t)B * ((L - 1) / GROUP) * D * sizeof(float) : 0;
}

// what a training step of 16-bit tensors is asked beside: room for its states, which several channels of a thread store together
static int rec_states_check(const float* states, int B, int L, int D, int dtype) {
    if (dtype == VIG_DTYPE_F32) return VIG_ERR_DTYPE;
    if (!vig_gated_recurrence_states_bytes(B, L, D)) return VIG_OK;
    return !states ? VIG_ERR_NULL : (uintptr_t)states % 16 ? VIG_ERR_ALIGN : VIG_OK;
}

static int rec_fwd(const void* x, const void* g, const float* h0, int64_t ld_h0, void* h, float* h_final, int64_t ld_final, float* states, bool keep,
                   int B, int L, int D, const int64_t* strides_x, const int64_t* strides_g, const int64_t* strides_h,
                   float gate_logit_normalizer, int reverse, int dtype, int32_t* status_dev, void* stream) {
    if (const int e = rec_check(B, L, D, gate_logit_normalizer, dtype)) return e;
    if (B > 1 && ((h0 && ld_h0 < 0) || (h_final && ld_final < D))) return VIG_ERR_ARG;
    if (!B || !D || !L) return rec_empty(h0, ld_h0, h_final, ld_final, B, D, (cudaStream_t)stream);
    if (!x || !g || !h) return VIG_ERR_NULL;
    if (keep) if (const int e = rec_states_check(states, B, L, D, dtype)) return e;
    RecParams p{};
    p.states = states; p.keep = keep && L > GROUP;
    p.x = x; p.g = g; p.s0 = h0; p.ld_s0 = ld_h0; p.out = h; p.s_end = h_final; p.ld_end = ld_final;
    two(p.sx, strides_x, L, D); two(p.sg, strides_g, L, D); two(p.so, strides_h, L, D);
    p.B = B; p.L = L; p.D = D;
    p.inv_norm = gate_logit_normalizer > 0.f ? 1.f / gate_logit_normalizer : 0.f;
    p.from_end = reverse != 0;
    p.status = status_dev;
    return rec_dispatch<false>(p, dtype, (cudaStream_t)stream);
}

static int rec_bwd(const void* g, const void* h, const float* states, bool walk, const float* h0, const void* d_h, const float* d_final, void* d_x, void* d_g,
                   float* d_h0, int B, int L, int D, const int64_t* strides_g, const int64_t* strides_h, const int64_t* strides_dh,
                   float gate_logit_normalizer, int reverse, int dtype, int32_t* status_dev, void* stream) {
    if (const int e = rec_check(B, L, D, gate_logit_normalizer, dtype)) return e;
    if (!B || !D || !L) return rec_empty(d_final, D, d_h0, D, B, D, (cudaStream_t)stream);
    if (!g || !h || !d_h || !d_x || !d_g) return VIG_ERR_NULL;
    if (walk) if (const int e = rec_states_check(states, B, L, D, dtype)) return e;
    RecParams p{};
    p.states = const_cast<float*>(states); p.walk = walk;
    p.x = d_h; p.g = g; p.h_in = h; p.h0 = h0; p.s0 = d_final; p.ld_s0 = D; p.out = d_x; p.out_g = d_g; p.s_end = d_h0; p.ld_end = D;
    two(p.sx, strides_dh, L, D); two(p.sg, strides_g, L, D); two(p.sh, strides_h, L, D); two(p.so, nullptr, L, D); two(p.sog, nullptr, L, D);
    p.B = B; p.L = L; p.D = D;
    p.inv_norm = gate_logit_normalizer > 0.f ? 1.f / gate_logit_normalizer : 0.f;
    p.from_end = reverse == 0;
    p.status = status_dev;
    return rec_dispatch<true>(p, dtype, (cudaStream_t)stream);
}

extern "C" int vig_gated_recurrence_fwd(const void* x, const void* g, const float* h0, int64_t ld_h0, void* h, float* h_final, int64_t ld_final,
                                        int B, int L, int D, const int64_t* strides_x, const int64_t* strides_g, const int64_t* strides_h,
                                        float gate_logit_normalizer, int reverse, int dtype, int32_t* status_dev, void* stream) {
    return rec_fwd(x, g, h0, ld_h0, h, h_final, ld_final, nullptr, false, B, L, D, strides_x, strides_g, strides_h, gate_logit_normalizer, reverse, dtype, status_dev, stream);
}

extern "C" int vig_gated_recurrence_bwd(const void* g, const void* h, const float* h0, const void* d_h, const float* d_final, void* d_x, void* d_g, float* d_h0,
                                        int B, int L, int D, const int64_t* strides_g, const int64_t* strides_h, const int64_t* strides_dh,
                                        float gate_logit_normalizer, int reverse, int dtype, int32_t* status_dev, void* stream) {
    return rec_bwd(g, h, nullptr, false, h0, d_h, d_final, d_x, d_g, d_h0, B, L, D, strides_g, strides_h, strides_dh, gate_logit_normalizer, reverse, dtype, status_dev, stream);
}

extern "C" int vig_gated_recurrence_train_fwd(const void* x, const void* g, const float* h0, int64_t ld_h0, void* h, float* h_final, int64_t ld_final, float* states,
                                              int B, int L, int D, const int64_t* strides_x, const int64_t* strides_g, const int64_t* strides_h,
                                              float gate_logit_normalizer, int reverse, int dtype, int32_t* status_dev, void* stream) {
    return rec_fwd(x, g, h0, ld_h0, h, h_final, ld_final, states, true, B, L, D, strides_x, strides_g, strides_h, gate_logit_normalizer, reverse, dtype, status_dev, stream);
}

extern "C" int vig_gated_recurrence_train_bwd(const void* g, const void* x, const float* states, const float* h0, const void* d_h, const float* d_final, void* d_x, void* d_g,
                                              float* d_h0, int B, int L, int D, const int64_t* strides_g, const int64_t* strides_x, const int64_t* strides_dh,
                                              float gate_logit_normalizer, int reverse, int dtype, int32_t* status_dev, void* stream) {
    return rec_bwd(g, x, states, true, h0, d_h, d_final, d_x, d_g, d_h0, B, L, D, strides_g, strides_x, strides_dh, gate_logit_normalizer, reverse, dtype, status_dev, stream);
}
