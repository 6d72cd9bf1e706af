// What the forward and the backward of the selective scan share: how the lanes of a warp divide a tile of tokens, and how states go from tile to tile.
//
// A CTA has CT neighbouring channels of one sequence, and each of its warps a tile of 64 tokens at a time: warp w tiles w, w + W, w + 2 W, ...  Within a tile a
// warp takes one channel after the other: lane = 4 * run + part, a run being 8 tokens and a part S of the NB = 4 S states that are gone over together.  So
// the work of a channel and tile is 8 x S products a lane, two values to an instruction (f32x2); the eight runs are joined by a scan over the lanes.
// The state that enters a tile comes from the warp of the tile before through shared memory (`carry`): everything that does not depend on it is done before it
// is waited for, and what the next warp needs is sent on before the outputs are computed.  Warps meet nowhere else: while one waits for its rows,
// others compute.  The maps (B and C, the same for all channels of a group)
// are read once for a tile: the forward keeps them in registers over a warp's channels, the backward in tensor memory, where each lane has a row of its own.
#pragma once
#include "tc_common.cuh"

namespace vig {
namespace scan {

using namespace tc;

constexpr int TILE = 64, RUN = 8, PARTS = 4;
constexpr unsigned ALL = 0xffffffffu;

constexpr float LOG2E_REST = (float)(1.4426950408889634 - (double)LOG2E);   // what log2(e) has behind fp32's digits

template <typename T> __device__ __forceinline__ float param_at(const void* p, int i, int f32) { return f32 ? ((const float*)p)[i] : DType<T>::to_f(((const T*)p)[i]); }

// exp(-|x|) of a pair: what the product with log2(e) loses is put back, or steps of -10 would be 5e-7 off all along a sequence
__device__ __forceinline__ F2 exp_minus_abs(F2 x) {
    // -|x|, and not below where exp is 0 in fp32: a step of -inf, or of a type's lowest value, is one of nothing, and would be inf - inf here
    const F2 ax = f2_make(fmaxf(-fabsf(f2_lo(x)), -150.f), fmaxf(-fabsf(f2_hi(x)), -150.f));
    const F2 k = f2_make(LOG2E, LOG2E), t = f2_mul(ax, k);
    const F2 lost = f2_fma(ax, f2_make(LOG2E_REST, LOG2E_REST), f2_fma(ax, k, t ^ 0x8000000080000000ull));
    const F2 e = f2_make(ex2(f2_lo(t)), ex2(f2_hi(t)));
    return f2_fma(e, f2_mul(lost, f2_make(LN2, LN2)), e);
}
// max(x, 0), which keeps a NaN
__device__ __forceinline__ float positive(float x) { float y; asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x)); return y; }
// Of a pair of values, max(x, 0) + log(1 + e), e = exp(-|x|): a step of 1e-4 has to keep its own precision, so log(1 + e) is e times a polynomial of least
// relative error on [0, 1] (by exchange; 3.3e-8 with the coefficients' digits as they stand, 1.6e-7 in fp32 arithmetic).
__device__ __forceinline__ F2 softplus(F2 x) {
    const F2 e = exp_minus_abs(x);
    constexpr float c[] = {1.f, -0.499999017f, 0.333299637f, -0.249541342f, 0.196759388f, -0.153055921f, 0.106036551f, -0.0569595359f, 0.0198514629f, -0.00324402563f};
    F2 s = f2_make(c[9], c[9]);
#pragma unroll
    for (int i = 8; i >= 0; --i) s = f2_fma(s, e, f2_make(c[i], c[i]));
    return f2_fma(s, e, f2_make(positive(f2_lo(x)), positive(f2_hi(x))));
}
// softplus'(x)
__device__ __forceinline__ float slope(float x) {
    const float e = f2_lo(exp_minus_abs(f2_make(x, x))), r = rcp(1.f + e);
    return x < 0.f ? e * r : r;
}
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-x * LOG2E)); }

// A rate as it is taken: within +-2.3e38, so that its product with log2(e) is finite and with a step of nothing (a token behind the end of a sequence is one)
// leaves a state as it was, where infinity * 0 would be a NaN.  Of a step above 1e-36 such a rate leaves nothing, as an infinite one does.
__device__ __forceinline__ float rate_of(float A) { return A < -2.3e38f ? -2.3e38f : A > 2.3e38f ? 2.3e38f : A; }

// where the row of token t of a tile's map lies: eight lanes that read token j of their runs read eight neighbouring rows
__device__ __forceinline__ int row_of(int t) { return (t % RUN) * RUN + t / RUN; }

__device__ __forceinline__ void copy16(void* dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory"); }
__device__ __forceinline__ void copy8(void* dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory"); }
__device__ __forceinline__ void copy4(void* dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory"); }
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// NC values of a row into shared memory of the lane's own: in pieces of what pointers and strides allow, or one at a time; values from `have` on are zeros
template <typename T, int NC> __device__ __forceinline__ void fetch(T* dst, const T* src, int have, int piece) {
    constexpr int BYTES = NC * (int)sizeof(T);
    if (have >= NC && piece >= 8) {
        if (BYTES % 16 == 0 && piece >= 16) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) copy16((char*)dst + 16 * i, (const char*)src + 16 * i);
        } else {
#pragma unroll
            for (int i = 0; i < BYTES / 8; ++i) copy8((char*)dst + 8 * i, (const char*)src + 8 * i);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) dst[i] = i < have ? src[i] : DType<T>::from_f(0.f);
}

// [64 tokens][Npad] of a map of this tile, by a warp; tokens from `len` on and states from N on are zeros
template <typename T> __device__ __forceinline__ void fetch_map(T* dst, const T* src, int64_t stride, int64_t t0, int len, int N, int Npad, int piece, int lane) {
    if (piece >= 16) {
        const int n16 = Npad * (int)sizeof(T) / 16, have = N * (int)sizeof(T) / 16;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int t = lane + 32 * r;
            char* to = (char*)(dst + row_of(t) * Npad);
            const char* from = (const char*)(src + (t0 + t) * stride);
            for (int k = 0; k < n16; ++k) {
                if (t0 + t < len && k < have) copy16(to + 16 * k, from + 16 * k);
                else *(uint4*)(to + 16 * k) = make_uint4(0u, 0u, 0u, 0u);
            }
        }
    } else if (piece >= 4) {
        const int words = Npad * (int)sizeof(T) / 4, have = N * (int)sizeof(T) / 4;
        for (int t = lane; t < TILE; t += 32) {
            char* to = (char*)(dst + row_of(t) * Npad);
            const char* from = (const char*)(src + (t0 + t) * stride);
#pragma unroll 4
            for (int k = 0; k < words; ++k) {
                if (t0 + t < len && k < have) copy4(to + 4 * k, from + 4 * k);
                else *(uint32_t*)(to + 4 * k) = 0u;
            }
        }
    } else {
        for (int t = lane; t < TILE; t += 32)
            for (int n = 0; n < Npad; ++n) dst[row_of(t) * Npad + n] = t0 + t < len && n < N ? src[(t0 + t) * stride + n] : DType<T>::from_f(0.f);
    }
}

// a row's words as they lie in shared memory
template <int WORDS> __device__ __forceinline__ void words(uint32_t* to, const void* from) {
    if constexpr (WORDS % 4 == 0) {
#pragma unroll
        for (int i = 0; i < WORDS / 4; ++i) { const uint4 w = ((const uint4*)from)[i]; to[4 * i] = w.x; to[4 * i + 1] = w.y; to[4 * i + 2] = w.z; to[4 * i + 3] = w.w; }
    } else {
#pragma unroll
        for (int i = 0; i < WORDS / 2; ++i) { const uint2 w = ((const uint2*)from)[i]; to[2 * i] = w.x; to[2 * i + 1] = w.y; }
    }
}

// NC values of a row into registers: in pieces of what pointers and strides allow, or one at a time; values from `have` on are zeros
template <typename T, int NC> __device__ __forceinline__ void read(float* f, const T* src, int have, int piece) {
    constexpr int BYTES = NC * (int)sizeof(T);
    T e[NC];
    if (have >= NC && piece >= 8) {
        if (BYTES % 16 == 0 && piece >= 16) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) { const uint4 w = ((const uint4*)src)[i]; memcpy((char*)e + 16 * i, &w, 16); }
        } else {
#pragma unroll
            for (int i = 0; i < BYTES / 8; ++i) { const uint2 w = ((const uint2*)src)[i]; memcpy((char*)e + 8 * i, &w, 8); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NC; ++i) e[i] = i < have ? src[i] : DType<T>::from_f(0.f);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) f[i] = DType<T>::to_f(e[i]);
}

// NC values out of registers, as far as they exist
template <typename T, int NC> __device__ __forceinline__ void put(T* dst, const float* v, int have, int piece) {
    T e[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) e[i] = DType<T>::from_f(v[i]);
    constexpr int BYTES = NC * (int)sizeof(T);
    if (have >= NC && piece >= 8) {
        if (BYTES % 16 == 0 && piece >= 16) {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) { uint4 w; memcpy(&w, (const char*)e + 16 * i, 16); ((uint4*)dst)[i] = w; }
        } else {
#pragma unroll
            for (int i = 0; i < BYTES / 8; ++i) { uint2 w; memcpy(&w, (const char*)e + 8 * i, 8); ((uint2*)dst)[i] = w; }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) if (i < have) dst[i] = e[i];
}

// One value for each of 8 tokens and 4 parts, summed over the parts; part p keeps tokens 2 p and 2 p + 1
__device__ __forceinline__ float2 over_parts(const float* v, int part) {
    float w[4];
    const bool hi = part & 2, odd = part & 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (hi ? v[4 + i] : v[i]) + __shfl_xor_sync(ALL, hi ? v[i] : v[4 + i], 2);
    float2 r;
    r.x = (odd ? w[2] : w[0]) + __shfl_xor_sync(ALL, odd ? w[0] : w[2], 1);
    r.y = (odd ? w[3] : w[1]) + __shfl_xor_sync(ALL, odd ? w[1] : w[3], 1);
    return r;
}

__device__ __forceinline__ F2 f2_shfl_up(F2 v, int lanes) { return f2_make(__shfl_up_sync(ALL, f2_lo(v), lanes), __shfl_up_sync(ALL, f2_hi(v), lanes)); }
__device__ __forceinline__ F2 f2_shfl_down(F2 v, int lanes) { return f2_make(__shfl_down_sync(ALL, f2_lo(v), lanes), __shfl_down_sync(ALL, f2_hi(v), lanes)); }
__device__ __forceinline__ F2 f2_shfl(F2 v, int lane) { return f2_make(__shfl_sync(ALL, f2_lo(v), lane), __shfl_sync(ALL, f2_hi(v), lane)); }

// The unit's 2^x is below the value by 0.1 to 0.5 of 2^-24 on average over arguments from 0 to -0.6, and tokens of like steps multiply that up.  Its argument, rounded once with
// the product, is raised by what makes 0.2 of it good, which leaves between -0.27 and 0.12 and 2^0 = 1: dA of training 8 x 1024 x 256 x 16 fp32 1.6e-6 -> 7.6e-7
// from 64 bits (5.7e-7 with expf), at the same time.
constexpr float EX2_LOW = 0.2f / 16777216.f * LOG2E;

// decays of a run, exp(delta A) with A in log2 units
template <int S> __device__ __forceinline__ void decays(F2 (*a)[S / 2], const float* delta, const F2* A2) {
#pragma unroll
    for (int j = 0; j < RUN; ++j)
#pragma unroll
        for (int s = 0; s < S / 2; ++s) {
            const F2 x = f2_fma(f2_make(delta[j], delta[j]), A2[s], f2_make(EX2_LOW, EX2_LOW));
            a[j][s] = f2_make(ex2(f2_lo(x)), ex2(f2_hi(x)));
        }
}

// A run's own sum E of h = a h + b, from nothing, and the product P of its decays
template <int S> __device__ __forceinline__ void own_sum(F2* P, F2* E, const F2 (*a)[S / 2], const F2 (*b)[S / 2]) {
#pragma unroll
    for (int j = 0; j < RUN; ++j)
#pragma unroll
        for (int s = 0; s < S / 2; ++s) {
            E[s] = j ? f2_fma(a[j][s], E[s], b[j][s]) : b[j][s];
            P[s] = j ? f2_mul(P[s], a[j][s]) : a[j][s];
        }
}

// 0, or NaN where a run's product of decays is past 2^32: of four it might leave the range.  Asked only where decays may be growth at all.
__device__ __forceinline__ F2 grown(F2 P) {
    const F2 two = f2_mul(P, P);
    return f2_mul(f2_mul(two, two), 0ull);
}

// The states that enter each lane's run, of Q channels, from the runs' own sums and the states h0 that enter the tile; E of the last run becomes what leaves the
// tile.  Runs are joined over the lanes by doubling.  An infinite state times a product that has left the type's range would be a NaN where the recurrence
// token by token keeps the infinity, and so would be a state of nothing times decays that grow (A above 0, or negative steps) past the range: with a sum that is
// not finite, or (`grows`: where a decay may be above 1) a run's product past 2^32, of which four are multiplied, the runs follow one another.
template <int S, int Q>
__device__ __forceinline__ void entering(F2 (*in)[S / 2], F2 (*E)[S / 2], F2 (*P)[S / 2], const F2 (*h0)[S / 2], const F2 (*a)[RUN][S / 2], const F2 (*b)[RUN][S / 2], int run, int part, bool grows) {
    F2 probe = 0ull;                                             // 0, or NaN
    if (grows) {
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int s = 0; s < S / 2; ++s) probe = f2_add(probe, grown(P[q][s]));
    }
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int s = 0; s < S / 2; ++s) probe = f2_fma(h0[q][s], 0ull, f2_fma(E[q][s], 0ull, probe));
    if (__any_sync(ALL, !(f2_lo(probe) + f2_hi(probe) == 0.f))) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            F2 now[S / 2];
#pragma unroll
            for (int s = 0; s < S / 2; ++s) now[s] = h0[q][s];
#pragma unroll 1
            for (int r = 0; r < RUN; ++r) {
                F2 end[S / 2];
#pragma unroll
                for (int s = 0; s < S / 2; ++s) { if (run == r) in[q][s] = now[s]; end[s] = now[s]; }
#pragma unroll
                for (int j = 0; j < RUN; ++j)
#pragma unroll
                    for (int s = 0; s < S / 2; ++s) end[s] = f2_fma(a[q][j][s], end[s], b[q][j][s]);
#pragma unroll
                for (int s = 0; s < S / 2; ++s) now[s] = f2_shfl(end[s], r * PARTS + part);
            }
#pragma unroll
            for (int s = 0; s < S / 2; ++s) E[q][s] = now[s];
        }
        return;
    }
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int s = 0; s < S / 2; ++s) E[q][s] = f2_fma(P[q][s], run == 0 ? h0[q][s] : 0ull, E[q][s]);
#pragma unroll
    for (int d = 1; d < RUN; d *= 2)
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int s = 0; s < S / 2; ++s) {
                const F2 e = f2_shfl_up(E[q][s], d * PARTS);
                E[q][s] = f2_fma(P[q][s], run >= d ? e : 0ull, E[q][s]);
                if (2 * d < RUN) P[q][s] = f2_mul(P[q][s], f2_shfl_up(P[q][s], d * PARTS));
            }
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int s = 0; s < S / 2; ++s) {
            const F2 e = f2_shfl_up(E[q][s], PARTS);
            in[q][s] = run == 0 ? h0[q][s] : e;
        }
}

// What a tile's warp leaves for the warp of the next one, with a word that counts the tiles that are through.  The word is polled: a wait on an mbarrier of shared
// memory resumes too late for steps of a few hundred cycles (8 x 4096 x 768 2.3 ms for 1.7).  A wait is bounded; one that runs out raises the status
// and the CTA's flag, after which nobody waits any more.  Lanes leave together, because instructions on tensor memory follow that want the whole warp.
struct Handover {
    volatile int* given_up;
    int32_t* status;
    __device__ __forceinline__ void await(const uint32_t* flag, uint32_t want) const {
        const uint32_t addr = smem_u32(flag);
#pragma unroll 1
        for (uint32_t i = 0;; ++i) {
            uint32_t got;
            asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(got) : "r"(addr) : "memory");
            if (got == want) break;
            if ((i & 63u) == 63u && (i >= (1u << 24) || *given_up)) {
                *given_up = 1;
                if (status) atomicOr(status, 1);
                break;
            }
        }
        __syncwarp();
    }
    __device__ __forceinline__ void pass(uint32_t* flag, uint32_t value) const {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(smem_u32(flag)), "r"(value) : "memory");
    }
};

// Tensor memory, 16 or 32 columns of a lane's own row: the whole warp at once, and nothing that takes the values is moved ahead of the wait
template <int N> __device__ __forceinline__ void recall(uint32_t from, float* v) {
    __syncwarp();
    if constexpr (N == 32) tc_ld32(from, v);
    else tc_ld16(from, v);
}
template <int N> __device__ __forceinline__ void landed(float* v) {
    __syncwarp();
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < N; i += 8)
        asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]), "+f"(v[i + 6]), "+f"(v[i + 7]));
}
template <int N> __device__ __forceinline__ void keep(uint32_t to, const float* v) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < N; i += 16) tc_st16(to + i, (const uint32_t*)v + i);
}
__device__ __forceinline__ void kept() {
    __syncwarp();
    tc_wait_st();
}

// ... and, at the barrier that this takes, whether `any` holds for one of the CTA's threads
__device__ __forceinline__ uint32_t tmem_take(uint32_t* slot, int columns, bool& any) {
    __syncwarp();
    if (threadIdx.x < 32) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    any = __syncthreads_or(any);
    tc_fence_after();
    return *slot;
}
__device__ __forceinline__ void tmem_give(uint32_t tmem, int columns) {
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x < 32) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
    }
}

// S states of a lane's 8 tokens of a map, out of global memory; tokens from `len` on and states from N on are zeros
template <typename T, int S> __device__ __forceinline__ void map_of(float* m, const T* src, int64_t stride, int64_t t0, int len, int n, int N, int piece) {
    constexpr int BYTES = S * (int)sizeof(T);
    const bool whole = n + S <= N && piece >= BYTES;
#pragma unroll
    for (int j = 0; j < RUN; ++j) {
        const T* from = src + (t0 + j) * stride + n;
        T e[S];
#pragma unroll
        for (int s = 0; s < S; ++s) e[s] = DType<T>::from_f(0.f);
        if (t0 + j < len) {
            if (whole) {
                if constexpr (BYTES == 16) { const uint4 w = *(const uint4*)from; memcpy(e, &w, 16); }
                else if constexpr (BYTES == 8) { const uint2 w = *(const uint2*)from; memcpy(e, &w, 8); }
                else { const uint32_t w = *(const uint32_t*)from; memcpy(e, &w, 4); }
            } else {
#pragma unroll
                for (int s = 0; s < S; ++s) if (n + s < N) e[s] = from[s];
            }
        }
#pragma unroll
        for (int s = 0; s < S; ++s) m[j * S + s] = DType<T>::to_f(e[s]);
    }
}

// S values of a row in shared memory, as pairs
template <typename T, int S> __device__ __forceinline__ void pairs(F2* out, const T* row) {
    T e[S];
    if constexpr (S * sizeof(T) == 16) { const uint4 w = *(const uint4*)row; memcpy(e, &w, 16); }
    else if constexpr (S * sizeof(T) == 8) { const uint2 w = *(const uint2*)row; memcpy(e, &w, 8); }
    else { const uint32_t w = *(const uint32_t*)row; memcpy(e, &w, 4); }
#pragma unroll
    for (int s = 0; s < S / 2; ++s) out[s] = f2_make(DType<T>::to_f(e[2 * s]), DType<T>::to_f(e[2 * s + 1]));
}

struct Params {
    const void *u, *dt, *z, *b, *c, *skip, *bias, *dy;
    const float *A, *h0, *d_final;
    const int32_t* lengths;
    void *y, *d_u, *d_dt, *d_z;
    float *h_final, *states, *d_h0;
    float *part_b, *part_c, *part_A, *part_skip, *part_bias;     // shares of the gradients that are sums: [channel tiles of a group][B, L, G, N], [B][D, N], [B][D]
    int64_t s_u[2], s_dt[2], s_z[2], s_y[2], s_dy[2], s_b[3], s_c[3], ld_h0, ld_final;
    int B, L, D, N, G, skip_f32, bias_f32, softplus;
    int32_t* status;
    int tiles, ctiles;                                           // tiles of tokens; CTAs of a group's channels
    int piece, piece_maps;                                       // bytes of a copy that pointers and strides allow: rows, maps
};

// a length is a number from 0 to L, whatever the caller's memory holds
__device__ __forceinline__ int length_of(const Params& p, int b) { return p.lengths ? min(max(p.lengths[b], 0), p.L) : p.L; }

}  // namespace scan
}  // namespace vig
