// Selective scan: states h[d, n] of D channels with N states each, driven by inputs u, steps delta and maps B, C that change from token to token.
//
//   delta_t = softplus(dt_t + bias)   (or dt_t + bias),   h_t[d, n] = exp(delta_t[d] A[d, n]) h_{t-1}[d, n] + delta_t[d] u_t[d] B_t[n],
//   y_t[d] = (sum_n C_t[n] h_t[d, n] + D[d] u_t[d]) silu(z_t[d]).
//
// Every (token, channel, state) costs an exponential and three multiply-adds, every (token, channel) three 16-bit values in and one out: with 16
// states the exponentials bound it (MUFU, 16 a cycle and SM), not memory.  So each is taken once: the warps of a CTA take tiles of the same channels'
// tokens in turn and hand the state from tile to tile, within a tile a warp's lanes divide tokens and states (scan_common.cuh); two passes over
// independent chunks would take every exponential twice.  1 x 16384 x 768 x 16 bf16 306 us, 8 x 4096 x 768 x 16 336 (45 and 90 by the exponentials), training the
// latter 383 + 1055 + 45: issue slots at 41 to 45 %, ten warps an SM, 15 instructions a (token, channel, state) forward and 41 backward, the polls among them.
// Sixteen channels and four warps is the backward's only shape: one long sequence, 1 x 16384 x 768, leaves it 48 CTAs and takes 346 + 2852 + 23.
#include <type_traits>
#include "scan_common.cuh"

namespace vig {
using namespace scan;

// A CTA's shared memory: for every warp the rows and maps of its next tile, which are under way while it works on one, and steps and inputs a channel at a
// time; A, the states between tiles and their flags, bias and skip.  Of the tile at hand, u and z wait for the outputs in tensor memory.
template <typename T, int S, int CT> struct FwdSmem {
    static constexpr int NB = PARTS * S, ROWS = TILE * CT * (int)sizeof(T);
    static constexpr int STASH = 2 * CT * (int)sizeof(T) / 4, COLUMNS = 2 * (STASH < 16 ? 16 : STASH);   // words of a row's u and z; of both rows of a lane
    static __host__ __device__ int padded(int N) { return (N + NB - 1) / NB * NB; }
    static __host__ __device__ int warp_bytes(int N) {
        const int Np = padded(N);
        return 3 * ROWS + 2 * TILE * Np * (int)sizeof(T) + (Np > NB ? 3 : 2) * CT * TILE * 4;
    }
    static int bytes(int N, int W) { return W * warp_bytes(N) + (2 * CT * padded(N) + CT * padded(N) / NB + 2 * CT + 4) * 4; }
};

// LEAVE: the states that enter each tile are written too, for a backward
template <typename T, int S, int CT, int W, bool LEAVE>
__global__ void __launch_bounds__(32 * W, (S == 4 ? 12 : 16) / W) scan_fwd_kernel(const Params p) {
    using M = FwdSmem<T, S, CT>;
    constexpr int NB = M::NB, THREADS = 32 * W, HALF = M::STASH / 2;
    extern __shared__ __align__(16) char room[];
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, run = lane / PARTS, part = lane % PARTS;
    const int Npad = M::padded(p.N), Dg = p.D / p.G;
    const int ct = blockIdx.x % p.ctiles, g = blockIdx.x / p.ctiles % p.G, b = blockIdx.x / p.ctiles / p.G;
    const int c0 = ct * CT, have = min(CT, Dg - c0), d = g * Dg + c0;             // channels of the CTA, the first one's index
    const int len = length_of(p, b), ntiles = (len + TILE - 1) / TILE;
    char* const mine = room + warp * M::warp_bytes(p.N);
    T *const ru = (T*)mine, *const rdt = ru + TILE * CT, *const rz = rdt + TILE * CT, *const mB = rz + TILE * CT, *const mC = mB + TILE * Npad;
    float *const delta = (float*)(mC + TILE * Npad), *const x = delta + CT * TILE;
    float* const ys = Npad > NB ? x + CT * TILE : delta;         // with one block of states a channel's steps are done with when its sums are there
    float *const sA = (float*)(room + W * M::warp_bytes(p.N)), *const carry = sA + CT * Npad, *const bias = carry + CT * Npad, *const skip = bias + CT;
    uint32_t* const flags = (uint32_t*)(skip + CT);
    int* const given_up = (int*)(flags + CT * Npad / NB);
    const Handover hand{given_up, p.status};

    const float none = p.softplus ? -1.f : 0.f;                  // a state that is not there: a step of +inf leaves nothing of it, and no NaN, which would go back to all tokens ahead
    bool grows = !p.softplus;                                    // whether a decay may be above 1
    for (int i = tid; i < CT * Npad; i += THREADS) {
        const int c = i / Npad, n = i - c * Npad;
        const bool in = c < have && n < p.N;
        sA[i] = in ? rate_of(p.A[(int64_t)(d + c) * p.N + n]) * LOG2E : none;
        grows |= sA[i] > 0.f;
        carry[i] = in && p.h0 ? p.h0[b * p.ld_h0 + (int64_t)(d + c) * p.N + n] : 0.f;
    }
    for (int i = tid; i < CT; i += THREADS) {
        bias[i] = p.bias && i < have ? param_at<T>(p.bias, d + i, p.bias_f32) : 0.f;
        skip[i] = p.skip && i < have ? param_at<T>(p.skip, d + i, p.skip_f32) : 0.f;
    }
    for (int i = tid; i < CT * Npad / NB; i += THREADS) flags[i] = 0;
    if (tid == 0) *given_up = 0;
    const uint32_t tmem_base = tmem_take(&tmem_slot, (W > 4 ? 2 : 1) * M::COLUMNS, grows);
    const uint32_t tmem = tmem_base + ((uint32_t)(32 * (warp & 3)) << 16) + (warp >> 2) * M::COLUMNS;
    const T *u = (const T*)p.u + b * p.s_u[0] + d, *dt = (const T*)p.dt + b * p.s_dt[0] + d, *z = p.z ? (const T*)p.z + b * p.s_z[0] + d : nullptr;
    const T *gB = (const T*)p.b + b * p.s_b[0] + g * p.s_b[2], *gC = (const T*)p.c + b * p.s_c[0] + g * p.s_c[2];
    T* const y = (T*)p.y + b * p.s_y[0] + d;
    auto bring = [&](int tile) {
        const int64_t t0 = (int64_t)tile * TILE;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int t = lane + 32 * r;
            if (t0 + t < len) {
                fetch<T, CT>(rdt + t * CT, dt + (t0 + t) * p.s_dt[1], have, p.piece);
                fetch<T, CT>(ru + t * CT, u + (t0 + t) * p.s_u[1], have, p.piece);
                if (z) fetch<T, CT>(rz + t * CT, z + (t0 + t) * p.s_z[1], have, p.piece);
            }
        }
        fetch_map<T>(mB, gB, p.s_b[1], t0, len, p.N, Npad, p.piece_maps, lane);
        fetch_map<T>(mC, gC, p.s_c[1], t0, len, p.N, Npad, p.piece_maps, lane);
    };
    if (warp < ntiles) bring(warp);
    const bool whole = p.N % (PARTS * S) == 0 && (uintptr_t)p.states % 16 == 0;

    for (int tile = warp; tile < ntiles; tile += W) {
        const int64_t t0 = (int64_t)tile * TILE;
        float* const left = LEAVE ? p.states + (((int64_t)b * p.tiles + tile) * p.D + d) * p.N + part * S : nullptr;
        copies_done();
        __syncwarp();
#pragma unroll 1
        for (int r = 0; r < 2; ++r) {
            const int t = lane + 32 * r;
            const bool in = t0 + t < len;                        // behind the end a token changes nothing
            alignas(16) uint32_t stash[M::COLUMNS / 2];
            words<HALF>(stash, ru + t * CT);
            words<HALF>(stash + HALF, rz + t * CT);
            keep<M::COLUMNS / 2>(tmem + r * (M::COLUMNS / 2), (const float*)stash);
            float uf[CT], df[CT];
            read<T, CT>(uf, ru + t * CT, CT, 16);
            read<T, CT>(df, rdt + t * CT, CT, 16);
#pragma unroll
            for (int c = 0; c < CT; c += 2) {
                F2 dl = f2_add(f2_make(df[c], df[c + 1]), *(const F2*)(bias + c));
                if (p.softplus) dl = softplus(dl);
                const F2 xi = f2_mul(dl, f2_make(uf[c], uf[c + 1]));
                delta[c * TILE + t] = in ? f2_lo(dl) : 0.f;
                delta[(c + 1) * TILE + t] = in ? f2_hi(dl) : 0.f;
                x[c * TILE + t] = in ? f2_lo(xi) : 0.f;
                x[(c + 1) * TILE + t] = in ? f2_hi(xi) : 0.f;
            }
        }
        __syncwarp();

        for (int n0 = 0; n0 < Npad; n0 += NB) {
            F2 B[RUN][S / 2], C[RUN][S / 2];
#pragma unroll
            for (int j = 0; j < RUN; ++j) {
                const int at = (j * RUN + run) * Npad + n0 + part * S;
                pairs<T, S>(B[j], mB + at);
                pairs<T, S>(C[j], mC + at);
            }
            __syncwarp();
            if (n0 + NB >= Npad && tile + W < ntiles) bring(tile + W);       // all of this tile is elsewhere by now
            if (W > 1 && !n0 && tile < W) hand.await(flags + have / W, (uint32_t)tile);    // warps begin some channels apart, or each hiccup of one is all the others'
#pragma unroll 1
            for (int c = 0; c < have; ++c) {
                float* const h_at = carry + c * Npad + n0 + part * S;
                uint32_t* const flag = flags + n0 / NB * CT + c;
                F2 A2[S / 2], a[1][RUN][S / 2], in[1][RUN][S / 2], P[1][S / 2], E[1][S / 2], h0[1][S / 2], h[1][S / 2];
                pairs<float, S>(A2, sA + c * Npad + n0 + part * S);
                float dl[RUN], xr[RUN], yv[RUN];
#pragma unroll
                for (int k = 0; k < RUN; k += 4) {
                    *(float4*)(dl + k) = *(const float4*)(delta + c * TILE + run * RUN + k);
                    *(float4*)(xr + k) = *(const float4*)(x + c * TILE + run * RUN + k);
                }
                decays<S>(a[0], dl, A2);
#pragma unroll
                for (int j = 0; j < RUN; ++j)
#pragma unroll
                    for (int s = 0; s < S / 2; ++s) in[0][j][s] = f2_mul(f2_make(xr[j], xr[j]), B[j][s]);
                own_sum<S>(P[0], E[0], a[0], in[0]);
                hand.await(flag, (uint32_t)tile);
                pairs<float, S>(h0[0], h_at);
                entering<S, 1>(h, E, P, h0, a, in, run, part, grows);
                __syncwarp();
                if (run == RUN - 1) {
#pragma unroll
                    for (int s = 0; s < S / 2; ++s) *(F2*)(h_at + 2 * s) = E[0][s];
                }
                hand.pass(flag, (uint32_t)tile + 1);
                if (LEAVE && run == 0) {
                    float* to = left + c * p.N + n0;
                    if (whole) {
                        if constexpr (S == 4) *(ulonglong2*)to = make_ulonglong2(h0[0][0], h0[0][1]);
                        else *(F2*)to = h0[0][0];
                    } else {
#pragma unroll
                        for (int s = 0; s < S; ++s) if (n0 + part * S + s < p.N) to[s] = s & 1 ? f2_hi(h0[0][s / 2]) : f2_lo(h0[0][s / 2]);
                    }
                }
#pragma unroll
                for (int j = 0; j < RUN; ++j) {
                    F2 sum = 0ull;
#pragma unroll
                    for (int s = 0; s < S / 2; ++s) {
                        h[0][s] = f2_fma(a[0][j][s], h[0][s], in[0][j][s]);
                        sum = s ? f2_fma(C[j][s], h[0][s], sum) : f2_mul(C[j][s], h[0][s]);
                    }
                    yv[j] = f2_lo(sum) + f2_hi(sum);
                }
                float2 got = over_parts(yv, part);
                float2* const ya = (float2*)(ys + c * TILE + run * RUN + part * 2);
                if (n0) { const float2 was = *ya; got.x += was.x; got.y += was.y; }
                *ya = got;
            }
        }
        kept();
        __syncwarp();
#pragma unroll 1
        for (int r = 0; r < 2; ++r) {
            const int t = lane + 32 * r;
            alignas(16) uint32_t stash[M::COLUMNS / 2];
            recall<M::COLUMNS / 2>(tmem + r * (M::COLUMNS / 2), (float*)stash);
            landed<M::COLUMNS / 2>((float*)stash);
            if (t0 + t < len) {
                float uf[CT], out[CT];
                read<T, CT>(uf, (const T*)stash, CT, 16);
                if (p.skip) {
#pragma unroll
                    for (int c = 0; c < CT; ++c) out[c] = fmaf(skip[c], uf[c], ys[c * TILE + t]);
                } else {                                         // (0 times an infinite input is a NaN)
#pragma unroll
                    for (int c = 0; c < CT; ++c) out[c] = ys[c * TILE + t];
                }
                if (z) {
                    read<T, CT>(uf, (const T*)(stash + HALF), CT, 16);
#pragma unroll
                    for (int c = 0; c < CT; ++c) out[c] *= uf[c] * sigmoid(uf[c]);
                }
                put<T, CT>(y + (t0 + t) * p.s_y[1], out, have, p.piece);
            }
        }
        __syncwarp();
    }
    // behind the end the outputs are zeros
    for (int64_t at = (int64_t)len + tid; at < p.L; at += THREADS) {
        const float out[CT] = {};
        put<T, CT>(y + at * p.s_y[1], out, have, p.piece);
    }
    tmem_give(tmem_base, (W > 4 ? 2 : 1) * M::COLUMNS);          // (a barrier too)
    if (p.h_final) {
        for (int i = tid; i < CT * Npad; i += THREADS) {
            const int c = i / Npad, n = i - c * Npad;
            if (c < have && n < p.N) p.h_final[b * p.ld_final + (int64_t)(d + c) * p.N + n] = carry[i];
        }
    }
}

// Backward, from the states that enter each tile (the forward wrote them) and the tiles from the last to the first.  With g_t = dL/dh_t,
//   g_t = C_t dy_t + a_{t+1} g_{t+1},  dC_t = sum_d h_t dy_t,  dB_t = sum_d g_t delta_t u_t,  du_t = delta_t sum_n g_t B_t + D dy_t,
//   ddelta_t = sum_n g_t (a_t h_{t-1} A + u_t B_t),  dA = sum g_t a_t h_{t-1} delta_t,
// dy being d_out silu(z).  What goes from tile to tile is a_t g_t of a tile's first token.  A lane keeps the decays and states of its run in registers; the sums
// of the maps' gradients over the CTA's channels are in tensor memory beside the maps.  The shares of CTAs, sequences and warps are added in a fixed order by
// sum_kernel.
constexpr int BS = 2, BNB = PARTS * BS, BCT = 16, BW = 4, BTHREADS = 32 * BW;     // states of a lane, of a block; channels and warps of a CTA

struct BwdSmem {
    static __host__ __device__ int padded(int N) { return (N + BNB - 1) / BNB * BNB; }
    static __host__ __device__ int warp_floats(int N) { return 4 * BCT * TILE + 2 * BCT * padded(N); }
    static int bytes(int N) { return (BW * warp_floats(N) + 2 * BCT * padded(N) + BCT * padded(N) / BNB + 2 * BCT + 2 * BW * BCT + 8) * 4; }
};
// columns of tensor memory: a power of two, 32 at least
static __host__ __device__ int bwd_columns(int N) {
    int c = 64;
    while (c < BwdSmem::padded(N) / BNB * 64) c *= 2;
    return c;
}

// NC values a lane summed over the lanes: lane i has the sum of value i / (32 / NC)
template <int NC> __device__ __forceinline__ float over_lanes(float* v, int lane) {
    int bit = 16;
#pragma unroll
    for (int n = NC / 2; n; n /= 2, bit /= 2) {
        const bool up = lane & bit;
#pragma unroll
        for (int i = 0; i < NC / 2; ++i)
            if (i < n) v[i] = (up ? v[i + n] : v[i]) + __shfl_xor_sync(ALL, up ? v[i] : v[i + n], bit);
    }
    float r = v[0];
#pragma unroll
    for (; bit; bit /= 2) r += __shfl_xor_sync(ALL, r, bit);
    return r;
}

template <typename T>
__global__ void __launch_bounds__(BTHREADS, 3) scan_bwd_kernel(const Params p) {
    constexpr int S = BS, NB = BNB, CT = BCT, W = BW, THREADS = BTHREADS;
    extern __shared__ __align__(16) char smem[];
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, run = lane / PARTS, part = lane % PARTS;
    const int Npad = BwdSmem::padded(p.N), Dg = p.D / p.G, columns = bwd_columns(p.N);
    const int ct = blockIdx.x % p.ctiles, g = blockIdx.x / p.ctiles % p.G, b = blockIdx.x / p.ctiles / p.G;
    const int c0 = ct * CT, have = min(CT, Dg - c0), d = g * Dg + c0;
    const int len = length_of(p, b), ntiles = (len + TILE - 1) / TILE;
    float *const delta = (float*)smem + warp * BwdSmem::warp_floats(p.N), *const x = delta + CT * TILE, *const dys = x + CT * TILE, *const ys = dys + CT * TILE;
    float *const st = ys + CT * TILE, *const dA = st + CT * Npad;          // states that enter the tile; the warp's share of dA
    float *const gb = x, *const ga = dys;                        // sum g B, sum g a h A: where a channel's inputs are done with
    float *const sA = (float*)smem + W * BwdSmem::warp_floats(p.N), *const carry = sA + CT * Npad, *const bias = carry + CT * Npad, *const skip = bias + CT;
    float* const shares = skip + CT;                             // the warps' shares of dD and dbias
    uint32_t* const flags = (uint32_t*)(shares + 2 * W * CT);
    int* const given_up = (int*)(flags + CT * Npad / NB);
    const Handover hand{given_up, p.status};

    const float none = p.softplus ? -1.f : 0.f;                  // a state that is not there: a step of +inf leaves nothing of it, and no NaN, which would go back to all tokens ahead
    bool grows = !p.softplus;                                    // whether a decay may be above 1
    for (int i = tid; i < CT * Npad; i += THREADS) {
        const int c = i / Npad, n = i - c * Npad;
        const bool in = c < have && n < p.N;
        sA[i] = in ? rate_of(p.A[(int64_t)(d + c) * p.N + n]) : none;
        grows |= sA[i] > 0.f;
        carry[i] = in && p.d_final ? p.d_final[((int64_t)b * p.D + d + c) * p.N + n] : 0.f;
    }
    for (int i = lane; i < 2 * CT * Npad; i += 32) st[i] = 0.f;
    for (int i = tid; i < CT; i += THREADS) {
        bias[i] = p.bias && i < have ? param_at<T>(p.bias, d + i, p.bias_f32) : 0.f;
        skip[i] = p.skip && i < have ? param_at<T>(p.skip, d + i, p.skip_f32) : 0.f;
    }
    for (int i = tid; i < CT * Npad / NB; i += THREADS) flags[i] = 0;
    if (tid == 0) *given_up = 0;
    const uint32_t tmem_base = tmem_take(&tmem_slot, columns, grows), tmem = tmem_base + ((uint32_t)(32 * warp) << 16);      // [state block][B, C, dB, dC][8 tokens x 2 states]
    const T *u = (const T*)p.u + b * p.s_u[0] + d, *dt = (const T*)p.dt + b * p.s_dt[0] + d, *z = p.z ? (const T*)p.z + b * p.s_z[0] + d : nullptr;
    const T* dy = (const T*)p.dy + b * p.s_dy[0] + d;
    const T *gB = (const T*)p.b + b * p.s_b[0] + g * p.s_b[2], *gC = (const T*)p.c + b * p.s_c[0] + g * p.s_c[2];
    float sum_skip = 0.f, sum_bias = 0.f;                        // of channel lane / 2

    for (int back = warp; back < ntiles; back += W) {
        const int tile = ntiles - 1 - back;
        const int64_t t0 = (int64_t)tile * TILE;
        const float* from = p.states + (((int64_t)b * p.tiles + tile) * p.D + d) * p.N;
        for (int i = lane; i < have * p.N; i += 32) copy4(st + (p.N == Npad ? i : i / p.N * Npad + i % p.N), from + i);
        for (int n0 = 0; n0 < Npad; n0 += NB) {
            float mb[RUN * S], mc[RUN * S];
            map_of<T, S>(mb, gB, p.s_b[1], t0 + run * RUN, len, n0 + part * S, p.N, p.piece_maps);
            map_of<T, S>(mc, gC, p.s_c[1], t0 + run * RUN, len, n0 + part * S, p.N, p.piece_maps);
            keep<16>(tmem + n0 / NB * 64, mb);
            keep<16>(tmem + n0 / NB * 64 + 16, mc);
#pragma unroll
            for (int k = 0; k < RUN * S; ++k) mb[k] = 0.f;
            keep<16>(tmem + n0 / NB * 64 + 32, mb);
            keep<16>(tmem + n0 / NB * 64 + 48, mb);
        }
        kept();
#pragma unroll 1
        for (int t = lane; t < TILE; t += 32) {
            const bool in = t0 + t < len;
            const int64_t at = in ? t0 + t : t0;
            float uf[CT], df[CT], gf[CT];
            read<T, CT>(uf, u + at * p.s_u[1], have, p.piece);
            read<T, CT>(df, dt + at * p.s_dt[1], have, p.piece);
            read<T, CT>(gf, dy + at * p.s_dy[1], have, p.piece);
#pragma unroll
            for (int c = 0; c < CT; c += 2) {
                F2 dl = f2_add(f2_make(df[c], df[c + 1]), *(const F2*)(bias + c));
                if (p.softplus) dl = softplus(dl);
                const F2 xi = f2_mul(dl, f2_make(uf[c], uf[c + 1]));
                delta[c * TILE + t] = in ? f2_lo(dl) : 0.f;
                delta[(c + 1) * TILE + t] = in ? f2_hi(dl) : 0.f;
                x[c * TILE + t] = in ? f2_lo(xi) : 0.f;
                x[(c + 1) * TILE + t] = in ? f2_hi(xi) : 0.f;
            }
            if (z) {
                read<T, CT>(uf, z + at * p.s_z[1], have, p.piece);
#pragma unroll
                for (int c = 0; c < CT; ++c) gf[c] *= uf[c] * sigmoid(uf[c]);
            }
#pragma unroll
            for (int c = 0; c < CT; ++c) dys[c * TILE + t] = in ? gf[c] : 0.f;
        }
        copies_done();
        __syncwarp();
        // (warps side by side here, not some channels apart as in the forward: they share the instructions that are fetched, 1371 -> 1198 us)

        // CAREFUL: a decay may be above 1, so that products of them may leave the range.  A form of its own: the questions in one form for all cost 7 % (1040 -> 1113 us).
        const auto channel = [&](int c, auto careful) {
            constexpr bool CAREFUL = decltype(careful)::value;
            // read again where they are used: registers are what this kernel is short of
            auto row = [&](float* v, const float* from) {
                *(float4*)v = *(const float4*)(from + c * TILE + run * RUN);
                *(float4*)(v + 4) = *(const float4*)(from + c * TILE + run * RUN + 4);
            };
            float s_y[RUN], s_b[RUN], s_a[RUN];                  // what is summed over the states
#pragma unroll
            for (int j = 0; j < RUN; ++j) s_y[j] = s_b[j] = s_a[j] = 0.f;
#pragma unroll 1
            for (int n0 = 0; n0 < Npad; n0 += NB) {
                const int at = c * Npad + n0 + part * S;
                const uint32_t col = tmem + n0 / NB * 64;
                const int live = p.N - n0 - part * S;            // the lane's states that there are, or more; of the others nothing goes back
                float mb[RUN * S], mc[RUN * S], md[RUN * S], xr[RUN], dr[RUN];
                // g of token j, from what the token behind it gives back
                const auto gradient = [&](int j, const float* dy, F2 q) {
                    const F2 g = f2_make(fmaf(mc[2 * j], dy[j], f2_lo(q)), fmaf(mc[2 * j + 1], dy[j], f2_hi(q)));
                    return CAREFUL ? f2_make(live > 0 ? f2_lo(g) : 0.f, live > 1 ? f2_hi(g) : 0.f) : g;
                };
                recall<16>(col, mb);
                recall<16>(col + 16, mc);
                F2 A[1], P[1], E[1], h0[1], h[RUN + 1][1], a[RUN][1], in[RUN][1], Q = 0ull, Pb;
                pairs<float, S>(A, sA + at);
                {
                    const F2 A2[1] = {f2_mul(A[0], f2_make(LOG2E, LOG2E))};
                    float dl[RUN];
                    row(dl, delta);
                    decays<S>(a, dl, A2);
                }
                row(xr, x);
                row(dr, dys);
                landed<16>(mb);
                landed<16>(mc);
                kept();                                          // what the channel ahead has added, long since
                recall<16>(col + 48, md);
#pragma unroll
                for (int j = 0; j < RUN; ++j) in[j][0] = f2_make(xr[j] * mb[2 * j], xr[j] * mb[2 * j + 1]);
                if (CAREFUL) {
#pragma unroll
                    for (int j = 0; j < RUN; ++j) a[j][0] = f2_make(live > 0 ? f2_lo(a[j][0]) : 0.f, live > 1 ? f2_hi(a[j][0]) : 0.f);
                }
                own_sum<S>(P, E, a, in);
                Pb = P[0];
#pragma unroll
                for (int j = RUN - 1; j >= 0; --j) Q = f2_mul(a[j][0], gradient(j, dr, Q));
                pairs<float, S>(h0, st + at);
                entering<S, 1>(&h[0], &E, &P, &h0, &a, &in, run, part, CAREFUL);
                landed<16>(md);
#pragma unroll
                for (int j = 0; j < RUN; ++j) {
                    h[j + 1][0] = f2_fma(a[j][0], h[j][0], in[j][0]);
                    s_y[j] = fmaf(mc[2 * j], f2_lo(h[j + 1][0]), fmaf(mc[2 * j + 1], f2_hi(h[j + 1][0]), s_y[j]));
                    md[2 * j] = fmaf(f2_lo(h[j + 1][0]), dr[j], md[2 * j]);
                    md[2 * j + 1] = fmaf(f2_hi(h[j + 1][0]), dr[j], md[2 * j + 1]);
                }
                keep<16>(col + 48, md);
                recall<16>(col + 32, md);
                // from the other end: q_t = a_t g_t is what token t - 1 gets
                uint32_t* const flag = flags + n0 / NB * CT + c;
                float* const q_at = carry + at;
                F2 q0[1], behind;                                // what enters the tile; what a run's last token gets
                bool slow = false;
                hand.await(flag, (uint32_t)back);
                pairs<float, S>(q0, q_at);
                if (CAREFUL) {                                   // as in `entering`
                    const F2 probe = f2_fma(q0[0], 0ull, f2_fma(Q, 0ull, grown(Pb)));
                    slow = __any_sync(ALL, !(f2_lo(probe) + f2_hi(probe) == 0.f));
                }
                if (slow) {
                    float dy8[RUN];
                    row(dy8, dys);
                    Q = q0[0];
#pragma unroll 1
                    for (int r = RUN - 1; r >= 0; --r) {
                        if (run == r) behind = Q;
#pragma unroll
                        for (int j = RUN - 1; j >= 0; --j) Q = f2_mul(a[j][0], gradient(j, dy8, Q));
                        Q = f2_shfl(Q, r * PARTS + part);
                    }
                } else {
                    Q = f2_fma(Pb, run == RUN - 1 ? q0[0] : 0ull, Q);
#pragma unroll
                    for (int k = 1; k < RUN; k *= 2) {
                        const F2 e = f2_shfl_down(Q, k * PARTS);
                        Q = f2_fma(Pb, run + k < RUN ? e : 0ull, Q);
                        if (2 * k < RUN) Pb = f2_mul(Pb, f2_shfl_down(Pb, k * PARTS));
                    }
                }
                __syncwarp();
                if (run == 0) *(F2*)q_at = Q;
                hand.pass(flag, (uint32_t)back + 1);
                if (!slow) {
                    const F2 e = f2_shfl_down(Q, PARTS);
                    behind = run == RUN - 1 ? q0[0] : e;
                }
                Q = behind;
                float dl[RUN];
                row(dl, delta);
                row(xr, x);
                row(dr, dys);
                landed<16>(md);
                F2 dAs = 0ull;
#pragma unroll
                for (int j = RUN - 1; j >= 0; --j) {
                    const F2 gr = gradient(j, dr, Q);
                    s_b[j] = fmaf(f2_lo(gr), mb[2 * j], fmaf(f2_hi(gr), mb[2 * j + 1], s_b[j]));
                    md[2 * j] = fmaf(f2_lo(gr), xr[j], md[2 * j]);
                    md[2 * j + 1] = fmaf(f2_hi(gr), xr[j], md[2 * j + 1]);
                    Q = f2_mul(a[j][0], gr);
                    const F2 f = f2_mul(Q, h[j][0]);
                    s_a[j] = fmaf(f2_lo(f), f2_lo(A[0]), fmaf(f2_hi(f), f2_hi(A[0]), s_a[j]));
                    dAs = f2_make(fmaf(f2_lo(f), dl[j], f2_lo(dAs)), fmaf(f2_hi(f), dl[j], f2_hi(dAs)));
                }
                keep<16>(col + 32, md);
                // dA over the runs: a lane of an even run keeps the first state's sum, of an odd one the second's
                const bool odd = run & 1;
                float v = (odd ? f2_hi(dAs) : f2_lo(dAs)) + __shfl_xor_sync(ALL, odd ? f2_lo(dAs) : f2_hi(dAs), PARTS);
                v += __shfl_xor_sync(ALL, v, 2 * PARTS);
                v += __shfl_xor_sync(ALL, v, 4 * PARTS);
                if (run < 2) dA[at + run] += v;
            }
            const int to = c * TILE + run * RUN + part * 2;
            if (z) *(float2*)(ys + to) = over_parts(s_y, part);
            *(float2*)(gb + to) = over_parts(s_b, part);
            *(float2*)(ga + to) = over_parts(s_a, part);
        };
        if (grows) {
#pragma unroll 1
            for (int c = 0; c < have; ++c) channel(c, std::true_type{});
        } else {
#pragma unroll 1
            for (int c = 0; c < have; ++c) channel(c, std::false_type{});
        }
        kept();
        // the tile's maps have their gradients from this CTA's channels
        for (int n0 = 0; n0 < Npad; n0 += NB) {
            float mb[RUN * S], mc[RUN * S];
            recall<16>(tmem + n0 / NB * 64 + 32, mb);
            recall<16>(tmem + n0 / NB * 64 + 48, mc);
            landed<16>(mb);
            landed<16>(mc);
#pragma unroll
            for (int j = 0; j < RUN; ++j) {
                const int64_t at = t0 + run * RUN + j;
                const int64_t to = ((((int64_t)ct * p.B + b) * p.L + at) * p.G + g) * p.N + n0 + part * S;
#pragma unroll
                for (int s = 0; s < S; ++s)
                    if (at < len && n0 + part * S + s < p.N) { p.part_b[to + s] = mb[j * S + s]; p.part_c[to + s] = mc[j * S + s]; }
            }
        }
        float keep_skip[CT], keep_bias[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) keep_skip[c] = keep_bias[c] = 0.f;
#pragma unroll 1
        for (int t = lane; t < TILE; t += 32) {
            if (t0 + t >= len) break;
            const int64_t at = t0 + t, row = ((int64_t)b * p.L + at) * p.D + d;
            float uf[CT], gf[CT], zf[CT], out[CT];
            read<T, CT>(uf, u + at * p.s_u[1], have, p.piece);
            read<T, CT>(gf, dy + at * p.s_dy[1], have, p.piece);
            if (z) {
                read<T, CT>(zf, z + at * p.s_z[1], have, p.piece);
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    const float s = sigmoid(zf[c]);
                    out[c] = gf[c] * fmaf(skip[c], uf[c], ys[c * TILE + t]) * s * fmaf(zf[c], 1.f - s, 1.f);
                    gf[c] *= zf[c] * s;
                }
                put<T, CT>((T*)p.d_z + row, out, have, p.piece);
            }
            if (p.skip) {
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    out[c] = fmaf(gb[c * TILE + t], delta[c * TILE + t], skip[c] * gf[c]);
                    keep_skip[c] = fmaf(gf[c], uf[c], keep_skip[c]);
                }
            } else {                                             // (0 times an infinite gradient is a NaN)
#pragma unroll
                for (int c = 0; c < CT; ++c) out[c] = gb[c * TILE + t] * delta[c * TILE + t];
            }
            put<T, CT>((T*)p.d_u + row, out, have, p.piece);
            if (p.softplus) read<T, CT>(zf, dt + at * p.s_dt[1], have, p.piece);
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                out[c] = fmaf(gb[c * TILE + t], uf[c], ga[c * TILE + t]);
                if (p.softplus) out[c] *= slope(zf[c] + bias[c]);
                keep_bias[c] += out[c];
            }
            put<T, CT>((T*)p.d_dt + row, out, have, p.piece);
        }
        __syncwarp();
        sum_skip += over_lanes<CT>(keep_skip, lane);
        sum_bias += over_lanes<CT>(keep_bias, lane);
    }
    // behind the end all gradients are zeros
    for (int64_t at = (int64_t)len + tid; at < p.L; at += THREADS) {
        const float none[CT] = {};
        const int64_t row = ((int64_t)b * p.L + at) * p.D + d;
        put<T, CT>((T*)p.d_u + row, none, have, p.piece);
        put<T, CT>((T*)p.d_dt + row, none, have, p.piece);
        if (z) put<T, CT>((T*)p.d_z + row, none, have, p.piece);
    }
    for (int64_t i = (int64_t)len * p.N + tid; i < (int64_t)p.L * p.N; i += THREADS) {
        const int64_t at = ((((int64_t)ct * p.B + b) * p.L + i / p.N) * p.G + g) * p.N + i % p.N;
        p.part_b[at] = 0.f;
        p.part_c[at] = 0.f;
    }
    if (!(lane & 1)) { shares[warp * CT + lane / 2] = sum_skip; shares[(W + warp) * CT + lane / 2] = sum_bias; }
    tmem_give(tmem_base, columns);                               // (a barrier too)
    for (int i = tid; i < CT * Npad; i += THREADS) {
        const int c = i / Npad, n = i - c * Npad;
        if (c < have && n < p.N) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) v += dA[(w - warp) * BwdSmem::warp_floats(p.N) + i];
            const int64_t at = ((int64_t)b * p.D + d + c) * p.N + n;
            p.part_A[at] = v;
            if (p.d_h0) p.d_h0[at] = carry[i];
        }
    }
    if (tid < have) {
        float v = 0.f, v2 = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) { v += shares[w * CT + tid]; v2 += shares[(W + w) * CT + tid]; }
        p.part_skip[(int64_t)b * p.D + d + tid] = v;
        p.part_bias[(int64_t)b * p.D + d + tid] = v2;
    }
}

// dst[i] = sum over k of src[k][i], in the order of k
struct SumJob { const float* src; void* dst; int64_t n; int count, type, blocks; };
struct SumJobs { SumJob job[5]; };

__global__ void __launch_bounds__(256) sum_kernel(const SumJobs jobs) {
    pdl_wait();
    int block = blockIdx.x, k = 0;
    while (k < 4 && block >= jobs.job[k].blocks) block -= jobs.job[k++].blocks;
    const SumJob& j = jobs.job[k];
    const int64_t i = (int64_t)block * 256 + threadIdx.x;
    if (i >= j.n) return;
    float v = 0.f;
#pragma unroll 8
    for (int c = 0; c < j.count; ++c) v += j.src[c * j.n + i];
    if (j.type == VIG_DTYPE_F32) ((float*)j.dst)[i] = v;
    else if (j.type == VIG_DTYPE_BF16) ((__nv_bfloat16*)j.dst)[i] = __float2bfloat16_rn(v);
    else ((__half*)j.dst)[i] = __float2half_rn(v);
}

// One token: four lanes of a (sequence, channel) take its states four at a time.  All a lane needs is under way before the first of it is used.
struct StepParams {
    const void *u, *dt, *z, *b, *c, *skip, *bias;
    const float* A;
    float* state;
    void* y;
    int64_t s_u, s_dt, s_z, s_y, s_b[2], s_c[2], ld_state;
    int B, D, N, G, skip_f32, bias_f32, softplus, whole;
};

template <typename T> __global__ void __launch_bounds__(128) scan_step_kernel(const StepParams p) {
    const int64_t i = ((int64_t)blockIdx.x * 128 + threadIdx.x) / 4, last = (int64_t)p.B * p.D - 1;
    const int part = threadIdx.x % 4, b = (int)(min(i, last) / p.D), d = (int)(min(i, last) % p.D);
    const bool in = i <= last;
    const T *mb = (const T*)p.b + b * p.s_b[0] + d / (p.D / p.G) * p.s_b[1], *mc = (const T*)p.c + b * p.s_c[0] + d / (p.D / p.G) * p.s_c[1];
    float* h = p.state + b * p.ld_state + (int64_t)d * p.N;
    const float* A = p.A + (int64_t)d * p.N;
    const float u = DType<T>::to_f(((const T*)p.u)[b * p.s_u + d]), zv = p.z ? DType<T>::to_f(((const T*)p.z)[b * p.s_z + d]) : 0.f;
    float dl = DType<T>::to_f(((const T*)p.dt)[b * p.s_dt + d]) + (p.bias ? param_at<T>(p.bias, d, p.bias_f32) : 0.f);
    const float skip = p.skip ? param_at<T>(p.skip, d, p.skip_f32) : 0.f;
    if (p.softplus) dl = f2_lo(softplus(f2_make(dl, dl)));
    const float x = dl * u;
    float y = 0.f;
    for (int n0 = part * 4; n0 < p.N; n0 += 16) {
        float hv[4], av[4], bv[4], cv[4];
        const bool whole = p.whole && n0 + 4 <= p.N;
        if (whole) {
            *(float4*)hv = *(const float4*)(h + n0);
            *(float4*)av = *(const float4*)(A + n0);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool ok = n0 + k < p.N;
            bv[k] = ok ? DType<T>::to_f(mb[n0 + k]) : 0.f;
            cv[k] = ok ? DType<T>::to_f(mc[n0 + k]) : 0.f;
            if (!whole) { hv[k] = ok ? h[n0 + k] : 0.f; av[k] = ok ? A[n0 + k] : 0.f; }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            hv[k] = fmaf(ex2(fmaf(dl, rate_of(av[k]) * LOG2E, EX2_LOW)), hv[k], x * bv[k]);
            y = fmaf(cv[k], hv[k], y);
        }
        if (in) {
            if (whole) {
                *(float4*)(h + n0) = *(const float4*)hv;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) if (n0 + k < p.N) h[n0 + k] = hv[k];
            }
        }
    }
    y += __shfl_xor_sync(ALL, y, 2);
    y += __shfl_xor_sync(ALL, y, 1);
    if (in && part == 0) {
        if (p.skip) y = fmaf(skip, u, y);
        if (p.z) y *= zv * sigmoid(zv);
        ((T*)p.y)[b * p.s_y + d] = DType<T>::from_f(y);
    }
}

static int piece_of(int64_t value) { return value % 16 == 0 ? 16 : value % 8 == 0 ? 8 : value % 4 == 0 ? 4 : 1; }
static void narrow(int& piece, const void* ptr, const int64_t* strides, int count, int size) {
    if (!ptr) return;
    piece = min(piece, piece_of((int64_t)(uintptr_t)ptr));
    for (int i = 0; i < count; ++i) piece = min(piece, piece_of(strides[i] * size));
}
template <typename T, int S, int CT, int W> int fwd_launch(Params& p, cudaStream_t s) {
    p.ctiles = (p.D / p.G + CT - 1) / CT;
    const int64_t grid = (int64_t)p.B * p.G * p.ctiles;
    const int smem = FwdSmem<T, S, CT>::bytes(p.N, W);
    if (grid >= (1ll << 31)) return VIG_ERR_SHAPE;
    const auto kernel = p.states ? scan_fwd_kernel<T, S, CT, W, true> : scan_fwd_kernel<T, S, CT, W, false>;
    if (const cudaError_t e = ensure_smem_attr((const void*)kernel, smem)) return (int)e;
    kernel<<<(unsigned)grid, 32 * W, smem, s>>>(p);
    return (int)cudaGetLastError();
}
template <typename T> int bwd_launch(Params& p, cudaStream_t s) {
    const int64_t grid = (int64_t)p.B * p.G * p.ctiles;
    const int smem = BwdSmem::bytes(p.N);
    if (grid >= (1ll << 31)) return VIG_ERR_SHAPE;
    if (const cudaError_t e = ensure_smem_attr((const void*)scan_bwd_kernel<T>, smem)) return (int)e;
    scan_bwd_kernel<T><<<(unsigned)grid, BTHREADS, smem, s>>>(p);
    return (int)cudaGetLastError();
}

// Sixteen channels a CTA where that gives every SM two CTAs, else eight, or four with more warps along the tokens (a warp by itself takes 5 cycles an
// instruction: 1 x 16384 x 768 1004 / 531 / 303 us; 16 x 4096 x 768 711 / 705 / 817).
template <typename T, int S> int fwd_width(Params& p, cudaStream_t s) {
    const int64_t wide = (int64_t)p.B * p.G * ((p.D / p.G + 15) / 16);
    // one or two tiles are one or two warps' work: the others of a CTA would only hold its registers (64 x 64 x 768 x 16 170 us with four warps, 75 with one)
    if (p.tiles <= 1) return wide >= 4 * device_sms() ? fwd_launch<T, S, 16, 1>(p, s) : fwd_launch<T, S, 4, 1>(p, s);
    if (p.tiles == 2 && wide >= 4 * device_sms()) return fwd_launch<T, S, 16, 2>(p, s);
    const auto fits = [&](int bytes) { return bytes <= 227 * 1024; };      // (maps of many states in fp32)
    if (wide >= 2 * device_sms() && fits(FwdSmem<T, S, 16>::bytes(p.N, 4))) return fwd_launch<T, S, 16, 4>(p, s);
    if (wide >= device_sms() || !fits(FwdSmem<T, S, 4>::bytes(p.N, 6))) return fwd_launch<T, S, 8, 4>(p, s);
    return fwd_launch<T, S, 4, 6>(p, s);
}

static int check(const vig_selective_scan_args* a, bool grads) {
    if (!a) return VIG_ERR_NULL;
    const auto type_ok = [&](int t) { return t == a->dtype || t == VIG_DTYPE_F32; };
    if (a->dtype < VIG_DTYPE_F32 || a->dtype > VIG_DTYPE_F16 || (a->skip && !type_ok(a->skip_dtype)) || (a->dt_bias && !type_ok(a->bias_dtype))) return VIG_ERR_DTYPE;
    if (a->B < 0 || a->L < 0 || a->D < 0 || a->N < 1 || a->N > 64 || a->G < 1 || a->D % a->G) return VIG_ERR_SHAPE;
    if ((int64_t)a->B * a->D >= (1ll << 31) || a->D >= (1 << 28) || a->L >= (1 << 30)) return VIG_ERR_SHAPE;
    if (!a->B || !a->D) return VIG_OK;
    if (!a->A || (a->L && (!a->u || !a->dt || !a->b || !a->c || (!grads && !a->y)))) return VIG_ERR_NULL;
    if (grads && (!a->d_A || (a->L && (!a->d_b || !a->d_c || !a->states || !a->d_y || !a->d_u || !a->d_dt || (a->z && !a->d_z))))) return VIG_ERR_NULL;
    return VIG_OK;
}

static Params params_of(const vig_selective_scan_args* a, bool grads) {
    Params p{};
    p.u = a->u; p.dt = a->dt; p.z = a->z; p.b = a->b; p.c = a->c; p.skip = a->skip; p.bias = a->dt_bias; p.dy = a->d_y;
    p.A = a->A; p.h0 = a->h0; p.d_final = a->d_final; p.lengths = a->lengths; p.y = a->y; p.d_u = a->d_u; p.d_dt = a->d_dt; p.d_z = a->d_z;
    p.h_final = a->h_final; p.states = a->states; p.d_h0 = a->d_h0;
    for (int i = 0; i < 2; ++i) { p.s_u[i] = a->s_u[i]; p.s_dt[i] = a->s_dt[i]; p.s_z[i] = a->s_z[i]; p.s_y[i] = a->s_y[i]; p.s_dy[i] = a->s_dy[i]; }
    for (int i = 0; i < 3; ++i) { p.s_b[i] = a->s_b[i]; p.s_c[i] = a->s_c[i]; }
    p.ld_h0 = a->ld_h0; p.ld_final = a->ld_final;
    p.B = a->B; p.L = a->L; p.D = a->D; p.N = a->N; p.G = a->G; p.softplus = a->softplus;
    p.skip_f32 = a->skip_dtype == VIG_DTYPE_F32; p.bias_f32 = a->bias_dtype == VIG_DTYPE_F32;
    p.tiles = (p.L + TILE - 1) / TILE;
    p.status = a->status;
    const int size = a->dtype == VIG_DTYPE_F32 ? 4 : 2;
    p.piece = p.piece_maps = 16;
    narrow(p.piece, p.u, p.s_u, 2, size); narrow(p.piece, p.dt, p.s_dt, 2, size); narrow(p.piece, p.z, p.s_z, 2, size);
    const int64_t rows[1] = {p.D}, group[1] = {p.D / p.G}, n[1] = {p.N};
    narrow(p.piece, p.u, group, 1, size);                        // a group begins where a piece may begin
    if (grads) {
        narrow(p.piece, p.dy, p.s_dy, 2, size);
        narrow(p.piece, p.d_u, rows, 1, size); narrow(p.piece, p.d_dt, rows, 1, size); narrow(p.piece, p.d_z, rows, 1, size);
    } else {
        narrow(p.piece, p.y, p.s_y, 2, size);
    }
    narrow(p.piece_maps, p.b, p.s_b, 3, size); narrow(p.piece_maps, p.c, p.s_c, 3, size); narrow(p.piece_maps, p.b, n, 1, size);
    return p;
}

}  // namespace vig

using namespace vig;

extern "C" size_t vig_selective_scan_states_bytes(int B, int L, int D, int N) {
    return B > 0 && L > 0 && D > 0 && N > 0 ? (size_t)B * ((L + TILE - 1) / TILE) * D * N * sizeof(float) : 0;
}

extern "C" int vig_selective_scan_fwd(const vig_selective_scan_args* a, void* stream) {
    if (const int e = check(a, false)) return e;
    if (!a->B || !a->D) return VIG_OK;
    Params p = params_of(a, false);
    switch (a->dtype) {
        case VIG_DTYPE_F32: return p.N <= 8 ? fwd_width<float, 2>(p, (cudaStream_t)stream) : fwd_width<float, 4>(p, (cudaStream_t)stream);
        case VIG_DTYPE_BF16: return p.N <= 8 ? fwd_width<__nv_bfloat16, 2>(p, (cudaStream_t)stream) : fwd_width<__nv_bfloat16, 4>(p, (cudaStream_t)stream);
        default: return p.N <= 8 ? fwd_width<__half, 2>(p, (cudaStream_t)stream) : fwd_width<__half, 4>(p, (cudaStream_t)stream);
    }
}

extern "C" size_t vig_selective_scan_bwd_workspace_bytes(int B, int L, int D, int N, int G) {
    if (B <= 0 || L < 0 || D <= 0 || N <= 0 || G <= 0) return 0;
    const size_t ctiles = (D / G + BCT - 1) / BCT;
    return sizeof(float) * (2 * ctiles * B * L * G * N + (size_t)B * D * (N + 2));
}

extern "C" int vig_selective_scan_bwd(const vig_selective_scan_args* a, void* stream) {
    if (const int e = check(a, true)) return e;
    if (!a->B || !a->D) return VIG_OK;
    if (!a->workspace || a->workspace_bytes < vig_selective_scan_bwd_workspace_bytes(a->B, a->L, a->D, a->N, a->G)) return VIG_ERR_WORKSPACE;
    const cudaStream_t s = (cudaStream_t)stream;
    Params p = params_of(a, true);
    p.ctiles = (p.D / p.G + BCT - 1) / BCT;
    const int64_t maps = (int64_t)p.B * p.L * p.G * p.N, rows = (int64_t)p.B * p.D;
    p.part_b = (float*)a->workspace;
    p.part_c = p.part_b + p.ctiles * maps;
    p.part_A = p.part_c + p.ctiles * maps;
    p.part_skip = p.part_A + rows * p.N;
    p.part_bias = p.part_skip + rows;
    int e;
    switch (a->dtype) {
        case VIG_DTYPE_F32: e = bwd_launch<float>(p, s); break;
        case VIG_DTYPE_BF16: e = bwd_launch<__nv_bfloat16>(p, s); break;
        default: e = bwd_launch<__half>(p, s); break;
    }
    if (e) return e;
    SumJobs jobs{};
    int64_t grid = 0;
    const auto add = [&](int k, const float* src, void* dst, int64_t n, int count, int type) {
        const int64_t blocks = dst ? (n + 255) / 256 : 0;
        jobs.job[k] = SumJob{src, dst, n, count, type, (int)blocks};
        grid += blocks;
    };
    add(0, p.part_b, a->d_b, maps, p.ctiles, a->dtype);
    add(1, p.part_c, a->d_c, maps, p.ctiles, a->dtype);
    add(2, p.part_A, a->d_A, (int64_t)p.D * p.N, p.B, VIG_DTYPE_F32);
    add(3, p.part_skip, a->d_skip, p.D, p.B, a->skip_dtype);
    add(4, p.part_bias, a->d_bias, p.D, p.B, a->bias_dtype);
    if (grid >= (1ll << 31)) return VIG_ERR_SHAPE;
    return (int)launch_next(sum_kernel, dim3((unsigned)grid), dim3(256), 0, s, jobs);
}

extern "C" int vig_selective_scan_step(const vig_selective_scan_args* a, void* stream) {
    if (!a) return VIG_ERR_NULL;
    if (a->L != 1) return VIG_ERR_SHAPE;
    if (const int e = check(a, false)) return e;
    if (!a->B || !a->D) return VIG_OK;
    if (!a->h_final) return VIG_ERR_NULL;
    StepParams p{a->u, a->dt, a->z, a->b, a->c, a->skip, a->dt_bias, a->A, a->h_final, a->y, a->s_u[0], a->s_dt[0], a->s_z[0], a->s_y[0], {a->s_b[0], a->s_b[2]},
                 {a->s_c[0], a->s_c[2]}, a->ld_final, a->B, a->D, a->N, a->G, a->skip_dtype == VIG_DTYPE_F32, a->bias_dtype == VIG_DTYPE_F32, a->softplus};
    p.whole = p.N % 4 == 0 && ((uintptr_t)p.state | (uintptr_t)p.A) % 16 == 0 && p.ld_state % 4 == 0;
    const int64_t grid = ((int64_t)p.B * p.D + 31) / 32;
    const cudaStream_t s = (cudaStream_t)stream;
    switch (a->dtype) {
        case VIG_DTYPE_F32: scan_step_kernel<float><<<(unsigned)grid, 128, 0, s>>>(p); break;
        case VIG_DTYPE_BF16: scan_step_kernel<__nv_bfloat16><<<(unsigned)grid, 128, 0, s>>>(p); break;
        default: scan_step_kernel<__half><<<(unsigned)grid, 128, 0, s>>>(p); break;
    }
    return (int)cudaGetLastError();
}
