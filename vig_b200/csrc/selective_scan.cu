// Selective scan: states h[d, n] of D channels with N states each, driven by inputs u, steps delta and maps B, C that change from token to token.
//
//   delta_t = softplus(dt_t + bias)   (or dt_t + bias),   h_t[d, n] = exp(delta_t[d] A[d, n]) h_{t-1}[d, n] + delta_t[d] u_t[d] B_t[n],
//   y_t[d] = (sum_n C_t[n] h_t[d, n] + D[d] u_t[d]) silu(z_t[d]).
//
// Every (token, channel, state) costs an exponential and three multiply-adds, every (token, channel) three 16-bit values in and one out: with 16
// states the exponentials bound it (MUFU, 16 a cycle and SM), not memory.  So each is taken once: a CTA walks its channels' tokens in tiles, and
// within a tile a warp's lanes divide tokens and states (scan_common.cuh) and join their runs by a scan over the lanes, where two passes over
// independent chunks would take every exponential twice.
#include "scan_common.cuh"

namespace vig {
using namespace scan;

template <typename T, int S, int CPW> struct FwdSmem {
    static constexpr int NC = 2 * CPW, CT = WARPS * CPW;         // channels of a thread ahead of and behind the scan, of the CTA
    static constexpr int SLOT = NC * (int)sizeof(T), ROWS = 3 * THREADS * SLOT;
    static __host__ __device__ int padded(int N) { return (N + 4 * S - 1) / (4 * S) * (4 * S); }
    static int bytes(int N) { return 2 * ROWS + 4 * TILE * padded(N) * (int)sizeof(T) + 3 * CT * TILE * 4 + 2 * CT * padded(N) * 4; }
};

template <typename T, int S, int CPW>
__global__ void __launch_bounds__(THREADS, 3) scan_fwd_kernel(const Params p) {
    using M = FwdSmem<T, S, CPW>;
    constexpr int NC = M::NC, CT = M::CT, NB = 4 * S;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, run = lane / PARTS, part = lane % PARTS;
    const int Npad = M::padded(p.N), Dg = p.D / p.G;
    const int ct = blockIdx.x % p.ctiles, g = blockIdx.x / p.ctiles % p.G, b = blockIdx.x / p.ctiles / p.G;
    const int c0 = ct * CT, have = min(CT, Dg - c0), d0 = g * Dg + c0;            // channels of the CTA, the first one's index
    const int len = length_of(p, b), ntiles = (len + TILE - 1) / TILE;
    T* const slots = (T*)smem;
    T* const maps = (T*)(smem + 2 * M::ROWS);
    float* const delta = (float*)(maps + 4 * TILE * Npad);
    float* const x = delta + CT * TILE;
    float* const ys = x + CT * TILE;
    float* const sA = ys + CT * TILE;
    float* const sh = sA + CT * Npad;

    // ahead of and behind the scan a thread has one token and NC channels
    const int t = tid % TILE, cl = tid / TILE * NC, mine = min(max(have - cl, 0), NC), d = d0 + cl;
    float bias[NC], skip[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        bias[i] = p.bias && i < mine ? param_at<T>(p.bias, d + i, p.bias_f32) : 0.f;
        skip[i] = p.skip && i < mine ? param_at<T>(p.skip, d + i, p.skip_f32) : 0.f;
    }
    for (int i = tid; i < CT * Npad; i += THREADS) {
        const int c = i / Npad, n = i - c * Npad;
        const bool in = c < have && n < p.N;
        sA[i] = in ? p.A[(int64_t)(d0 + c) * p.N + n] * LOG2E : 0.f;
        sh[i] = in && p.h0 ? p.h0[b * p.ld_h0 + (int64_t)(d0 + c) * p.N + n] : 0.f;
    }
    const T *u = (const T*)p.u + b * p.s_u[0] + d, *dt = (const T*)p.dt + b * p.s_dt[0] + d, *z = p.z ? (const T*)p.z + b * p.s_z[0] + d : nullptr;
    const T *mb = (const T*)p.b + b * p.s_b[0] + g * p.s_b[2], *mc = (const T*)p.c + b * p.s_c[0] + g * p.s_c[2];
    T* const y = (T*)p.y + b * p.s_y[0] + d;
    auto slot = [&](int buf, int k) { return slots + ((buf * 3 + k) * THREADS + tid) * NC; };
    auto map = [&](int buf, int k) { return maps + (buf * 2 + k) * TILE * Npad; };
    auto bring = [&](int tile, int buf) {
        const int64_t at = (int64_t)tile * TILE + t;
        if (at < len) {
            fetch<T, NC>(slot(buf, 0), u + at * p.s_u[1], mine, p.piece);
            fetch<T, NC>(slot(buf, 1), dt + at * p.s_dt[1], mine, p.piece);
            if (z) fetch<T, NC>(slot(buf, 2), z + at * p.s_z[1], mine, p.piece);
        }
        fetch_map<T>(map(buf, 0), mb, p.s_b[1], tile * TILE, len, p.N, Npad, p.piece_maps);
        fetch_map<T>(map(buf, 1), mc, p.s_c[1], tile * TILE, len, p.N, Npad, p.piece_maps);
    };
    if (ntiles) bring(0, 0);

    for (int tile = 0; tile < ntiles; ++tile) {
        const int buf = tile & 1, at = tile * TILE + t;
        copies_done();
        __syncthreads();                                         // the tile's maps are there; nobody is left in the tile before
        if (tile + 1 < ntiles) bring(tile + 1, buf ^ 1);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float dl = 0.f, xi = 0.f;                            // behind the end a token changes nothing
            if (at < len && i < mine) {
                dl = DType<T>::to_f(slot(buf, 1)[i]) + bias[i];
                if (p.softplus) dl = softplus<T>(dl);
                xi = dl * DType<T>::to_f(slot(buf, 0)[i]);
            }
            delta[(cl + i) * TILE + t] = dl;
            x[(cl + i) * TILE + t] = xi;
        }
        __syncthreads();

        for (int n0 = 0; n0 < Npad; n0 += NB) {
            F2 B[RUN][S / 2], C[RUN][S / 2];
#pragma unroll
            for (int j = 0; j < RUN; ++j) {
                const int at = (j * RUN + run) * Npad + n0 + part * S;
                pairs<T, S>(B[j], map(buf, 0) + at);
                pairs<T, S>(C[j], map(buf, 1) + at);
            }
#pragma unroll 1
            for (int ci = 0; ci < CPW; ++ci) {
                const int c = warp * CPW + ci;
                if (c >= have) break;
                float* const h_at = sh + c * Npad + n0 + part * S;
                F2 A2[S / 2], h0[S / 2], h[S / 2];
                pairs<float, S>(A2, sA + c * Npad + n0 + part * S);
                pairs<float, S>(h0, h_at);
                if (p.states && run == 0) {
                    float* to = p.states + (((int64_t)b * p.tiles + tile) * p.D + d0 + c) * p.N + n0 + part * S;
#pragma unroll
                    for (int s = 0; s < S; ++s) if (n0 + part * S + s < p.N) to[s] = s & 1 ? f2_hi(h0[s / 2]) : f2_lo(h0[s / 2]);
                }
                float dl[RUN], xr[RUN], yv[RUN];
                *(float4*)dl = *(const float4*)(delta + c * TILE + run * RUN);
                *(float4*)(dl + 4) = *(const float4*)(delta + c * TILE + run * RUN + 4);
                *(float4*)xr = *(const float4*)(x + c * TILE + run * RUN);
                *(float4*)(xr + 4) = *(const float4*)(x + c * TILE + run * RUN + 4);
                F2 a[RUN][S / 2];
                decays<S>(a, dl, A2);
                entering<S>(h, h0, a, B, xr, run, lane);
#pragma unroll
                for (int j = 0; j < RUN; ++j) {
                    const F2 xj = f2_make(xr[j], xr[j]);
                    F2 sum = 0ull;
#pragma unroll
                    for (int s = 0; s < S / 2; ++s) {
                        h[s] = f2_fma(a[j][s], h[s], f2_mul(xj, B[j][s]));
                        sum = s ? f2_fma(C[j][s], h[s], sum) : f2_mul(C[j][s], h[s]);
                    }
                    yv[j] = f2_lo(sum) + f2_hi(sum);
                }
                float2 got = over_parts(yv, part);
                float2* const ya = (float2*)(ys + c * TILE + run * RUN + part * 2);
                if (n0) { const float2 was = *ya; got.x += was.x; got.y += was.y; }
                *ya = got;
                __syncwarp();
                if (run == RUN - 1) {
#pragma unroll
                    for (int s = 0; s < S / 2; ++s) *(F2*)(h_at + 2 * s) = h[s];
                }
                __syncwarp();
            }
        }
        __syncthreads();
        if (at < len && mine) {
            float out[NC];
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                if (i < mine) {
                    out[i] = fmaf(skip[i], DType<T>::to_f(slot(buf, 0)[i]), ys[(cl + i) * TILE + t]);
                    if (z) { const float v = DType<T>::to_f(slot(buf, 2)[i]); out[i] *= v * sigmoidf_(v); }
                } else {
                    out[i] = 0.f;
                }
            }
            put<T, NC>(y + at * p.s_y[1], out, mine, p.piece);
        }
    }
    // behind the end the outputs are zeros
    for (int64_t at = (int64_t)len + t; at < p.L; at += TILE) {
        const float out[NC] = {};
        if (mine) put<T, NC>(y + at * p.s_y[1], out, mine, p.piece);
    }
    if (p.h_final) {
        __syncthreads();
        for (int i = tid; i < CT * Npad; i += THREADS) {
            const int c = i / Npad, n = i - c * Npad;
            if (c < have && n < p.N) p.h_final[b * p.ld_final + (int64_t)(d0 + c) * p.N + n] = sh[i];
        }
    }
}

// Backward, from the states that enter each tile (the forward wrote them) and the tiles from the last to the first.  With g_t = dL/dh_t,
//   g_t = C_t dy_t + a_{t+1} g_{t+1},  dC_t = sum_d h_t dy_t,  dB_t = sum_d g_t delta_t u_t,  du_t = delta_t sum_n g_t B_t + D dy_t,
//   ddelta_t = sum_n g_t (a_t h_{t-1} A + u_t B_t),  dA = sum g_t a_t h_{t-1} delta_t,
// dy being d_out silu(z).  A lane keeps the decays and states of its run; the maps' gradients add up in registers over the warp's channels, then
// over the CTA's warps, and the shares of CTAs, of sequences and of tokens are added in a fixed order by sum_kernel.
template <typename T, int S, int CPW> struct BwdSmem {
    static constexpr int NC = 2 * CPW, CT = WARPS * CPW, NB = 4 * S;
    static constexpr int SLOT = NC * (int)sizeof(T), ROWS = 4 * THREADS * SLOT;
    static __host__ __device__ int padded(int N) { return (N + NB - 1) / NB * NB; }
    static int bytes(int N) {
        const int Np = padded(N);
        return 2 * ROWS + 4 * TILE * Np * (int)sizeof(T) + 6 * CT * TILE * 4 + 4 * CT * Np * 4 + 8 * CT * Np * 4 + WARPS * TILE * NB * 2 * 4 + 2 * NC * THREADS * 4;
    }
};

template <typename T, int S, int CPW>
__global__ void __launch_bounds__(THREADS, 2) scan_bwd_kernel(const Params p) {
    using M = BwdSmem<T, S, CPW>;
    constexpr int NC = M::NC, CT = M::CT, NB = M::NB;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, run = lane / PARTS, part = lane % PARTS;
    const int Npad = M::padded(p.N), Dg = p.D / p.G;
    const int ct = blockIdx.x % p.ctiles, g = blockIdx.x / p.ctiles % p.G, b = blockIdx.x / p.ctiles / p.G;
    const int c0 = ct * CT, have = min(CT, Dg - c0), d0 = g * Dg + c0;
    const int len = length_of(p, b), ntiles = (len + TILE - 1) / TILE;
    T* const slots = (T*)smem;
    T* const maps = (T*)(smem + 2 * M::ROWS);
    float* const delta = (float*)(maps + 4 * TILE * Npad);
    float* const x = delta + CT * TILE;
    float* const dys = x + CT * TILE;
    float* const ys = dys + CT * TILE;                           // sum C h,
    float* const gb = ys + CT * TILE;                            // sum g B,
    float* const ga = gb + CT * TILE;                            // sum g a h A
    float* const sA = ga + CT * TILE;
    float* const sq = sA + CT * Npad;                            // a g of the token behind the tile
    float* const sh = sq + CT * Npad;                            // states that enter the tile, two buffers
    float* const dA = sh + 2 * CT * Npad;                        // a lane's share of dA: [channel][state block][lane][S]
    float* const shares = dA + 8 * CT * Npad;            // a warp's dB and dC: [dB, dC][warp][token][NB]
    float* const tok = shares + WARPS * TILE * NB * 2;           // a thread's shares of dD and dbias: [2 NC][thread]

    const int t = tid % TILE, cl = tid / TILE * NC, mine = min(max(have - cl, 0), NC), d = d0 + cl;
    float bias[NC], skip[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        bias[i] = p.bias && i < mine ? param_at<T>(p.bias, d + i, p.bias_f32) : 0.f;
        skip[i] = p.skip && i < mine ? param_at<T>(p.skip, d + i, p.skip_f32) : 0.f;
        tok[i * THREADS + tid] = 0.f;
        tok[(NC + i) * THREADS + tid] = 0.f;
    }
    for (int i = tid; i < CT * Npad; i += THREADS) {
        const int c = i / Npad, n = i - c * Npad;
        const bool in = c < have && n < p.N;
        sA[i] = in ? p.A[(int64_t)(d0 + c) * p.N + n] : 0.f;
        sq[i] = in && p.d_final ? p.d_final[((int64_t)b * p.D + d0 + c) * p.N + n] : 0.f;
    }
    for (int i = tid; i < CT * Npad * 8; i += THREADS) dA[i] = 0.f;
    const T *u = (const T*)p.u + b * p.s_u[0] + d, *dt = (const T*)p.dt + b * p.s_dt[0] + d, *z = p.z ? (const T*)p.z + b * p.s_z[0] + d : nullptr;
    const T* dy = (const T*)p.dy + b * p.s_dy[0] + d;
    const T *mb = (const T*)p.b + b * p.s_b[0] + g * p.s_b[2], *mc = (const T*)p.c + b * p.s_c[0] + g * p.s_c[2];
    auto slot = [&](int buf, int k) { return slots + ((buf * 4 + k) * THREADS + tid) * NC; };
    auto map = [&](int buf, int k) { return maps + (buf * 2 + k) * TILE * Npad; };
    auto bring = [&](int tile, int buf) {
        const int64_t at = (int64_t)tile * TILE + t;
        if (at < len) {
            fetch<T, NC>(slot(buf, 0), u + at * p.s_u[1], mine, p.piece);
            fetch<T, NC>(slot(buf, 1), dt + at * p.s_dt[1], mine, p.piece);
            if (z) fetch<T, NC>(slot(buf, 2), z + at * p.s_z[1], mine, p.piece);
            fetch<T, NC>(slot(buf, 3), dy + at * p.s_dy[1], mine, p.piece);
        }
        fetch_map<T>(map(buf, 0), mb, p.s_b[1], tile * TILE, len, p.N, Npad, p.piece_maps);
        fetch_map<T>(map(buf, 1), mc, p.s_c[1], tile * TILE, len, p.N, Npad, p.piece_maps);
        const float* st = p.states + (((int64_t)b * p.tiles + tile) * p.D + d0) * p.N;
        for (int i = tid; i < CT * Npad; i += THREADS) {
            const int c = i / Npad, n = i - c * Npad;
            float* to = sh + buf * CT * Npad + i;
            if (c < have && n < p.N) copy4(to, st + c * p.N + n);
            else *to = 0.f;
        }
    };
    if (ntiles) bring(ntiles - 1, (ntiles - 1) & 1);

    for (int tile = ntiles - 1; tile >= 0; --tile) {
        const int buf = tile & 1, at = tile * TILE + t;
        copies_done();
        __syncthreads();
        if (tile) bring(tile - 1, buf ^ 1);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float dl = 0.f, xi = 0.f, di = 0.f;
            if (at < len && i < mine) {
                dl = DType<T>::to_f(slot(buf, 1)[i]) + bias[i];
                if (p.softplus) dl = softplus<T>(dl);
                xi = dl * DType<T>::to_f(slot(buf, 0)[i]);
                di = DType<T>::to_f(slot(buf, 3)[i]);
                if (z) { const float v = DType<T>::to_f(slot(buf, 2)[i]); di *= v * sigmoidf_(v); }
            }
            delta[(cl + i) * TILE + t] = dl;
            x[(cl + i) * TILE + t] = xi;
            dys[(cl + i) * TILE + t] = di;
        }
        __syncthreads();

        for (int n0 = 0; n0 < Npad; n0 += NB) {
            F2 B[RUN][S / 2], C[RUN][S / 2], dB[RUN][S / 2], dC[RUN][S / 2];
#pragma unroll
            for (int j = 0; j < RUN; ++j) {
                const int at = (j * RUN + run) * Npad + n0 + part * S;
                pairs<T, S>(B[j], map(buf, 0) + at);
                pairs<T, S>(C[j], map(buf, 1) + at);
#pragma unroll
                for (int s = 0; s < S / 2; ++s) { dB[j][s] = 0ull; dC[j][s] = 0ull; }
            }
#pragma unroll 1
            for (int ci = 0; ci < CPW; ++ci) {
                const int c = warp * CPW + ci;
                if (c >= have) break;
                const int at = c * Npad + n0 + part * S;
                F2 A[S / 2], A2[S / 2], h0[S / 2], h[RUN + 1][S / 2], a[RUN][S / 2];
                pairs<float, S>(A, sA + at);
                pairs<float, S>(h0, sh + buf * CT * Npad + at);
#pragma unroll
                for (int s = 0; s < S / 2; ++s) A2[s] = f2_mul(A[s], f2_make(LOG2E, LOG2E));
                float dl[RUN], xr[RUN], dr[RUN], sums[RUN];
#pragma unroll
                for (int k = 0; k < RUN; k += 4) {
                    *(float4*)(dl + k) = *(const float4*)(delta + c * TILE + run * RUN + k);
                    *(float4*)(xr + k) = *(const float4*)(x + c * TILE + run * RUN + k);
                    *(float4*)(dr + k) = *(const float4*)(dys + c * TILE + run * RUN + k);
                }
                decays<S>(a, dl, A2);
                entering<S>(h[0], h0, a, B, xr, run, lane);
#pragma unroll
                for (int j = 0; j < RUN; ++j) {
                    const F2 xj = f2_make(xr[j], xr[j]), dj = f2_make(dr[j], dr[j]);
                    F2 sum = 0ull;
#pragma unroll
                    for (int s = 0; s < S / 2; ++s) {
                        h[j + 1][s] = f2_fma(a[j][s], h[j][s], f2_mul(xj, B[j][s]));
                        sum = s ? f2_fma(C[j][s], h[j + 1][s], sum) : f2_mul(C[j][s], h[j + 1][s]);
                        dC[j][s] = f2_fma(h[j + 1][s], dj, dC[j][s]);
                    }
                    sums[j] = f2_lo(sum) + f2_hi(sum);
                }
                const int to = c * TILE + run * RUN + part * 2;
                auto leave = [&](float* into) {
                    float2 got = over_parts(sums, part);
                    if (n0) { const float2 was = *(const float2*)(into + to); got.x += was.x; got.y += was.y; }
                    *(float2*)(into + to) = got;
                };
                if (z) leave(ys);
                // from the other end: q_t = a_t g_t is what token t - 1 gets
                F2 P[S / 2], Q[S / 2], q0[S / 2];
                pairs<float, S>(q0, sq + at);
#pragma unroll
                for (int s = 0; s < S / 2; ++s) { Q[s] = run == RUN - 1 ? q0[s] : 0ull; P[s] = a[0][s]; }
#pragma unroll
                for (int j = RUN - 1; j >= 0; --j)
#pragma unroll
                    for (int s = 0; s < S / 2; ++s) {
                        Q[s] = f2_mul(a[j][s], f2_fma(C[j][s], f2_make(dr[j], dr[j]), Q[s]));
                        if (j) P[s] = f2_mul(P[s], a[j][s]);
                    }
#pragma unroll
                for (int k = 1; k < RUN; k *= 2)
#pragma unroll
                    for (int s = 0; s < S / 2; ++s) {
                        const F2 e = f2_shfl_down(Q[s], k * PARTS);
                        Q[s] = f2_fma(P[s], run + k < RUN ? e : 0ull, Q[s]);
                        if (2 * k < RUN) P[s] = f2_mul(P[s], f2_shfl_down(P[s], k * PARTS));
                    }
#pragma unroll
                for (int s = 0; s < S / 2; ++s) {
                    const F2 e = f2_shfl_down(Q[s], PARTS);
                    Q[s] = run == RUN - 1 ? q0[s] : e;
                }
                float sums_a[RUN];
                F2 dAs[S / 2];
                float* const dA_at = dA + ((c * (Npad / NB) + n0 / NB) * 32 + lane) * S;
                pairs<float, S>(dAs, dA_at);
#pragma unroll
                for (int j = RUN - 1; j >= 0; --j) {
                    const F2 xj = f2_make(xr[j], xr[j]), dj = f2_make(dr[j], dr[j]), lj = f2_make(dl[j], dl[j]);
                    F2 sb = 0ull, sa = 0ull;
#pragma unroll
                    for (int s = 0; s < S / 2; ++s) {
                        const F2 gr = f2_fma(C[j][s], dj, Q[s]);
                        sb = s ? f2_fma(gr, B[j][s], sb) : f2_mul(gr, B[j][s]);
                        dB[j][s] = f2_fma(gr, xj, dB[j][s]);
                        Q[s] = f2_mul(a[j][s], gr);
                        const F2 f = f2_mul(Q[s], h[j][s]);
                        sa = s ? f2_fma(f, A[s], sa) : f2_mul(f, A[s]);
                        dAs[s] = f2_fma(f, lj, dAs[s]);
                    }
                    sums[j] = f2_lo(sb) + f2_hi(sb);
                    sums_a[j] = f2_lo(sa) + f2_hi(sa);
                }
                leave(gb);
#pragma unroll
                for (int j = 0; j < RUN; ++j) sums[j] = sums_a[j];
                leave(ga);
#pragma unroll
                for (int s = 0; s < S / 2; ++s) *(F2*)(dA_at + 2 * s) = dAs[s];
                __syncwarp();
                if (run == 0) {
#pragma unroll
                    for (int s = 0; s < S / 2; ++s) *(F2*)(sq + at + 2 * s) = Q[s];
                }
                __syncwarp();
            }
            // the warps' shares of the maps' gradients, added and left for sum_kernel
            if (n0) __syncthreads();
#pragma unroll
            for (int j = 0; j < RUN; ++j)
#pragma unroll
                for (int s = 0; s < S / 2; ++s) {
                    const int at = (run * RUN + j) * NB + part * S + 2 * s;
                    *(F2*)(shares + warp * TILE * NB + at) = dB[j][s];
                    *(F2*)(shares + (WARPS + warp) * TILE * NB + at) = dC[j][s];
                }
            __syncthreads();
            for (int i = tid; i < 2 * TILE * NB; i += THREADS) {
                const int which = i / (TILE * NB), k = i - which * TILE * NB, tt = k / NB, n = n0 + k % NB;
                if (tile * TILE + tt < len && n < p.N) {
                    float v = 0.f;
#pragma unroll
                    for (int w = 0; w < WARPS; ++w) v += shares[(which * WARPS + w) * TILE * NB + k];
                    float* out = which ? p.part_c : p.part_b;
                    out[((((int64_t)ct * p.B + b) * p.L + tile * TILE + tt) * p.G + g) * p.N + n] = v;
                }
            }
        }
        // (the barrier ahead of the sums stands between the warps' sums over states and this)
        if (at < len && mine) {
            float du[NC], dd[NC], dz[NC];
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                du[i] = dd[i] = dz[i] = 0.f;
                if (i < mine) {
                    const int k = (cl + i) * TILE + t;
                    const float ui = DType<T>::to_f(slot(buf, 0)[i]);
                    du[i] = fmaf(gb[k], delta[k], skip[i] * dys[k]);
                    dd[i] = fmaf(gb[k], ui, ga[k]);
                    if (p.softplus) dd[i] *= sigmoidf_(DType<T>::to_f(slot(buf, 1)[i]) + bias[i]);
                    if (z) {
                        const float v = DType<T>::to_f(slot(buf, 2)[i]), s = sigmoidf_(v);
                        dz[i] = DType<T>::to_f(slot(buf, 3)[i]) * fmaf(skip[i], ui, ys[k]) * s * fmaf(v, 1.f - s, 1.f);
                    }
                    tok[i * THREADS + tid] = fmaf(dys[k], ui, tok[i * THREADS + tid]);
                    tok[(NC + i) * THREADS + tid] += dd[i];
                }
            }
            const int64_t row = ((int64_t)b * p.L + at) * p.D + d;
            put<T, NC>((T*)p.d_u + row, du, mine, p.piece);
            put<T, NC>((T*)p.d_dt + row, dd, mine, p.piece);
            if (z) put<T, NC>((T*)p.d_z + row, dz, mine, p.piece);
        }
    }
    // behind the end all gradients are zeros
    for (int64_t at = (int64_t)len + t; at < p.L; at += TILE) {
        const float none[NC] = {};
        const int64_t row = ((int64_t)b * p.L + at) * p.D + d;
        if (mine) {
            put<T, NC>((T*)p.d_u + row, none, mine, p.piece);
            put<T, NC>((T*)p.d_dt + row, none, mine, p.piece);
            if (z) put<T, NC>((T*)p.d_z + row, none, mine, p.piece);
        }
    }
    for (int64_t i = (int64_t)len * p.N + tid; i < (int64_t)p.L * p.N; i += THREADS) {
        const int64_t at = ((((int64_t)ct * p.B + b) * p.L + i / p.N) * p.G + g) * p.N + i % p.N;
        p.part_b[at] = 0.f;
        p.part_c[at] = 0.f;
    }
    __syncthreads();
    for (int i = tid; i < CT * Npad; i += THREADS) {
        const int c = i / Npad, n = i - c * Npad;
        if (c < have && n < p.N) {
            float v = 0.f;
            const float* from = dA + ((c * (Npad / NB) + n / NB) * 32 + n % NB / S) * S + n % S;
            for (int r = 0; r < RUN; ++r) v += from[r * PARTS * S];
            const int64_t at = ((int64_t)b * p.D + d0 + c) * p.N + n;
            p.part_A[at] = v;
            if (p.d_h0) p.d_h0[at] = sq[i];
        }
    }
    if (tid < have) {
        const float *from = tok + tid % NC * THREADS + tid / NC * TILE, *from2 = from + NC * THREADS;
        float v = 0.f, v2 = 0.f;
        for (int k = 0; k < TILE; ++k) { v += from[k]; v2 += from2[k]; }
        if (p.part_skip) p.part_skip[(int64_t)b * p.D + d0 + tid] = v;
        if (p.part_bias) p.part_bias[(int64_t)b * p.D + d0 + tid] = v2;
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
    if (p.softplus) dl = softplus<T>(dl);
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
            hv[k] = fmaf(ex2(dl * (av[k] * LOG2E)), hv[k], x * bv[k]);
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
        y = fmaf(skip, u, y);
        if (p.z) y *= zv * sigmoidf_(zv);
        ((T*)p.y)[b * p.s_y + d] = DType<T>::from_f(y);
    }
}

static int piece_of(int64_t value) { return value % 16 == 0 ? 16 : value % 8 == 0 ? 8 : value % 4 == 0 ? 4 : 1; }
static void narrow(int& piece, const void* ptr, const int64_t* strides, int count, int size) {
    if (!ptr) return;
    piece = min(piece, piece_of((int64_t)(uintptr_t)ptr));
    for (int i = 0; i < count; ++i) piece = min(piece, piece_of(strides[i] * size));
}
template <int CT> void place(Params& p) { p.ctiles = (p.D / p.G + CT - 1) / CT; }

template <typename T, int S, int CPW> int fwd_launch(Params& p, cudaStream_t s) {
    place<WARPS * CPW>(p);
    const int64_t grid = (int64_t)p.B * p.G * p.ctiles;
    const int smem = FwdSmem<T, S, CPW>::bytes(p.N);
    if (grid >= (1ll << 31)) return VIG_ERR_SHAPE;
    if (const cudaError_t e = ensure_smem_attr((const void*)scan_fwd_kernel<T, S, CPW>, smem)) return (int)e;
    scan_fwd_kernel<T, S, CPW><<<(unsigned)grid, THREADS, smem, s>>>(p);
    return (int)cudaGetLastError();
}
template <typename T, int S, int CPW> int bwd_launch(Params& p, cudaStream_t s) {
    place<WARPS * CPW>(p);
    const int64_t grid = (int64_t)p.B * p.G * p.ctiles;
    const int smem = BwdSmem<T, S, CPW>::bytes(p.N);
    if (grid >= (1ll << 31)) return VIG_ERR_SHAPE;
    if (const cudaError_t e = ensure_smem_attr((const void*)scan_bwd_kernel<T, S, CPW>, smem)) return (int)e;
    scan_bwd_kernel<T, S, CPW><<<(unsigned)grid, THREADS, smem, s>>>(p);
    return (int)cudaGetLastError();
}

// channels of a CTA of the backward: fewer where the maps of many states need the room
constexpr int bwd_ct(int N) { return N <= 64 ? 4 * WARPS : WARPS; }

template <typename T> int fwd_pick(Params& p, cudaStream_t s) {
    return p.N <= 8 ? fwd_launch<T, 2, 4>(p, s) : fwd_launch<T, 4, 4>(p, s);
}
template <typename T> int bwd_pick(Params& p, cudaStream_t s) { return p.N <= 64 ? bwd_launch<T, 2, 4>(p, s) : bwd_launch<T, 2, 1>(p, s); }

static int check(const vig_selective_scan_args* a, bool grads) {
    if (!a) return VIG_ERR_NULL;
    const auto type_ok = [&](int t) { return t == a->dtype || t == VIG_DTYPE_F32; };
    if (a->dtype < VIG_DTYPE_F32 || a->dtype > VIG_DTYPE_F16 || (a->skip && !type_ok(a->skip_dtype)) || (a->dt_bias && !type_ok(a->bias_dtype))) return VIG_ERR_DTYPE;
    if (a->B < 0 || a->L < 0 || a->D < 0 || a->N < 1 || a->N > 128 || a->G < 1 || a->D % a->G) return VIG_ERR_SHAPE;
    if ((int64_t)a->B * a->D >= (1ll << 31) || a->D >= (1 << 28) || a->L >= (1 << 30)) return VIG_ERR_SHAPE;
    if (!a->B || !a->D) return VIG_OK;
    if (!a->A || (a->L && (!a->u || !a->dt || !a->b || !a->c || (!grads && !a->y)))) return VIG_ERR_NULL;
    if (grads && (!a->d_b || !a->d_c || !a->d_A || (a->L && (!a->states || !a->d_y || !a->d_u || !a->d_dt || (a->z && !a->d_z))))) return VIG_ERR_NULL;
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
        case VIG_DTYPE_F32: return fwd_pick<float>(p, (cudaStream_t)stream);
        case VIG_DTYPE_BF16: return fwd_pick<__nv_bfloat16>(p, (cudaStream_t)stream);
        default: return fwd_pick<__half>(p, (cudaStream_t)stream);
    }
}

extern "C" size_t vig_selective_scan_bwd_workspace_bytes(int B, int L, int D, int N, int G) {
    if (B <= 0 || L < 0 || D <= 0 || N <= 0 || G <= 0) return 0;
    const size_t ctiles = (D / G + bwd_ct(N) - 1) / bwd_ct(N);
    return sizeof(float) * (2 * ctiles * B * L * G * N + (size_t)B * D * (N + 2));
}

extern "C" int vig_selective_scan_bwd(const vig_selective_scan_args* a, void* stream) {
    if (const int e = check(a, true)) return e;
    if (!a->B || !a->D) return VIG_OK;
    if (!a->workspace || a->workspace_bytes < vig_selective_scan_bwd_workspace_bytes(a->B, a->L, a->D, a->N, a->G)) return VIG_ERR_WORKSPACE;
    const cudaStream_t s = (cudaStream_t)stream;
    Params p = params_of(a, true);
    p.ctiles = (p.D / p.G + bwd_ct(p.N) - 1) / bwd_ct(p.N);
    const int64_t maps = (int64_t)p.B * p.L * p.G * p.N, rows = (int64_t)p.B * p.D;
    p.part_b = (float*)a->workspace;
    p.part_c = p.part_b + p.ctiles * maps;
    p.part_A = p.part_c + p.ctiles * maps;
    p.part_skip = p.part_A + rows * p.N;
    p.part_bias = p.part_skip + rows;
    int e;
    switch (a->dtype) {
        case VIG_DTYPE_F32: e = bwd_pick<float>(p, s); break;
        case VIG_DTYPE_BF16: e = bwd_pick<__nv_bfloat16>(p, s); break;
        default: e = bwd_pick<__half>(p, s); break;
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
