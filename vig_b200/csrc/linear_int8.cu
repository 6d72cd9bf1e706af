// Product of 8-bit integers: y[m, n] = x_scales[m] w_scales[n] sum_k x[m, k] w[n, k] + bias[n].  Sums are 32-bit integers and exact; scales and bias are
// applied in fp32 and y is rounded once.  Three forms:
//   pairs   (rows on 16 bytes): tcgen05.mma kind::i8 on CTA pairs, tiles of 256 x 256, k boxes of 128 bytes through TMA, as gemm_pair.cu does for 16 bits: the
//           integer product is twice as fast and brings in half the bytes.  65536 x 768 x 2304 takes 97 us; 77 without the epilogue's work, 89 without its
//           stores; 70 would be the products by themselves, 54 the bytes (302 of 354 MB are the output).
//   skinny  (rows on 16 bytes, up to 64 of them): W is read once, by all SMs, straight into fragments of mma.sync; a warp takes 16 columns and a share of k.
//           768 x 2304 with W in L2, this form and pairs: 8 rows 2.4 and 6.6 us, 32 rows 5.1 and 6.7, 64 rows 6.8 and 6.9.  With W out of memory: 8 rows 4.2 and
//           7.3, 24 rows 7.7 and 7.4, 64 rows 11.9 and 7.5, so that there a border at 16 would be the better one.
//   any     everything else: mma.sync on 64 x 64 tiles through shared memory.
#include "tc_common.cuh"

namespace vig {
namespace {

using namespace tc;

struct Int8Params {
    const int8_t *x, *w;
    const float *xs, *ws;
    const void* bias;
    void* y;
    int64_t ldx, ldw, ldy, M;
    int N, K;
};

__device__ __forceinline__ void mma_s8(int* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ float bias_at(const void* bias, int n) { return bias ? DType<T>::to_f(((const T*)bias)[n]) : 0.f; }

// ---------------------------------------------------------------------------------------------------
// Pairs.  Roles, rings and the two forms (streaming; W's columns stationary) as in gemm_pair.cu.
constexpr int I8_BK = 128, I8_A = 128 * I8_BK, I8_B = 128 * I8_BK;       // one CTA's k box of x: its 128 rows; of W: its half of 256
constexpr int I8_EPI = 8, I8_THREADS = 64 + 32 * I8_EPI, I8_MAX_ST = 8, I8_BARS = 8 * (2 * I8_MAX_ST + 5);
constexpr int I8_BOX = 32 * 128;                                         // an epilogue warp's way out: 32 rows of 128 bytes, whole lines (of 64 bytes: 106 us for 65536 x 768 x 2304)
constexpr int I8_COLS = I8_EPI * 2 * 128 * 4;                            // every epilogue warp's scales of W and biases, of its 128 columns
constexpr int I8_RING = 227 * 1024 - 1024 - I8_EPI * I8_BOX - I8_COLS - I8_BARS - 16;
// D of 32-bit integers, A and B of signed bytes, both along k
constexpr uint32_t I8_IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((256u >> 3) << 17) | ((256u >> 4) << 24);

__device__ __forceinline__ void mma_pair_i8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], da, db, %3, p;\n\t}"
                 ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(I8_IDESC), "r"(accumulate), "r"(DESC_HI) : "memory");
}

__device__ __forceinline__ void prefetch_2d(const CUtensorMap* map, int c0, int c1) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(c0), "r"(c1) : "memory");
}

struct I8Maps { CUtensorMap x, w, o; };

// byte of (row, 16-byte piece) in a box, swizzled as the tensor map of the output says
__device__ __forceinline__ int box_at(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }

template <typename T, bool STAT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8_THREADS, 1)
int8_pair_kernel(const __grid_constant__ I8Maps maps, const Int8Params p, int KB, int ntn, int ntm, int nst, int boxed, int32_t* status) {
    constexpr int BN = 256, COLS = 128, PIECE = 128 / (int)sizeof(T), STAGE = I8_A + (STAT ? 0 : I8_B), V = 16 / (int)sizeof(T);
    extern __shared__ uint8_t i8_smem_raw[];
    uint8_t* smem = i8_smem_raw + ((1024u - (smem_u32(i8_smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_rank();
    const int pair = (int)blockIdx.x >> 1, step = (int)gridDim.x >> 1, ntiles = ntm * ntn;
    const uint32_t off_ring = STAT ? (uint32_t)KB * I8_B : 0u, off_out = off_ring + (uint32_t)nst * STAGE, off_cols = off_out + I8_EPI * I8_BOX, off_bar = off_cols + I8_COLS;
    const uint32_t bar_full = sbase + off_bar, bar_empty = bar_full + 8 * I8_MAX_ST, bar_acc_full = bar_empty + 8 * I8_MAX_ST, bar_acc_empty = bar_acc_full + 16,
                   bar_w = bar_acc_empty + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + off_bar + I8_BARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const Waiter waiter{abort_flag, status};

    if (tid == 0) {
        mbar_init(bar_w, 1);
        for (int s = 0; s < nst; ++s) { mbar_init(bar_full + 8 * s, 1); mbar_init(bar_empty + 8 * s, 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(bar_acc_full + 8 * b, 1); mbar_init(bar_acc_empty + 8 * b, 2 * I8_EPI); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid == 32) {
        tma_prefetch_map(&maps.x); tma_prefetch_map(&maps.w);
        if (boxed) tma_prefetch_map(&maps.o);
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                      // the barriers of both CTAs exist
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {                                     // ---- TMA producer: my rows of x, my half of the rows of W; their bytes are counted by the even CTA
        uint32_t st = 0, phase = 0;
        if (STAT && lane == 0) {
            const int wrow = pair % ntn * BN + (rank ? BN / 2 : 0);
            if (rank == 0) mbar_expect_tx(bar_w, 2u * KB * I8_B);
            for (int kb = 0; kb < KB; ++kb) tma_load_2d_pair(sbase + kb * I8_B, &maps.w, kb * I8_BK, wrow, map_rank(bar_w, 0));
        }
        __syncwarp();
        for (int tile = pair; tile < ntiles; tile += step) {
            const int row = (tile / ntn) * 256 + 128 * (int)rank, wrow = tile % ntn * BN + (rank ? BN / 2 : 0);
            for (int kb = 0; kb < KB; ++kb) {
                // the MMAs of a ring ago have read the stage, in both CTAs; asked first, since a wait costs hundreds of cycles even when its phase is over
                if (!mbar_test_wait(bar_empty + 8 * st, phase ^ 1u)) waiter.wait_lite(bar_empty + 8 * st, phase ^ 1u);
                if (*abort_flag) break;
                if (lane == 0) {
                    if (rank == 0) mbar_expect_tx(bar_full + 8 * st, 2 * STAGE);
                    const uint32_t bar = map_rank(bar_full + 8 * st, 0), dst = sbase + off_ring + st * STAGE;
                    tma_load_2d_pair(dst, &maps.x, kb * I8_BK, row, bar);
                    // the pairs of a row tile want the same box at the same time: it is on its way to L2 a tile ahead
                    if (STAT && tile % ntn == kb % ntn && tile + step < ntiles) prefetch_2d(&maps.x, kb * I8_BK, row + step / ntn * 256);
                    if (!STAT) tma_load_2d_pair(dst + I8_A, &maps.w, kb * I8_BK, wrow, bar);
                }
                __syncwarp();
                if (++st == (uint32_t)nst) { st = 0; phase ^= 1u; }
            }
            if (*abort_flag) break;
        }
        for (int s = 0; s < nst; ++s) {                  // no arrival is on its way to this CTA when it ends
            waiter.wait_lite(bar_empty + 8 * st, phase ^ 1u);
            if (++st == (uint32_t)nst) { st = 0; phase ^= 1u; }
        }
    } else if (warp == 1) {
        if (rank == 0) {                                 // ---- MMA issuer of the pair; the next stage and buffer are asked about ahead
            const bool issuer = lane == 0;
            uint32_t st = 0, phase = 0, it = 0, pre = 0, pre_acc = 0;
            const uint32_t lo0 = make_desc(sbase + off_ring), w_lo = make_desc(sbase);
            if (STAT) waiter.wait_lite(bar_w, 0);
            for (int tile = pair; tile < ntiles; tile += step, ++it) {
                const uint32_t buf = it & 1u;
                if (!pre_acc) waiter.wait_lite(bar_acc_empty + 8 * buf, ((it >> 1) & 1u) ^ 1u);
                if (*abort_flag) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * 256u;
                for (int kb = 0; kb < KB; ++kb) {
                    if (!pre) waiter.wait_lite(bar_full + 8 * st, phase);
                    tc_fence_after();
                    const uint32_t st_next = st + 1 == (uint32_t)nst ? 0u : st + 1, ph_next = st + 1 == (uint32_t)nst ? phase ^ 1u : phase;
                    const uint32_t a_lo = lo0 + st * (STAGE >> 4), b_lo = STAT ? w_lo + (uint32_t)kb * (I8_B >> 4) : a_lo + (I8_A >> 4);
#pragma unroll
                    for (uint32_t k4 = 0; k4 < 4; ++k4) { if (issuer) mma_pair_i8(d, a_lo + 2 * k4, b_lo + 2 * k4, (kb | k4) > 0 ? 1u : 0u); }
                    pre = mbar_test_wait(bar_full + 8 * st_next, ph_next);
                    if (kb + 1 == KB) pre_acc = mbar_test_wait(bar_acc_empty + 8 * (buf ^ 1u), (((it + 1) >> 1) & 1u) ^ 1u);
                    if (issuer) tc_commit_pair(bar_empty + 8 * st);
                    st = st_next; phase = ph_next;
                }
                if (issuer) tc_commit_pair(bar_acc_full + 8 * buf);
            }
        }
    } else {                                             // ---- epilogue: a warp has a quarter of the rows and half of the columns, a box of them at a time
        const int ew = warp - 2, part = ew >> 2;
        const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
        uint8_t* box = smem + off_out + ew * I8_BOX;
        const uint32_t drained = map_rank(bar_acc_empty, 0);
        float* const cols = reinterpret_cast<float*>(smem + off_cols) + ew * 2 * COLS;    // scales, and behind them biases
        int at_cols = -1;
        uint32_t it = 0;
        for (int tile = pair; tile < ntiles; tile += step, ++it) {
            const uint32_t buf = it & 1u, acc = tmem + lane_base + buf * 256u + COLS * part;
            const int row = (tile / ntn) * 256 + 128 * (int)rank + 32 * (warp & 3), col = (tile % ntn) * BN + COLS * part;
            const float xs = row + lane < p.M ? __ldg(p.xs + row + lane) : 0.f;
            if (col != at_cols) {                        // in the stationary form once
                at_cols = col;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < COLS; i += 32) {
                    const int n = col + i + lane;
                    cols[i + lane] = n < p.N ? __ldg(p.ws + n) : 0.f;
                    cols[COLS + i + lane] = n < p.N ? bias_at<T>(p.bias, n) : 0.f;
                }
            }
            waiter.wait_lite(bar_acc_full + 8 * buf, (it >> 1) & 1u);    // by the whole warp
            if (*abort_flag) break;
            tc_fence_after();
            __syncwarp();
#pragma unroll
            for (int k = 0; k < COLS; k += PIECE) {
                const int c = col + k;
                float g[PIECE];
#pragma unroll
                for (int i = 0; i < PIECE; i += 32) tc_ld32(acc + k + i, g + i);
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // the warp's earlier store has read the box
                __syncwarp();
                tc_wait_ld();
                if (k + PIECE == COLS) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(drained + 8 * buf);
                }
                // the same addresses for all lanes
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    T e[V];
                    float ws[V], b[V];
#pragma unroll
                    for (int i = 0; i < V; i += 4) {
                        *(float4*)(ws + i) = *(const float4*)(cols + k + j * V + i);
                        *(float4*)(b + i) = *(const float4*)(cols + COLS + k + j * V + i);
                    }
#pragma unroll
                    for (int i = 0; i < V; ++i) e[i] = DType<T>::from_f(fmaf((float)__float_as_int(g[j * V + i]), xs * ws[i], b[i]));
                    uint4 w;
                    memcpy(&w, e, 16);
                    *reinterpret_cast<uint4*>(box + box_at(lane, j)) = w;
                }
                if (boxed) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        if (row < p.M && c < p.N) tma_store_2d(&maps.o, c, row, smem_u32(box));      // rows past M are clipped by the tensor map
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                } else {                                 // rows off 16 bytes: a lane has a column
                    __syncwarp();
#pragma unroll
                    for (int i = lane; i < PIECE; i += 32) {
                        if (c + i >= p.N) break;
                        T* to = (T*)p.y + (int64_t)row * p.ldy + c + i;
                        for (int r = 0; r < 32 && row + r < p.M; ++r) to[r * p.ldy] = *reinterpret_cast<const T*>(box + box_at(r, i / V) + i % V * sizeof(T));
                    }
                    __syncwarp();
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // the stores have read their boxes
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                      // neither CTA ends while the other may still signal it
    if (tid == 0 && *abort_flag && status) atomicOr(status, 1);
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

bool map_of_bytes(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld) {
    MapKey key{};
    key.base = base; key.rank = 2; key.dtype = MAP_BYTES; key.swizzle = 1;
    key.dims[0] = (uint64_t)cols; key.dims[1] = (uint64_t)rows;
    key.strides[0] = (uint64_t)ld;
    key.box[0] = I8_BK; key.box[1] = 128;
    return encode_cached(m, key);
}
bool map_of_output(CUtensorMap* m, const Int8Params& p, int dtype) {
    const int size = dtype == VIG_DTYPE_F32 ? 4 : 2;
    MapKey key{};
    key.base = p.y; key.rank = 2; key.dtype = dtype; key.swizzle = 1;
    key.dims[0] = (uint64_t)p.N; key.dims[1] = (uint64_t)p.M;
    key.strides[0] = (uint64_t)p.ldy * size;
    key.box[0] = 128 / size; key.box[1] = 32;
    return encode_cached(m, key);
}

template <typename T> int pair_launch(const Int8Params& p, int dtype, int32_t* status, cudaStream_t s) {
    I8Maps maps{};
    const int boxed = (uintptr_t)p.y % 16 == 0 && p.ldy * (int)sizeof(T) % 16 == 0;
    if (!map_of_bytes(&maps.x, p.x, p.M, p.K, p.ldx) || !map_of_bytes(&maps.w, p.w, p.N, p.K, p.ldw) || (boxed && !map_of_output(&maps.o, p, dtype))) return VIG_ERR_DEVICE;
    const int ntn = (p.N + 255) / 256, KB = (p.K + I8_BK - 1) / I8_BK, all = device_sms() / 2;
    const int64_t ntm = (p.M + 255) / 256;
    if (ntm * ntn > INT32_MAX) return VIG_ERR_SHAPE;
    // stationary by the rule of the 16-bit form: where W's columns leave a ring of four boxes of x, nearly all pairs have a column and each has a tile
    const int xst = (I8_RING - KB * I8_B) / I8_A;
    const bool stat = xst >= 4 && all / ntn * ntn * 16 >= all * 15 && ntm * ntn >= all;
    const int nst = stat ? (xst < I8_MAX_ST ? xst : I8_MAX_ST) : I8_RING / (I8_A + I8_B);
    const int smem = (stat ? KB * I8_B + nst * I8_A : nst * (I8_A + I8_B)) + I8_EPI * I8_BOX + I8_COLS + I8_BARS + 16 + 1024;
    const int64_t pairs = stat ? all / ntn * ntn : ntm * ntn < all ? ntm * ntn : all;
    const auto kfn = stat ? int8_pair_kernel<T, true> : int8_pair_kernel<T, false>;
    if (const cudaError_t e = ensure_smem_attr((const void*)kfn, 227 * 1024)) return (int)e;
    kfn<<<2 * (unsigned)pairs, I8_THREADS, smem, s>>>(maps, p, KB, ntn, (int)ntm, nst, boxed, status);
    return (int)cudaGetLastError();
}

// ---------------------------------------------------------------------------------------------------
// Skinny.  W is the A operand (16 of its rows a CTA), tokens are the columns, MT tiles of 8.  The order of k within a sum is free: a lane takes 16 neighbouring bytes of
// a row, a word of them to each of four steps' fragments, so that a warp reads whole rows of 64 bytes and needs no shared memory.  Four warps share k.
template <typename T, int MT> __global__ void __launch_bounds__(128) int8_skinny_kernel(const Int8Params p) {
    __shared__ int sums[4][16 * 8 * MT];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3, n0 = blockIdx.x * 16;
    const int8_t *w0 = p.w + (int64_t)min(n0 + g, p.N - 1) * p.ldw, *w1 = p.w + (int64_t)min(n0 + g + 8, p.N - 1) * p.ldw;
    int acc[MT][4] = {};
    const int blocks = (p.K + 63) / 64;
#pragma unroll 4
    for (int kb = warp; kb < blocks; kb += 4) {
        const int k = kb * 64 + q * 16;
        const bool in = k < p.K;                         // rows are whole pieces of 16 bytes
        uint4 a0 = make_uint4(0u, 0u, 0u, 0u), a1 = a0;
        if (in) { a0 = __ldg((const uint4*)(w0 + k)); a1 = __ldg((const uint4*)(w1 + k)); }
        const uint32_t s0[4] = {a0.x, a1.x, a0.y, a1.y}, s1[4] = {a0.z, a1.z, a0.w, a1.w};
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int64_t m = i * 8 + g;
            uint4 b = make_uint4(0u, 0u, 0u, 0u);
            if (in && m < p.M) b = __ldg((const uint4*)(p.x + m * p.ldx + k));
            mma_s8(acc[i], s0, b.x, b.y);
            mma_s8(acc[i], s1, b.z, b.w);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[warp][(i * 8 + q * 2 + (e & 1)) * 16 + g + (e >> 1) * 8] = acc[i][e];   // [token][column of y]
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * 8 * MT; i += 128) {
        const int m = i / 16, n = n0 + i % 16;
        if (m < p.M && n < p.N) {
            const int v = sums[0][i] + sums[1][i] + sums[2][i] + sums[3][i];
            ((T*)p.y)[m * p.ldy + n] = DType<T>::from_f(fmaf((float)v, p.xs[m] * p.ws[n], bias_at<T>(p.bias, n)));
        }
    }
}

template <typename T> int skinny_launch(const Int8Params& p, cudaStream_t s) {
    const unsigned grid = (unsigned)((p.N + 15) / 16);
    if (p.M <= 8) int8_skinny_kernel<T, 1><<<grid, 128, 0, s>>>(p);
    else if (p.M <= 16) int8_skinny_kernel<T, 2><<<grid, 128, 0, s>>>(p);
    else if (p.M <= 32) int8_skinny_kernel<T, 4><<<grid, 128, 0, s>>>(p);
    else int8_skinny_kernel<T, 8><<<grid, 128, 0, s>>>(p);
    return (int)cudaGetLastError();
}

// ---------------------------------------------------------------------------------------------------
// Any sizes and alignment: 64 x 64 tiles, four warps of 32 x 32, k in steps of 64 through shared memory with rows of 80 bytes.  The next step's words are on their
// way while one is worked on.  A word of a row that does not begin on 4 bytes is put together from the two that hold it, as far as both are the
// tensor's; at its ends from bytes.
constexpr int BM = 64, BN = 64, BK = 64, PITCH = 80;

__device__ __forceinline__ uint32_t word_at(const int8_t* row, int k, int K, uintptr_t begin, uintptr_t end) {
    if (k >= K) return 0;
    const uintptr_t a = (uintptr_t)row + k, low = a & ~(uintptr_t)3;
    const uint32_t shift = (uint32_t)(a & 3) * 8;
    uint32_t v;
    if (low >= begin && low + (shift ? 8 : 4) <= end) {
        v = *(const uint32_t*)low;
        if (shift) v = __funnelshift_r(v, *(const uint32_t*)(low + 4), shift);
        const int left = K - k;
        return left >= 4 ? v : v & ((1u << (8 * left)) - 1u);
    }
    v = 0;
    for (int i = 0; i < 4; ++i) if (k + i < K) v |= (uint32_t)(uint8_t)row[k + i] << (8 * i);
    return v;
}

// Rows laid out on 16 bytes, zeros behind them: a thread puts 16 bytes together
__global__ void __launch_bounds__(256) int8_lay_out_kernel(const int8_t* src, int64_t ld, uint4* dst, int64_t rows, int K, int pieces) {
    const uintptr_t begin = (uintptr_t)src, end = begin + (uintptr_t)((rows - 1) * ld + K);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * pieces; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / pieces;
        const int k = (int)(i - row * pieces) * 16;
        const int8_t* from = src + row * ld;
        dst[i] = make_uint4(word_at(from, k, K, begin, end), word_at(from, k + 4, K, begin, end), word_at(from, k + 8, K, begin, end), word_at(from, k + 12, K, begin, end));
    }
}

template <typename T> __global__ void __launch_bounds__(128) int8_any_kernel(const Int8Params p) {
    __shared__ __align__(16) int8_t xs[BM * PITCH], ws[BN * PITCH];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    const int64_t m0 = (int64_t)blockIdx.x * BM;
    const int n0 = blockIdx.y * BN, wm = (warp & 1) * 32, wn = (warp >> 1) * 32;
    const uintptr_t x_begin = (uintptr_t)p.x, x_end = x_begin + (uintptr_t)((p.M - 1) * p.ldx + p.K), w_begin = (uintptr_t)p.w, w_end = w_begin + (uintptr_t)((int64_t)(p.N - 1) * p.ldw + p.K);
    int acc[2][4][4] = {};
    // a thread has word tid % 16 of rows tid / 16 + 8 i
    const int kw = tid % 16 * 4, r0 = tid / 16;
    uint32_t nx[8], nw[8];
    auto bring = [&](int k0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t m = m0 + r0 + 8 * i;
            const int n = n0 + r0 + 8 * i;
            nx[i] = m < p.M ? word_at(p.x + m * p.ldx, k0 + kw, p.K, x_begin, x_end) : 0u;
            nw[i] = n < p.N ? word_at(p.w + (int64_t)n * p.ldw, k0 + kw, p.K, w_begin, w_end) : 0u;
        }
    };
    bring(0);
    for (int k0 = 0; k0 < p.K; k0 += BK) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            *(uint32_t*)(xs + (r0 + 8 * i) * PITCH + kw) = nx[i];
            *(uint32_t*)(ws + (r0 + 8 * i) * PITCH + kw) = nw[i];
        }
        __syncthreads();
        bring(k0 + BK);
#pragma unroll
        for (int k = 0; k < BK; k += 32) {
            uint32_t a[2][4], b[4][2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int8_t* r = xs + (wm + i * 16 + g) * PITCH + k + q * 4;
                a[i][0] = *(const uint32_t*)r; a[i][1] = *(const uint32_t*)(r + 8 * PITCH); a[i][2] = *(const uint32_t*)(r + 16); a[i][3] = *(const uint32_t*)(r + 8 * PITCH + 16);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int8_t* r = ws + (wn + j * 8 + g) * PITCH + k + q * 4;
                b[j][0] = *(const uint32_t*)r; b[j][1] = *(const uint32_t*)(r + 16);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) mma_s8(acc[i][j], a[i], b[j][0], b[j][1]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t m = m0 + wm + i * 16 + h * 8 + g;
            if (m >= p.M) continue;
            const float s = p.xs[m];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int n = n0 + wn + j * 8 + q * 2 + e;
                    if (n < p.N) ((T*)p.y)[m * p.ldy + n] = DType<T>::from_f(fmaf((float)acc[i][j][2 * h + e], s * p.ws[n], bias_at<T>(p.bias, n)));
                }
        }
}

template <typename T> int any_launch(const Int8Params& p, cudaStream_t s) {
    const int64_t gm = (p.M + BM - 1) / BM, gn = (p.N + BN - 1) / BN;
    if (gm >= (1ll << 31) || gn > 65535) return VIG_ERR_SHAPE;
    int8_any_kernel<T><<<dim3((unsigned)gm, (unsigned)gn), 128, 0, s>>>(p);
    return (int)cudaGetLastError();
}

template <typename T> int int8_launch(const Int8Params& p, int dtype, int32_t* status, cudaStream_t s) {
    const bool on_16 = p.K % 16 == 0 && ((uintptr_t)p.x | (uintptr_t)p.w) % 16 == 0 && (p.ldx | p.ldw) % 16 == 0 && p.ldx >= p.K && p.ldw >= p.K;
    if (!on_16 || !p.K) return any_launch<T>(p, s);
    if (p.M <= 64) return skinny_launch<T>(p, s);
    return pair_launch<T>(p, dtype, status, s);
}

}  // namespace
}  // namespace vig

using namespace vig;

// Codes may be -128, whose product is 2^14: 2^17 of them are one more than a signed sum of 32 bits holds
constexpr int I8_MOST_K = 131071;

// Off 16 bytes the 64 x 64 form takes what is little, and what is more is laid out first: 65536 x 333 x 576 536 us as it lies.
extern "C" int vig_linear_int8_laid_out_first(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0 || K > I8_MOST_K / 16 * 16) return 0;
    const bool on_16 = K % 16 == 0 && ((uintptr_t)x | (uintptr_t)w) % 16 == 0 && (ldx | ldw) % 16 == 0 && ldx >= K && ldw >= K;
    return !on_16 && (double)M * N * K >= 1 << 24;
}

extern "C" int vig_int8_rows_lay_out(const void* src, int64_t ld, void* dst, int64_t rows, int K, void* stream) {
    if (rows < 0 || K < 0 || K > I8_MOST_K) return VIG_ERR_SHAPE;
    if (!rows || !K) return VIG_OK;
    if (!src || !dst) return VIG_ERR_NULL;
    if ((uintptr_t)dst % 16) return VIG_ERR_ALIGN;
    const int pieces = (K + 15) / 16;
    const int64_t blocks = (rows * pieces + 255) / 256, most = (int64_t)device_sms() * 16;
    int8_lay_out_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, (cudaStream_t)stream>>>((const int8_t*)src, ld, (uint4*)dst, rows, K, pieces);
    return (int)cudaGetLastError();
}

extern "C" int vig_linear_int8_fwd(const void* x, int64_t ldx, const float* x_scales, const void* w, int64_t ldw, const float* w_scales, const void* bias, void* y,
                                   int64_t ldy, int64_t M, int N, int K, int dtype, int32_t* status_dev, void* stream) {
    if (dtype < VIG_DTYPE_F32 || dtype > VIG_DTYPE_F16) return VIG_ERR_DTYPE;
    if (M < 0 || N < 0 || K < 0 || K > I8_MOST_K || M > INT32_MAX - 1024 || N > 4194240) return VIG_ERR_SHAPE;
    if (!M || !N) return VIG_OK;
    if (!x_scales || !w_scales || !y || (K && (!x || !w))) return VIG_ERR_NULL;
    const Int8Params p{(const int8_t*)x, (const int8_t*)w, x_scales, w_scales, bias, y, ldx, ldw, ldy, M, N, K};
    switch (dtype) {
        case VIG_DTYPE_F32: return int8_launch<float>(p, dtype, status_dev, (cudaStream_t)stream);
        case VIG_DTYPE_BF16: return int8_launch<__nv_bfloat16>(p, dtype, status_dev, (cudaStream_t)stream);
        default: return int8_launch<__half>(p, dtype, status_dev, (cudaStream_t)stream);
    }
}
