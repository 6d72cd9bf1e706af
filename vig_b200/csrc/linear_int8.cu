// Product of 8-bit integers: y[m, n] = x_scales[m] w_scales[n] sum_k x[m, k] w[n, k] + bias[n].  Sums are 32-bit integers and exact; scales and bias are
// applied in fp32 and y is rounded once.
#include "tc_common.cuh"

namespace vig {
namespace {

struct Int8Params {
    const int8_t *x, *w;
    const float *xs, *ws;
    const void* bias;
    void* y;
    int64_t ldx, ldw, ldy, M;
    int N, K, whole;                                             // whole: rows of x and w are whole 16-byte pieces on 16 bytes
};

__device__ __forceinline__ void mma_s8(int* c, const uint32_t* a, const uint32_t* b) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// Any sizes and alignment: 64 x 64 tiles, four warps of 32 x 32, k in steps of 64 through shared memory with rows of 80 bytes.
constexpr int BM = 64, BN = 64, BK = 64, PITCH = 80;

template <typename T> __global__ void __launch_bounds__(128) int8_any_kernel(const Int8Params p) {
    __shared__ __align__(16) int8_t xs[BM * PITCH], ws[BN * PITCH];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    const int64_t m0 = (int64_t)blockIdx.x * BM;
    const int n0 = blockIdx.y * BN, wm = (warp & 1) * 32, wn = (warp >> 1) * 32;
    int acc[2][4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += BK) {
        __syncthreads();
        if (p.whole) {
            for (int i = tid; i < (BM + BN) * 4; i += 128) {
                const int row = i / 4, k = k0 + i % 4 * 16;
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (k < p.K) {
                    if (row < BM) { if (m0 + row < p.M) v = *(const uint4*)(p.x + (m0 + row) * p.ldx + k); }
                    else if (n0 + row - BM < p.N) v = *(const uint4*)(p.w + (int64_t)(n0 + row - BM) * p.ldw + k);
                }
                *(uint4*)((row < BM ? xs + row * PITCH : ws + (row - BM) * PITCH) + i % 4 * 16) = v;
            }
        } else {
            for (int i = tid; i < (BM + BN) * BK; i += 128) {
                const int row = i / BK, k = k0 + i % BK;
                int8_t v = 0;
                if (k < p.K) {
                    if (row < BM) { if (m0 + row < p.M) v = p.x[(m0 + row) * p.ldx + k]; }
                    else if (n0 + row - BM < p.N) v = p.w[(int64_t)(n0 + row - BM) * p.ldw + k];
                }
                (row < BM ? xs + row * PITCH : ws + (row - BM) * PITCH)[i % BK] = v;
            }
        }
        __syncthreads();
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
                for (int j = 0; j < 4; ++j) mma_s8(acc[i][j], a[i], b[j]);
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
                    if (n < p.N) {
                        const float b = p.bias ? DType<T>::to_f(((const T*)p.bias)[n]) : 0.f;
                        ((T*)p.y)[m * p.ldy + n] = DType<T>::from_f(fmaf((float)acc[i][j][2 * h + e], s * p.ws[n], b));
                    }
                }
        }
}

template <typename T> int int8_launch(const Int8Params& p, cudaStream_t s) {
    const int64_t gm = (p.M + BM - 1) / BM, gn = (p.N + BN - 1) / BN;
    if (gm >= (1ll << 31) || gn > 65535) return VIG_ERR_SHAPE;
    int8_any_kernel<T><<<dim3((unsigned)gm, (unsigned)gn), 128, 0, s>>>(p);
    return (int)cudaGetLastError();
}

}  // namespace
}  // namespace vig

using namespace vig;

extern "C" int vig_linear_int8_fwd(const void* x, int64_t ldx, const float* x_scales, const void* w, int64_t ldw, const float* w_scales, const void* bias, void* y,
                                   int64_t ldy, int64_t M, int N, int K, int dtype, int32_t* status_dev, void* stream) {
    if (dtype < VIG_DTYPE_F32 || dtype > VIG_DTYPE_F16) return VIG_ERR_DTYPE;
    if (M < 0 || N < 0 || K < 0 || K > 131072 || M >= (1ll << 36) || N > 4194240) return VIG_ERR_SHAPE;
    if (!M || !N) return VIG_OK;
    if (!x_scales || !w_scales || !y || (K && (!x || !w))) return VIG_ERR_NULL;
    (void)status_dev;
    Int8Params p{(const int8_t*)x, (const int8_t*)w, x_scales, w_scales, bias, y, ldx, ldw, ldy, M, N, K, 0};
    p.whole = K % 16 == 0 && ((uintptr_t)x | (uintptr_t)w) % 16 == 0 && (ldx | ldw) % 16 == 0;
    switch (dtype) {
        case VIG_DTYPE_F32: return int8_launch<float>(p, (cudaStream_t)stream);
        case VIG_DTYPE_BF16: return int8_launch<__nv_bfloat16>(p, (cudaStream_t)stream);
        default: return int8_launch<__half>(p, (cudaStream_t)stream);
    }
}
