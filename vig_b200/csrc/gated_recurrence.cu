// Gated linear recurrence with one state per channel, h_t = a_t h_{t-1} + x_t, along either direction of a sequence: forward, all
// gradients, and the one-token form (the same call with L = 1 and the state updated in place).
//
// a_t = exp(g_t) from log-gates, or sigmoid(z_t)^(1/n) = exp(logsigmoid(z_t)/n) from raw logits z with n = gate_logit_normalizer.
// Gradients: u_t = a_t (dh_t + u_{t+1}), the same recurrence from the other end;  dx_t = dh_t + u_{t+1},  dg_t = u_t h_{t-1},
// dz_t = dg_t (1 - sigmoid(z_t)) / n,  dh_{-1} = u_0.  States, decays and sums are fp32; h is rounded once, to x's type, and the
// backward reads h_{t-1} as it was rounded, so that x is not read again.
// Bound by memory: 3 tensors forward (x, g in, h out), 5 backward (g, h, dh in, dx, dg out), about one exponential and a multiply-add a value.
#include "common.cuh"

namespace vig {

struct RecParams {
    const void *x, *g;              // backward: x is dh
    const void* h_in;               // backward: the forward's h
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
};

// decay of one token
template <bool LOGITS> __device__ __forceinline__ float decay_of(float g, float inv_norm) {
    return expf(LOGITS ? log_sigmoid(g) * inv_norm : g);
}

// ---------------------------------------------------------------------------------------------------
// A thread owns a channel and walks its sequence.
template <typename T, bool LOGITS, bool BWD>
__global__ void __launch_bounds__(128) rec_serial_kernel(const RecParams p) {
    const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (i >= (int64_t)p.B * p.D) return;
    const int b = (int)(i / p.D), d = (int)(i % p.D);
    const T* x = (const T*)p.x + b * p.sx[0] + d;
    const T* g = (const T*)p.g + b * p.sg[0] + d;
    const T* hin = BWD ? (const T*)p.h_in + b * p.sh[0] + d : nullptr;
    T* out = (T*)p.out + b * p.so[0] + d;
    T* outg = BWD ? (T*)p.out_g + b * p.sog[0] + d : nullptr;
    float s = p.s0 ? p.s0[b * p.ld_s0 + d] : 0.f;
    for (int k = 0; k < p.L; ++k) {
        const int64_t t = p.from_end ? p.L - 1 - k : k;
        const float gv = DType<T>::to_f(g[t * p.sg[1]]), a = decay_of<LOGITS>(gv, p.inv_norm);
        const float xv = DType<T>::to_f(x[t * p.sx[1]]);
        if (!BWD) {
            s = fmaf(a, s, xv);
            out[t * p.so[1]] = DType<T>::from_f(s);
        } else {
            const float dx = xv + s;
            s = a * dx;
            const int64_t before = p.from_end ? t - 1 : t + 1;
            const float hb = k + 1 < p.L ? DType<T>::to_f(hin[before * p.sh[1]]) : p.h0 ? p.h0[(int64_t)b * p.D + d] : 0.f;
            float dg = s * hb;
            if (LOGITS) dg *= p.inv_norm / (1.f + expf(gv));
            out[t * p.so[1]] = DType<T>::from_f(dx);
            outg[t * p.sog[1]] = DType<T>::from_f(dg);
        }
    }
    if (p.s_end) p.s_end[b * p.ld_end + d] = s;
}

template <typename T, bool LOGITS, bool BWD>
int rec_launch(const RecParams& p, cudaStream_t s) {
    const int64_t n = (int64_t)p.B * p.D;
    rec_serial_kernel<T, LOGITS, BWD><<<(unsigned)((n + 127) / 128), 128, 0, s>>>(p);
    return (int)cudaGetLastError();
}

template <bool BWD> int rec_dispatch(const RecParams& p, int dtype, cudaStream_t s) {
    switch (dtype) {
        case VIG_DTYPE_F32: return p.inv_norm > 0.f ? rec_launch<float, true, BWD>(p, s) : rec_launch<float, false, BWD>(p, s);
        case VIG_DTYPE_BF16: return p.inv_norm > 0.f ? rec_launch<__nv_bfloat16, true, BWD>(p, s) : rec_launch<__nv_bfloat16, false, BWD>(p, s);
        case VIG_DTYPE_F16: return p.inv_norm > 0.f ? rec_launch<__half, true, BWD>(p, s) : rec_launch<__half, false, BWD>(p, s);
    }
    return VIG_ERR_DTYPE;
}

// sizes every call has to have; VIG_OK with *empty set where there is nothing to do
static int rec_check(int B, int L, int D, float norm, int dtype) {
    if (dtype < VIG_DTYPE_F32 || dtype > VIG_DTYPE_F16) return VIG_ERR_DTYPE;
    if (B < 0 || L < 0 || D < 0 || (int64_t)B * D >= (1ll << 31)) return VIG_ERR_SHAPE;
    if (!(norm >= 0.f) || norm > 3.4e38f) return VIG_ERR_ARG;
    return VIG_OK;
}

// no token: the state that enters is the state that leaves
static int rec_empty(const float* s0, int64_t ld0, float* s_end, int64_t ld_end, int B, int D, cudaStream_t s) {
    if (!s_end || s_end == s0 || !B || !D) return VIG_OK;
    return (int)(s0 ? cudaMemcpy2DAsync(s_end, ld_end * 4, s0, ld0 * 4, (size_t)D * 4, B, cudaMemcpyDeviceToDevice, s)
                    : cudaMemset2DAsync(s_end, ld_end * 4, 0, (size_t)D * 4, B, s));
}

static void two(int64_t* dst, const int64_t* src, int L, int D) {
    dst[0] = src ? src[0] : (int64_t)L * D;
    dst[1] = src ? src[1] : D;
}

}  // namespace vig

using namespace vig;

extern "C" int vig_gated_recurrence_fwd(const void* x, const void* g, const float* h0, int64_t ld_h0, void* h, float* h_final, int64_t ld_final,
                                        int B, int L, int D, const int64_t* strides_x, const int64_t* strides_g, const int64_t* strides_h,
                                        float gate_logit_normalizer, int reverse, int dtype, void* stream) {
    if (const int e = rec_check(B, L, D, gate_logit_normalizer, dtype)) return e;
    if (B > 1 && ((h0 && ld_h0 < 0) || (h_final && ld_final < D))) return VIG_ERR_ARG;
    if (!B || !D || !L) return rec_empty(h0, ld_h0, h_final, ld_final, B, D, (cudaStream_t)stream);
    if (!x || !g || !h) return VIG_ERR_NULL;
    RecParams p{};
    p.x = x; p.g = g; p.s0 = h0; p.ld_s0 = ld_h0; p.out = h; p.s_end = h_final; p.ld_end = ld_final;
    two(p.sx, strides_x, L, D); two(p.sg, strides_g, L, D); two(p.so, strides_h, L, D);
    p.B = B; p.L = L; p.D = D;
    p.inv_norm = gate_logit_normalizer > 0.f ? 1.f / gate_logit_normalizer : 0.f;
    p.from_end = reverse != 0;
    return rec_dispatch<false>(p, dtype, (cudaStream_t)stream);
}

extern "C" int vig_gated_recurrence_bwd(const void* g, const void* h, const float* h0, const void* d_h, const float* d_final, void* d_x, void* d_g, float* d_h0,
                                        int B, int L, int D, const int64_t* strides_g, const int64_t* strides_h, const int64_t* strides_dh,
                                        float gate_logit_normalizer, int reverse, int dtype, void* stream) {
    if (const int e = rec_check(B, L, D, gate_logit_normalizer, dtype)) return e;
    if (!B || !D || !L) return rec_empty(d_final, D, d_h0, D, B, D, (cudaStream_t)stream);
    if (!g || !h || !d_h || !d_x || !d_g) return VIG_ERR_NULL;
    RecParams p{};
    p.x = d_h; p.g = g; p.h_in = h; p.h0 = h0; p.s0 = d_final; p.ld_s0 = D; p.out = d_x; p.out_g = d_g; p.s_end = d_h0; p.ld_end = D;
    two(p.sx, strides_dh, L, D); two(p.sg, strides_g, L, D); two(p.sh, strides_h, L, D); two(p.so, nullptr, L, D); two(p.sog, nullptr, L, D);
    p.B = B; p.L = L; p.D = D;
    p.inv_norm = gate_logit_normalizer > 0.f ? 1.f / gate_logit_normalizer : 0.f;
    p.from_end = reverse == 0;
    return rec_dispatch<true>(p, dtype, (cudaStream_t)stream);
}
