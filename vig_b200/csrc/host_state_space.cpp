// Host side of the operators of blocks with a selective state space: checks, outputs, workspaces, autograd nodes.  The Python entry points (ops.py) only
// name the arguments; what the checks reject raises here.
#include "host_checks.h"

namespace vig_host {

namespace {

void set2(int64_t* to, const Tensor& t) { if (t.defined()) { to[0] = t.stride(0); to[1] = t.stride(1); } }

// whether no two elements of a tensor that is written in place share memory
bool apart(const Tensor& t) {
    std::vector<std::pair<int64_t, int64_t>> dims;
    for (int64_t i = 0; i < t.dim(); ++i) {
        if (t.size(i) == 0) return true;
        if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
    }
    std::sort(dims.begin(), dims.end());
    int64_t reach = 1;                                           // elements that the smaller dimensions span
    for (const auto& [stride, size] : dims) {
        if (stride < reach) return false;
        reach += stride * (size - 1);
    }
    return true;
}

void no_grad_for(std::initializer_list<const Tensor*> ts, const char* msg) { if (wants_grad(ts)) not_implemented(msg); }

// int32 [B], or undefined
Tensor lengths_of(const OptT& given, const Tensor& x) {
    const Tensor n = get(given);
    if (!n.defined()) return n;
    same_device(n, x, "lengths");
    want_type(n.scalar_type() == at::kInt || n.scalar_type() == at::kLong, "lengths must be int32 or int64");
    want(n.dim() == 1 && n.size(0) == x.size(0), "lengths must be [B]; got " + shape_of(n));
    return n.scalar_type() == at::kInt ? n.contiguous() : n.clamp(0, x.size(1)).to(at::kInt);
}

// a parameter of x's dtype or float32
void check_param(const Tensor& t, const Tensor& x, int64_t n, const char* name) {
    if (!t.defined()) return;
    same_device(t, x, name);
    want_type(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, std::string(name) + " must have the input's dtype or float32");
    want(t.dim() == 1 && t.size(0) == n && t.is_contiguous(), std::string(name) + " must be a contiguous [D] tensor; got " + shape_of(t));
}

// ---- selective scan ----
struct Scan {
    Tensor u, dt, A, B, C, D, z, bias, h0, lengths;
};

void check_scan(const Scan& s, int dim) {
    const Tensor& u = s.u;
    on_gpu(u);
    code(u);
    const char* shape = dim == 3 ? "[B, L, D]" : "[B, D]";
    want(u.dim() == dim, std::string("u must be ") + shape + "; got " + shape_of(u));
    for (const auto& [t, name] : {std::pair<const Tensor*, const char*>{&s.dt, "dt"}, {&s.z, "z"}}) {
        if (!t->defined()) continue;
        same_device(*t, u, name);
        want_type(t->scalar_type() == u.scalar_type(), std::string(name) + " must have u's dtype");
        want(t->sizes() == u.sizes(), std::string(name) + " must have u's shape; got " + shape_of(*t) + " and " + shape_of(u));
        want(unit_last(*t), std::string("the last dimension of ") + name + " must be contiguous");
    }
    want(unit_last(u), "the last dimension of u must be contiguous");
    const int64_t D = u.size(-1);
    same_device(s.A, u, "A");
    want_type(s.A.scalar_type() == at::kFloat, "A must be float32");
    want(s.A.dim() == 2 && s.A.size(0) == D && s.A.is_contiguous(), "A must be a contiguous [D, N] tensor; got " + shape_of(s.A));
    const int64_t N = s.A.size(1);
    want(N >= 1 && N <= 64, "1 to 64 states a channel are supported; got " + std::to_string(N));
    for (const auto& [t, name] : {std::pair<const Tensor*, const char*>{&s.B, "B"}, {&s.C, "C"}}) {
        same_device(*t, u, name);
        want_type(t->scalar_type() == u.scalar_type(), std::string(name) + " must have u's dtype");
        bool ok = (t->dim() == dim || t->dim() == dim + 1) && t->dim() == s.B.dim() && t->size(-1) == N && unit_last(*t);
        for (int i = 0; ok && i + 1 < dim; ++i) ok = t->size(i) == u.size(i);
        if (ok && t->dim() == dim + 1) ok = t->size(dim - 1) >= 1 && t->size(dim - 1) == s.B.size(dim - 1) && D % t->size(dim - 1) == 0;
        want(ok, std::string(name) + (dim == 3 ? " must be [B, L, N] or [B, L, G, N]" : " must be [B, N] or [B, G, N]") + " with G dividing D, B and C alike, and a contiguous last dimension; got " + shape_of(*t));
    }
    check_param(s.D, u, D, "D");
    check_param(s.bias, u, D, "dt_bias");
    want(u.size(0) * D < (1ll << 31) && D < (1ll << 28) && (dim == 2 || u.size(1) < (1ll << 30)), "B * D must be below 2^31, D below 2^28 and L below 2^30");
}
void check_states(const Tensor& h, const Scan& s, const char* name) {
    same_device(h, s.u, name);
    want_type(h.scalar_type() == at::kFloat, std::string(name) + " must be float32");
    const int64_t N = s.A.size(1);
    want(h.dim() == 3 && h.size(0) == s.u.size(0) && h.size(1) == s.u.size(-1) && h.size(2) == N && (N == 1 || h.stride(2) == 1) && (h.size(1) <= 1 || h.stride(1) == N),
         std::string(name) + " must be [B, D, N] with contiguous [D, N]; got " + shape_of(h));
}

vig_selective_scan_args scan_args(const Scan& s, bool softplus) {
    vig_selective_scan_args a{};
    const int dim = (int)s.u.dim();
    a.B = (int32_t)s.u.size(0); a.L = dim == 3 ? (int32_t)s.u.size(1) : 1; a.D = (int32_t)s.u.size(-1); a.N = (int32_t)s.A.size(1);
    a.G = s.B.dim() == dim + 1 ? (int32_t)s.B.size(dim - 1) : 1;
    a.dtype = dtype_code(s.u); a.softplus = softplus;
    a.skip_dtype = s.D.defined() ? dtype_code(s.D) : 0; a.bias_dtype = s.bias.defined() ? dtype_code(s.bias) : 0;
    a.u = ptr(s.u); a.dt = ptr(s.dt); a.z = ptr(s.z); a.b = ptr(s.B); a.c = ptr(s.C); a.A = (const float*)ptr(s.A); a.skip = ptr(s.D); a.dt_bias = ptr(s.bias);
    a.lengths = (const int32_t*)ptr(s.lengths); a.h0 = (const float*)ptr(s.h0); a.ld_h0 = s.h0.defined() ? s.h0.stride(0) : 0;
    const auto rows = [&](int64_t* to, const Tensor& t) { if (t.defined()) { to[0] = t.stride(0); to[1] = dim == 3 ? t.stride(1) : 0; } };
    rows(a.s_u, s.u); rows(a.s_dt, s.dt); rows(a.s_z, s.z);
    const auto maps = [&](int64_t* to, const Tensor& t) { rows(to, t); to[2] = t.dim() == dim + 1 ? t.stride(dim - 1) : 0; };
    maps(a.s_b, s.B); maps(a.s_c, s.C);
    a.status = status_ptr(s.u.get_device());
    return a;
}

std::pair<Tensor, Tensor> scan_forward(const Scan& s, bool want_final, bool softplus, Tensor* states) {
    vig_selective_scan_args a = scan_args(s, softplus);
    const Tensor y = fresh(s.u.sizes(), s.u);
    Tensor fin;
    if (want_final) fin = fresh({a.B, a.D, a.N}, s.u, at::kFloat);
    if (states) {
        *states = fresh({(int64_t)(api.vig_selective_scan_states_bytes(a.B, a.L, a.D, a.N) / sizeof(float))}, s.u, at::kFloat);
        a.states = (float*)ptr(*states);
    }
    a.y = ptr(y); set2(a.s_y, y);
    a.h_final = (float*)ptr(fin); a.ld_final = (int64_t)a.D * a.N;
    ok(api.vig_selective_scan_fwd(&a, stream()), "vig_selective_scan_fwd");
    return {y, fin};
}

struct ScanNode : torch::autograd::Function<ScanNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const OptT& D, const OptT& z,
                                 const OptT& bias, const OptT& h0, const OptT& lengths, bool want_final, bool softplus) {
        at::AutoDispatchBelowADInplaceOrView guard;
        const Scan s{u, dt, A, B, C, get(D), get(z), get(bias), get(h0), get(lengths)};
        Tensor states;
        const auto [y, fin] = scan_forward(s, want_final, softplus, &states);
        ctx->save_for_backward({u, dt, A, B, C, s.D, s.z, s.bias, s.lengths, states});
        ctx->saved_data["softplus"] = softplus;
        ctx->saved_data["h0"] = s.h0.defined();
        variable_list out{y};
        if (want_final) out.push_back(fin);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list d) {
        const auto saved = ctx->get_saved_variables();
        once(d, saved);
        const Scan s{saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], saved[6], saved[7], Tensor(), saved[8]};
        c10::cuda::CUDAGuard dev(s.u.device());
        const bool with_h0 = ctx->saved_data["h0"].toBool();
        vig_selective_scan_args a = scan_args(s, ctx->saved_data["softplus"].toBool());
        const Tensor dy = d[0].defined() ? rows(d[0]) : at::zeros(s.u.sizes(), s.u.options());
        const Tensor df = d.size() > 1 && d[1].defined() ? d[1].contiguous() : Tensor();
        const bool none = a.B == 0 || a.D == 0;                  // no channel or no sequence: what is summed over them is zero
        const auto like = [&](const Tensor& t) { return !t.defined() ? Tensor() : none ? at::zeros(t.sizes(), t.options()) : fresh(t.sizes(), t); };
        const Tensor du = like(s.u), ddt = like(s.u), dz = like(s.z), dA = like(s.A), dB = like(s.B), dC = like(s.C), dD = like(s.D), dbias = like(s.bias);
        Tensor d0;
        if (with_h0) d0 = fresh({a.B, a.D, a.N}, s.u, at::kFloat);
        if (!none) {
            const size_t n = api.vig_selective_scan_bwd_workspace_bytes(a.B, a.L, a.D, a.N, a.G);
            const Tensor ws = fresh({(int64_t)n}, s.u, at::kByte);
            a.states = (float*)ptr(saved[9]);
            a.d_y = ptr(dy); set2(a.s_dy, dy); a.d_final = (const float*)ptr(df);
            a.d_u = ptr(du); a.d_dt = ptr(ddt); a.d_z = ptr(dz); a.d_b = ptr(dB); a.d_c = ptr(dC); a.d_A = (float*)ptr(dA); a.d_skip = ptr(dD); a.d_bias = ptr(dbias); a.d_h0 = (float*)ptr(d0);
            a.workspace = ptr(ws); a.workspace_bytes = n;
            ok(api.vig_selective_scan_bwd(&a, stream()), "vig_selective_scan_bwd");
        }
        return {du, ddt, dA, dB, dC, dD, dz, dbias, d0, Tensor(), Tensor(), Tensor()};
    }
};

// nullopt: the device's error word has to be registered first
std::optional<std::pair<Tensor, OptT>> selective_scan(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const OptT& D, const OptT& z, const OptT& bias,
                                       const OptT& h0, bool want_final, bool softplus, const OptT& lengths) {
    Scan s{u, dt, A, B, C, get(D), get(z), get(bias), get(h0), Tensor()};
    check_scan(s, 3);
    if (!status_known(u.get_device())) return std::nullopt;
    if (s.h0.defined()) check_states(s.h0, s, "initial_state");
    no_tangents({&u, &dt, &A, &B, &C, &s.D, &s.z, &s.bias, &s.h0});
    c10::cuda::CUDAGuard dev(u.device());
    s.lengths = lengths_of(lengths, u);
    if (wants_grad({&u, &dt, &A, &B, &C, &s.D, &s.z, &s.bias, &s.h0})) {
        const auto out = ScanNode::apply(u, dt, A, B, C, D, z, bias, h0, s.lengths.defined() ? OptT(s.lengths) : OptT(), want_final, softplus);
        return std::make_pair(out[0], want_final ? OptT(out[1]) : OptT());
    }
    const auto [y, fin] = scan_forward(s, want_final, softplus, nullptr);
    return std::make_pair(y, want_final ? OptT(fin) : OptT());
}

Tensor selective_scan_step(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& state, const OptT& D, const OptT& z, const OptT& bias,
                           bool softplus) {
    const Scan s{u, dt, A, B, C, get(D), get(z), get(bias), Tensor(), Tensor()};
    check_scan(s, 2);
    check_states(state, s, "state");
    want(apart(state), "the rows of state must not overlap: it is updated in place");
    no_tangents({&u, &dt, &A, &B, &C, &s.D, &s.z, &s.bias, &state});
    no_grad_for({&u, &dt, &A, &B, &C, &s.D, &s.z, &s.bias, &state}, "selective_scan_step updates its state in place and has no gradient: use selective_scan, or torch.no_grad()");
    c10::cuda::CUDAGuard dev(u.device());
    state.unsafeGetTensorImpl()->bump_version();
    const Tensor y = fresh(u.sizes(), u);
    vig_selective_scan_args a = scan_args(s, softplus);
    a.y = ptr(y); a.s_y[0] = y.stride(0);
    a.h_final = (float*)ptr(state); a.ld_final = state.stride(0);
    ok(api.vig_selective_scan_step(&a, stream()), "vig_selective_scan_step");
    return y;
}

// ---- causal convolution ----
void check_conv(const Tensor& x, const Tensor& w, const Tensor& bias, int dim) {
    on_gpu(x);
    code(x);
    want(x.dim() == dim && unit_last(x), std::string("x must be ") + (dim == 3 ? "[B, L, D]" : "[B, D]") + " with a contiguous last dimension; got " + shape_of(x));
    same_device(w, x, "weight");
    want_type(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, "weight must have x's dtype or float32");
    want(w.dim() == 2 && w.size(0) == x.size(-1) && w.is_contiguous(), "weight must be a contiguous [D, K] tensor; got " + shape_of(w));
    want(w.size(1) >= 1 && w.size(1) <= 8, "1 to 8 taps are supported; got " + std::to_string(w.size(1)));
    check_param(bias, x, x.size(-1), "bias");
    want_type(!bias.defined() || bias.scalar_type() == w.scalar_type(), "bias must have weight's dtype");
    want(x.size(0) * x.size(-1) < (1ll << 31) && x.size(-1) < (1ll << 28) && (dim == 2 || x.size(1) < (1ll << 30)), "B * D must be below 2^31, D below 2^28 and L below 2^30");
}
void check_window(const Tensor& s, const Tensor& x, const Tensor& w, const char* name) {
    same_device(s, x, name);
    want_type(s.scalar_type() == x.scalar_type(), std::string(name) + " must have x's dtype");
    want(s.dim() == 3 && s.size(0) == x.size(0) && s.size(1) == w.size(1) - 1 && s.size(2) == x.size(-1) && unit_last(s),
         std::string(name) + " must be [B, K - 1, D] with a contiguous last dimension; got " + shape_of(s));
}

std::pair<Tensor, Tensor> conv_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state, const Tensor& lengths, bool want_final, bool silu) {
    const Tensor y = fresh(x.sizes(), x);
    Tensor fin;
    int64_t sx[2], sy[2], ss[2] = {}, sf[2] = {};
    set2(sx, x); set2(sy, y); set2(ss, state);
    if (want_final) { fin = fresh({x.size(0), w.size(1) - 1, x.size(2)}, x); set2(sf, fin); }
    ok(api.vig_causal_conv_fwd(ptr(x), ptr(w), dtype_code(w), ptr(bias), ptr(state), ptr(y), ptr(fin), (const int32_t*)ptr(lengths), (int)x.size(0), (int)x.size(1), (int)x.size(2),
                               (int)w.size(1), sx, sy, ss, sf, silu, dtype_code(x), stream()), "vig_causal_conv_fwd");
    return {y, fin};
}

struct ConvNode : torch::autograd::Function<ConvNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptT& bias, const OptT& state, const OptT& lengths, bool want_final, bool silu) {
        at::AutoDispatchBelowADInplaceOrView guard;
        const auto [y, fin] = conv_forward(x, w, get(bias), get(state), get(lengths), want_final, silu);
        ctx->save_for_backward({x, w, get(bias), get(state), get(lengths)});
        ctx->saved_data["silu"] = silu;
        variable_list out{y};
        if (want_final) out.push_back(fin);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list d) {
        const auto saved = ctx->get_saved_variables();
        once(d, saved);
        const Tensor &x = saved[0], &w = saved[1], &bias = saved[2], &state = saved[3], &lengths = saved[4];
        c10::cuda::CUDAGuard dev(x.device());
        const Tensor dy = d[0].defined() ? rows(d[0]) : at::zeros(x.sizes(), x.options());
        const Tensor df = d.size() > 1 && d[1].defined() ? d[1].contiguous() : Tensor();
        const int B = (int)x.size(0), L = (int)x.size(1), D = (int)x.size(2), K = (int)w.size(1);
        const bool none = B == 0 || D == 0;
        const auto like = [&](const Tensor& t) { return !t.defined() ? Tensor() : none ? at::zeros(t.sizes(), t.options()) : fresh(t.sizes(), t); };
        const Tensor dx = like(x), dw = like(w), db = like(bias), ds = like(state);
        if (!none) {
            const size_t n = api.vig_causal_conv_bwd_workspace_bytes(B, L, D, K);
            const Tensor ws = fresh({(int64_t)n}, x, at::kByte);
            int64_t sx[2], ss[2] = {}, sd[2];
            set2(sx, x); set2(ss, state); set2(sd, dy);
            ok(api.vig_causal_conv_bwd(ptr(x), ptr(w), dtype_code(w), ptr(bias), ptr(state), ptr(dy), ptr(df), (const int32_t*)ptr(lengths), ptr(dx), ptr(dw), ptr(db), ptr(ds), B, L, D, K,
                                       sx, ss, sd, ctx->saved_data["silu"].toBool(), dtype_code(x), ptr(ws), n, stream()), "vig_causal_conv_bwd");
        }
        return {dx, dw, db, ds, Tensor(), Tensor(), Tensor()};
    }
};

std::pair<Tensor, OptT> causal_conv(const Tensor& x, const Tensor& w, const OptT& bias_, const OptT& state_, bool want_final, bool silu, const OptT& lengths_) {
    const Tensor bias = get(bias_), state = get(state_);
    check_conv(x, w, bias, 3);
    if (state.defined()) check_window(state, x, w, "initial_state");
    no_tangents({&x, &w, &bias, &state});
    c10::cuda::CUDAGuard dev(x.device());
    const Tensor lengths = lengths_of(lengths_, x);
    if (wants_grad({&x, &w, &bias, &state})) {
        const auto out = ConvNode::apply(x, w, bias_, state_, lengths.defined() ? OptT(lengths) : OptT(), want_final, silu);
        return {out[0], want_final ? OptT(out[1]) : OptT()};
    }
    const auto [y, fin] = conv_forward(x, w, bias, state, lengths, want_final, silu);
    return {y, want_final ? OptT(fin) : OptT()};
}

Tensor causal_conv_step(const Tensor& x, const Tensor& state, const Tensor& w, const OptT& bias_, bool silu) {
    const Tensor bias = get(bias_);
    check_conv(x, w, bias, 2);
    check_window(state, x, w, "state");
    want(apart(state), "the rows of state must not overlap: it is updated in place");
    no_tangents({&x, &w, &bias, &state});
    no_grad_for({&x, &w, &bias, &state}, "causal_conv_step updates its state in place and has no gradient: use causal_conv, or torch.no_grad()");
    c10::cuda::CUDAGuard dev(x.device());
    state.unsafeGetTensorImpl()->bump_version();
    const Tensor y = fresh(x.sizes(), x);
    int64_t ss[2];
    set2(ss, state);
    ok(api.vig_causal_conv_step(ptr(x), x.stride(0), ptr(state), ss, ptr(w), dtype_code(w), ptr(bias), ptr(y), y.stride(0), (int)x.size(0), (int)x.size(1), (int)w.size(1), silu,
                                dtype_code(x), stream()), "vig_causal_conv_step");
    return y;
}

// ---- layer norm ----
void check_layer(const Tensor& x, const Tensor& w, const Tensor& bias, std::initializer_list<std::pair<const Tensor*, const char*>> like) {
    on_gpu(x);
    code(x);
    want(x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) < (1ll << 30), "x must be [..., N] with 0 < N < 2^30");
    for (const auto& [t, name] : {std::pair<const Tensor*, const char*>{&w, "weight"}, {&bias, "bias"}}) {
        if (!t->defined()) continue;
        same_device(*t, x, name);
        want(t->dim() == 1 && t->size(0) == x.size(-1) && t->is_contiguous(), std::string(name) + " must be a contiguous [N] tensor");
        want_type(t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat, std::string(name) + " must have x's dtype or float32");
        want_type(t->scalar_type() == w.scalar_type(), "bias must have weight's dtype");
    }
    for (const auto& [t, name] : like) {
        if (!t->defined()) continue;
        same_device(*t, x, name);
        want_type(t->scalar_type() == x.scalar_type(), std::string(name) + " must have x's dtype");
        want(t->sizes() == x.sizes(), std::string(name) + " must have x's shape; got " + shape_of(*t) + " and " + shape_of(x));
    }
}

std::pair<Tensor, Tensor> layer_forward(const Tensor& x_, const Tensor& w, const Tensor& bias, const Tensor& res0, double eps) {
    const Tensor x = as_rows(x_), res = res0.defined() ? as_rows(res0) : res0, y = fresh(x_.sizes(), x);
    Tensor r;
    if (res.defined()) r = fresh(x_.sizes(), x);
    ok(api.vig_add_layernorm_train_fwd(ptr(x), ld(x), ptr(res), ld(res), ptr(w), ptr(bias), dtype_code(w), ptr(y), ptr(r), x.size(0), (int)x.size(1), (float)eps, dtype_code(x), stream()),
       "vig_add_layernorm_train_fwd");
    return {y, r};
}

std::tuple<Tensor, Tensor, Tensor> layer_backward(const Tensor& dy_, const Tensor& x_, const Tensor& res_, const Tensor& w, bool with_bias, const Tensor& dr_, double eps) {
    const Tensor x = as_rows(x_), dy = as_rows(dy_), dr = dr_.defined() ? as_rows(dr_) : dr_, res = res_.defined() ? as_rows(res_) : res_;
    const Tensor dx = fresh(x_.sizes(), x), dw = fresh(w.sizes(), w);
    Tensor db, ws;
    if (with_bias) db = fresh(w.sizes(), w);
    const size_t n = api.vig_add_layernorm_bwd_workspace_bytes(x.size(0), (int)x.size(1));
    if (n) ws = fresh({(int64_t)n}, x, at::kByte);
    ok(api.vig_add_layernorm_bwd(ptr(dy), ld(dy), ptr(x), ld(x), ptr(res), ld(res), ptr(w), dtype_code(w), ptr(dr), ld(dr), ptr(dx), ptr(dw), ptr(db), x.size(0), (int)x.size(1),
                                 (float)eps, dtype_code(x), ptr(ws), n, stream()), "vig_add_layernorm_bwd");
    return {dx, dw, db};
}

struct LayerNode : torch::autograd::Function<LayerNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptT& bias, const OptT& res, double eps) {
        at::AutoDispatchBelowADInplaceOrView guard;
        const auto [y, r] = layer_forward(x, w, get(bias), get(res), eps);
        // fp32: the sum, which is what it was; 16 bits: what was added, because the sum was rounded
        if (r.defined() && r.scalar_type() != at::kFloat) ctx->save_for_backward({x, w, *res});
        else ctx->save_for_backward({r.defined() ? r : x, w, Tensor()});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["bias"] = get(bias).defined();
        ctx->saved_data["residual"] = r.defined();
        variable_list out{y};
        // without a residual x itself, as a result of this node, so that what comes back through it is added before dx is rounded
        if (r.defined() || x.requires_grad()) out.push_back(r.defined() ? r : x);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list d) {
        const auto saved = ctx->get_saved_variables();
        once(d, saved);
        const Tensor &x = saved[0], &w = saved[1], &res = saved[2];
        c10::cuda::CUDAGuard dev(x.device());
        const Tensor dy = d[0].defined() ? d[0] : at::zeros(x.sizes(), x.options());
        const auto [dx, dw, db] = layer_backward(dy, x, res, w, ctx->saved_data["bias"].toBool(), d.size() > 1 ? d[1] : Tensor(), ctx->saved_data["eps"].toDouble());
        return {dx, dw, db, ctx->saved_data["residual"].toBool() ? dx : Tensor(), Tensor()};
    }
};

std::pair<Tensor, Tensor> add_layernorm_train(const Tensor& x, const Tensor& w, const OptT& bias_, const OptT& res_, double eps) {
    const Tensor res = get(res_), bias = get(bias_);
    check_layer(x, w, bias, {{&res, "residual"}});
    want(eps >= 0, "eps must not be negative");
    no_tangents({&x, &w, &bias, &res});
    c10::cuda::CUDAGuard dev(x.device());
    if (wants_grad({&x, &w, &bias, &res})) {
        const auto out = LayerNode::apply(x, w, bias_, res_, eps);
        return {out[0], out.size() > 1 ? out[1] : x};
    }
    const auto [y, r] = layer_forward(x, w, bias, res, eps);
    return {y, r.defined() ? r : x};
}

std::tuple<Tensor, Tensor, Tensor> add_layernorm_backward(const Tensor& dy, const Tensor& r, const Tensor& w, double eps, const OptT& dr_, const OptT& res_) {
    const Tensor dr = get(dr_), res = get(res_);
    check_layer(r, w, Tensor(), {{&dy, "d_y"}, {&dr, "d_r"}, {&res, "residual"}});
    want(eps >= 0, "eps must not be negative");
    no_tangents({&dy, &r, &w, &dr, &res});
    c10::cuda::CUDAGuard dev(r.device());
    return layer_backward(dy, r, res, w, true, dr, eps);
}

// ---- 8-bit product ----
// nullopt: the device's error word has to be registered first
std::optional<Tensor> linear_int8(const Tensor& q, const Tensor& scales, const Tensor& w, const Tensor& w_scales, const OptT& bias_, int64_t out) {
    const Tensor bias = get(bias_);
    const at::ScalarType type = out == VIG_DTYPE_F32 ? at::kFloat : out == VIG_DTYPE_BF16 ? at::kBFloat16 : at::kHalf;
    on_gpu(q);
    same_device(scales, q, "scales"); same_device(w, q, "weight"); same_device(w_scales, q, "weight_scales");
    want_type(q.scalar_type() == at::kChar && w.scalar_type() == at::kChar, "q and weight must be int8");
    want_type(scales.scalar_type() == at::kFloat && w_scales.scalar_type() == at::kFloat, "scales are float32");
    want(q.dim() >= 1 && w.dim() == 2 && q.size(-1) == w.size(1), "q must be [..., K] and weight [N, K]; got " + shape_of(q) + " and " + shape_of(w));
    want(unit_last(w), "the last dimension of weight must be contiguous");
    const int64_t K = w.size(1), N = w.size(0);
    auto sizes = q.sizes().vec();
    sizes.pop_back();
    const at::IntArrayRef lead(sizes);
    auto column = sizes;
    column.push_back(1);
    want(scales.sizes() == lead || scales.sizes() == at::IntArrayRef(column), "scales must have one value a row of q, [...] or [..., 1]; got " + shape_of(scales));
    want(w_scales.numel() == N && (w_scales.dim() == 1 || (w_scales.dim() == 2 && w_scales.size(1) == 1)), "weight_scales must be [N] or [N, 1]; got " + shape_of(w_scales));
    want(K <= 131071 && N <= 4194240, "K must be 131071 at most (larger sums leave 32 bits), N 4194240");
    if (bias.defined()) {
        same_device(bias, q, "bias");
        want_type(bias.scalar_type() == type, "bias must have the output's dtype");
        want(bias.dim() == 1 && bias.size(0) == N && bias.is_contiguous(), "bias must be a contiguous [N] tensor");
    }
    no_tangents({&scales, &w_scales, &bias});
    no_grad_for({&scales, &w_scales, &bias}, "linear_int8 has no gradient: use it under torch.no_grad()");
    if (!status_known(q.get_device())) return std::nullopt;
    c10::cuda::CUDAGuard dev(q.device());
    sizes.push_back(N);
    const Tensor y = fresh(sizes, q, type);
    const int64_t M = N ? y.numel() / N : 0;
    Tensor x = q.dim() == 2 && unit_last(q) ? q : rows(q.reshape({M ? M : (K ? q.numel() / K : 0), K})), w16 = w;
    const Tensor s = scales.contiguous(), ws = w_scales.contiguous();
    int64_t ldx = x.size(0) > 1 ? x.stride(0) : K, ldw = N > 1 ? w.stride(0) : K, width = K;
    if (api.vig_linear_int8_laid_out_first(ptr(x), ldx, ptr(w), ldw, M, (int)N, (int)K)) {
        width = (K + 15) / 16 * 16;
        const Tensor x2 = fresh({M, width}, q), w2 = fresh({N, width}, q);
        ok(api.vig_int8_rows_lay_out(ptr(x), ldx, ptr(x2), M, (int)K, stream()), "vig_int8_rows_lay_out");
        ok(api.vig_int8_rows_lay_out(ptr(w), ldw, ptr(w2), N, (int)K, stream()), "vig_int8_rows_lay_out");
        x = x2; w16 = w2; ldx = ldw = width;
    }
    ok(api.vig_linear_int8_fwd(ptr(x), ldx, (const float*)ptr(s), ptr(w16), ldw, (const float*)ptr(ws), ptr(bias), ptr(y), N, M, (int)N, (int)width, (int)out,
                               status_ptr(q.get_device()), stream()), "vig_linear_int8_fwd");
    return y;
}

}  // namespace

void bind_state_space(py::module_& m) {
    m.def("selective_scan", &selective_scan);
    m.def("selective_scan_step", &selective_scan_step);
    m.def("causal_conv", &causal_conv);
    m.def("causal_conv_step", &causal_conv_step);
    m.def("add_layernorm_train", &add_layernorm_train);
    m.def("add_layernorm_backward", &add_layernorm_backward);
    m.def("linear_int8", &linear_int8);
}

}  // namespace vig_host
