// Host side of the operators that train and serve a block with a gated recurrence: checks, outputs, workspaces, autograd nodes.  The
// Python entry points (ops.py) only name the arguments; what the checks reject raises here.
#include "host_checks.h"
#include <torch/csrc/autograd/python_variable.h>

namespace vig_host {

namespace {

struct S2 {                                    // (b, l) element strides of a [B, L, D] view
    int64_t s[2];
    explicit S2(const Tensor& t) { if (t.defined()) { s[0] = t.stride(0); s[1] = t.stride(1); } }
};

// ---- gated recurrence ----
void check_state(const Tensor& s, const Tensor& x, const char* name) {
    same_device(s, x, name);
    want_type(s.scalar_type() == at::kFloat, std::string(name) + " must be float32");
    want(s.dim() == 2 && s.size(0) == x.size(0) && s.size(1) == x.size(-1) && unit_last(s),
         std::string(name) + " must be [B, D] with a contiguous last dimension; got " + shape_of(s));
}
void check_rec(const Tensor& x, const Tensor& g, int dim, double norm) {
    on_gpu(x);
    same_device(g, x, "g");
    code(x);
    want_type(g.scalar_type() == x.scalar_type(), "x and g must share one dtype");
    want(x.dim() == dim && g.sizes() == x.sizes(), (dim == 3 ? "x and g must be [B, L, D]; got " : "x and g must be [B, D]; got ") + shape_of(x) + " and " + shape_of(g));
    want(unit_last(x) && unit_last(g), "the last dimension of x and g must be contiguous");
    want(norm == 0 || (norm >= 1e-30 && norm <= 1e30), "gate_logit_normalizer must be 0 (log-gates) or positive (raw logits; 1e-30 to 1e30)");
    want(x.size(0) * x.size(-1) < (1ll << 31) && x.size(-1) < (1ll << 28) && (dim == 2 || x.size(1) < (1ll << 30)), "B * D must be below 2^31, D below 2^28 and L below 2^30");
}

// `states` (16 bits, for a backward): what the gate gradient takes h_{t-1} from
void rec_forward(const Tensor& x, const Tensor& g, const Tensor& h0, const Tensor& h, const Tensor& fin, bool reverse, double norm, const Tensor& states = {}) {
    const S2 sx(x), sg(g), sh(h);
    if (states.defined())
        ok(api.vig_gated_recurrence_train_fwd(ptr(x), ptr(g), (const float*)ptr(h0), h0.defined() ? h0.stride(0) : 0, ptr(h), (float*)ptr(fin), fin.defined() ? fin.stride(0) : 0,
                                              (float*)ptr(states), (int)x.size(0), (int)x.size(1), (int)x.size(2), sx.s, sg.s, sh.s, (float)norm, reverse, dtype_code(x),
                                              status_ptr(x.get_device()), stream()), "vig_gated_recurrence_train_fwd");
    else ok(api.vig_gated_recurrence_fwd(ptr(x), ptr(g), (const float*)ptr(h0), h0.defined() ? h0.stride(0) : 0, ptr(h), (float*)ptr(fin), fin.defined() ? fin.stride(0) : 0,
                                    (int)x.size(0), (int)x.size(1), (int)x.size(2), sx.s, sg.s, sh.s, (float)norm, reverse, dtype_code(x), status_ptr(x.get_device()), stream()),
       "vig_gated_recurrence_fwd");
}

struct Rec : torch::autograd::Function<Rec> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& g, const OptT& h0_, bool want_final, bool reverse, double norm) {
        at::AutoDispatchBelowADInplaceOrView guard;
        const Tensor h0 = get(h0_), h = fresh(x.sizes(), x);
        Tensor fin;
        if (want_final) fin = fresh({x.size(0), x.size(2)}, x, at::kFloat);
        Tensor states;
        if (x.scalar_type() != at::kFloat)
            states = fresh({(int64_t)(api.vig_gated_recurrence_states_bytes((int)x.size(0), (int)x.size(1), (int)x.size(2)) / sizeof(float))}, x, at::kFloat);
        rec_forward(x, g, h0, h, fin, reverse, norm, states);
        ctx->save_for_backward({g, states.defined() ? x : h, h0, states});
        ctx->saved_data["reverse"] = reverse;
        ctx->saved_data["norm"] = norm;
        variable_list out{h};
        if (want_final) out.push_back(fin);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list d) {
        const auto saved = ctx->get_saved_variables();
        once(d, saved);
        // h, or x where there are states
        const Tensor g = rows(saved[0]), h = rows(saved[1]), h0 = saved[2].defined() ? saved[2].contiguous() : saved[2], states = saved[3];
        c10::cuda::CUDAGuard dev(g.device());
        const Tensor dh = d[0].defined() ? rows(d[0]) : at::zeros(h.sizes(), h.options());
        const Tensor df = d.size() > 1 && d[1].defined() ? d[1].contiguous() : Tensor();
        const Tensor dx = fresh(h.sizes(), h), dg = fresh(h.sizes(), h);
        Tensor d0;
        if (h0.defined()) d0 = fresh(h0.sizes(), h0);
        const S2 sg(g), sh(h), sd(dh);
        if (states.defined())
            ok(api.vig_gated_recurrence_train_bwd(ptr(g), ptr(h), (const float*)ptr(states), (const float*)ptr(h0), ptr(dh), (const float*)ptr(df), ptr(dx), ptr(dg), (float*)ptr(d0),
                                                  (int)h.size(0), (int)h.size(1), (int)h.size(2), sg.s, sh.s, sd.s, (float)ctx->saved_data["norm"].toDouble(),
                                                  ctx->saved_data["reverse"].toBool(), dtype_code(h), status_ptr(h.get_device()), stream()), "vig_gated_recurrence_train_bwd");
        else ok(api.vig_gated_recurrence_bwd(ptr(g), ptr(h), (const float*)ptr(h0), ptr(dh), (const float*)ptr(df), ptr(dx), ptr(dg), (float*)ptr(d0), (int)h.size(0),
                                        (int)h.size(1), (int)h.size(2), sg.s, sh.s, sd.s, (float)ctx->saved_data["norm"].toDouble(),
                                        ctx->saved_data["reverse"].toBool(), dtype_code(h), status_ptr(h.get_device()), stream()), "vig_gated_recurrence_bwd");
        return {dx, dg, d0, Tensor(), Tensor(), Tensor()};
    }
};

// nullopt: the device's error word has to be registered first
std::optional<std::pair<Tensor, OptT>> gated_recurrence(const Tensor& x, const Tensor& g, const OptT& h0_, bool want_final, bool reverse, double norm) {
    check_rec(x, g, 3, norm);
    if (!status_known(x.get_device())) return std::nullopt;
    const Tensor h0 = get(h0_);
    if (h0.defined()) check_state(h0, x, "initial_state");
    no_tangents({&x, &g, &h0});
    c10::cuda::CUDAGuard dev(x.device());
    if (wants_grad({&x, &g, &h0})) {
        const auto out = Rec::apply(x, g, h0_, want_final, reverse, norm);
        return std::make_pair(out[0], want_final ? OptT(out[1]) : OptT());
    }
    const Tensor h = fresh(x.sizes(), x);
    Tensor fin;
    if (want_final) fin = fresh({x.size(0), x.size(2)}, x, at::kFloat);
    rec_forward(x, g, h0, h, fin, reverse, norm);
    return std::make_pair(h, want_final ? OptT(fin) : OptT());
}

Tensor gated_recurrence_step(const Tensor& x, const Tensor& g, const Tensor& state, double norm) {
    check_rec(x, g, 2, norm);
    check_state(state, x, "state");
    want(state.size(0) <= 1 || state.stride(0) >= state.size(1), "the rows of state must not overlap: it is updated in place");
    no_tangents({&x, &g, &state});
    if (wants_grad({&x, &g, &state})) not_implemented("gated_recurrence_step updates its state in place and has no gradient: use gated_recurrence, or torch.no_grad()");
    c10::cuda::CUDAGuard dev(x.device());
    state.unsafeGetTensorImpl()->bump_version();
    const Tensor h = fresh(x.sizes(), x);
    const int64_t sx[2] = {x.stride(0), 0}, sg[2] = {g.stride(0), 0}, sh[2] = {h.stride(0), 0};
    ok(api.vig_gated_recurrence_fwd(ptr(x), ptr(g), (const float*)ptr(state), state.stride(0), ptr(h), (float*)ptr(state), state.stride(0), (int)x.size(0), 1, (int)x.size(1),
                                    sx, sg, sh, (float)norm, 0, dtype_code(x), status_ptr(x.get_device()), stream()), "vig_gated_recurrence_fwd");
    return h;
}

// ---- RMS norm ----
void check_norm(const Tensor& x, const Tensor& w, const Tensor& res) {
    on_gpu(x);
    same_device(w, x, "weight");
    code(x);
    want(x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) < (1ll << 30), "x must be [..., N] with 0 < N < 2^30");
    want(w.dim() == 1 && w.size(0) == x.size(-1) && w.is_contiguous(), "weight must be a contiguous [N] tensor");
    want_type(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, "weight must have x's dtype or float32");
    if (res.defined()) {
        same_device(res, x, "residual");
        want_type(res.scalar_type() == x.scalar_type(), "residual must have x's dtype");
        want(res.sizes() == x.sizes(), "residual must have x's shape; got " + shape_of(res) + " and " + shape_of(x));
    }
}

std::tuple<Tensor, Tensor, Tensor> add_rmsnorm_8bit(const Tensor& x_, const Tensor& w, const OptT& res_, double eps, int64_t out_type, int64_t group, bool prenorm) {
    const Tensor res0 = get(res_);
    check_norm(x_, w, res0);
    const int64_t N = x_.size(-1);
    want(group == 0 || group == N || ((group == 32 || group == 64 || group == 128) && N % group == 0), "group must be None, or 32, 64 or 128 and divide N");
    want(eps >= 0, "eps must not be negative");
    no_tangents({&x_, &w, &res0});
    // (without a row there is no gradient to lose)
    if (x_.numel() && wants_grad({&x_, &w, &res0})) not_implemented("add_rmsnorm_8bit has no gradient: use add_rmsnorm_train, or torch.no_grad()");
    c10::cuda::CUDAGuard dev(x_.device());
    const Tensor x = as_rows(x_), res = res0.defined() ? as_rows(res0) : res0;
    auto sizes = x_.sizes().vec();
    const Tensor q = fresh(sizes, x, out_type == VIG_OUT_E4M3 ? at::kFloat8_e4m3fn : at::kChar);
    Tensor r;
    if (prenorm && res.defined()) r = fresh(sizes, x);
    sizes.back() = group ? N / group : 1;
    const Tensor scales = fresh(sizes, x, at::kFloat);
    ok(api.vig_add_rmsnorm_8bit_fwd(ptr(x), ld(x), ptr(res), ld(res), ptr(w), dtype_code(w), ptr(q), (float*)ptr(scales), ptr(r), x.size(0), (int)N, (int)group,
                                    (float)eps, (int)out_type, dtype_code(x), stream()), "vig_add_rmsnorm_8bit_fwd");
    return {q, scales, r.defined() ? r : x_};
}

std::pair<Tensor, Tensor> norm_forward(const Tensor& x_, const Tensor& w, const Tensor& res0, double eps) {
    const Tensor x = as_rows(x_), res = res0.defined() ? as_rows(res0) : res0;
    const Tensor y = fresh(x_.sizes(), x);
    Tensor r;
    if (res.defined()) r = fresh(x_.sizes(), x);
    ok(api.vig_add_rmsnorm_train_fwd(ptr(x), ld(x), ptr(res), ld(res), ptr(w), dtype_code(w), ptr(y), ptr(r), x.size(0), (int)x.size(1), (float)eps, dtype_code(x), stream()),
       "vig_add_rmsnorm_train_fwd");
    return {y, r};
}

std::pair<Tensor, Tensor> norm_backward(const Tensor& dy_, const Tensor& x_, const Tensor& res_, const Tensor& w, const Tensor& dr_, double eps) {
    const Tensor x = as_rows(x_), dy = as_rows(dy_), dr = dr_.defined() ? as_rows(dr_) : dr_, res = res_.defined() ? as_rows(res_) : res_;
    const Tensor dx = fresh(x_.sizes(), x), dw = fresh(w.sizes(), w);
    const size_t n = api.vig_add_rmsnorm_bwd_workspace_bytes(x.size(0), (int)x.size(1));
    Tensor ws;
    if (n) ws = fresh({(int64_t)n}, x, at::kByte);
    ok(api.vig_add_rmsnorm_bwd(ptr(dy), ld(dy), ptr(x), ld(x), ptr(res), ld(res), ptr(w), dtype_code(w), ptr(dr), ld(dr), ptr(dx), ptr(dw), x.size(0), (int)x.size(1),
                               (float)eps, dtype_code(x), ptr(ws), n, stream()), "vig_add_rmsnorm_bwd");
    return {dx, dw};
}

struct Norm : torch::autograd::Function<Norm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptT& res, double eps) {
        at::AutoDispatchBelowADInplaceOrView guard;
        const auto [y, r] = norm_forward(x, w, get(res), eps);
        // fp32: the sum, which is what it was; 16 bits: what was added, because the sum was rounded
        if (r.defined() && r.scalar_type() != at::kFloat) ctx->save_for_backward({x, w, *res});
        else ctx->save_for_backward({r.defined() ? r : x, w, Tensor()});
        ctx->saved_data["eps"] = eps;
        variable_list out{y};
        if (r.defined()) out.push_back(r);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list d) {
        const auto saved = ctx->get_saved_variables();
        once(d, saved);
        const Tensor x = saved[0], w = saved[1], res = saved[2];
        c10::cuda::CUDAGuard dev(x.device());
        const Tensor dy = d[0].defined() ? d[0] : at::zeros(x.sizes(), x.options());
        const auto [dx, dw] = norm_backward(dy, x, res, w, d.size() > 1 ? d[1] : Tensor(), ctx->saved_data["eps"].toDouble());
        return {dx, dw, d.size() > 1 ? dx : Tensor(), Tensor()};
    }
};

std::pair<Tensor, Tensor> add_rmsnorm_train(const Tensor& x, const Tensor& w, const OptT& res_, double eps) {
    const Tensor res = get(res_);
    check_norm(x, w, res);
    want(eps >= 0, "eps must not be negative");
    no_tangents({&x, &w, &res});
    c10::cuda::CUDAGuard dev(x.device());
    if (wants_grad({&x, &w, &res})) {
        const auto out = Norm::apply(x, w, res_, eps);
        return {out[0], res.defined() ? out[1] : x};
    }
    const auto [y, r] = norm_forward(x, w, res, eps);
    return {y, r.defined() ? r : x};
}

std::pair<Tensor, Tensor> add_rmsnorm_backward(const Tensor& dy, const Tensor& r, const Tensor& w, double eps, const OptT& dr_, const OptT& res_) {
    const Tensor dr = get(dr_), res = get(res_);
    check_norm(r, w, dy);
    check_norm(r, w, dr);
    check_norm(r, w, res);
    want(eps >= 0, "eps must not be negative");
    no_tangents({&dy, &r, &w, &dr, &res});
    c10::cuda::CUDAGuard dev(r.device());
    return norm_backward(dy, r, res, w, dr, eps);
}

// ---- AdamW ----
// a list or tuple of tensors (None entries where allowed), looked at in place
struct Tensors {
    py::object fast;
    Py_ssize_t n = 0;
    Tensors(const py::object& seq, const char* name) {
        if (seq.is_none()) return;
        fast = py::reinterpret_steal<py::object>(PySequence_Fast(seq.ptr(), name));
        if (!fast) throw py::error_already_set();
        n = PySequence_Fast_GET_SIZE(fast.ptr());
    }
    const Tensor* at(Py_ssize_t i, const char* name, bool optional = false) const {
        if (!fast) return nullptr;
        PyObject* o = PySequence_Fast_GET_ITEM(fast.ptr(), i);
        if (optional && o == Py_None) return nullptr;
        want_type(THPVariable_Check(o), std::string(name) + " must hold tensors");
        return &THPVariable_Unpack(o);
    }
};

// whether the values of `t` lie in memory as those of `p` do
bool same_layout(const Tensor& t, const Tensor& p) {
    if (t.sizes() != p.sizes()) return false;
    if (t.strides() == p.strides()) return true;
    for (int64_t i = 0; i < p.dim(); ++i) if (p.size(i) > 1 && t.stride(i) != p.stride(i)) return false;
    return true;
}

void adamw_step(const py::object& params, const py::object& grads, const py::object& exp_avgs, const py::object& exp_avg_sqs, int64_t step, double lr, double beta1,
                double beta2, double eps, double weight_decay, const py::object& masters, const py::object& avg_scales, const py::object& sq_scales,
                const OptT& grad_scale, const OptT& found_inf) {
    const Tensors P(params, "params must be a list of tensors"), G(grads, "grads must be a list of tensors"), M(exp_avgs, "exp_avgs must be a list of tensors"),
        V(exp_avg_sqs, "exp_avg_sqs must be a list of tensors"), W(masters, "masters must be a list"), MS(avg_scales, "exp_avg_scales must be a list"),
        VS(sq_scales, "exp_avg_sq_scales must be a list");
    const Py_ssize_t n = P.n;
    want(step >= 1, "step counts from 1");
    want(lr >= 0 && std::isfinite(lr), "lr must be a number that is not negative");
    want(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "betas must be in [0, 1)");
    want(eps >= 0 && weight_decay >= 0, "eps and weight_decay must not be negative");
    for (const Tensors* t : {&G, &M, &V}) want(t->fast && t->n == n, "params, grads, exp_avgs and exp_avg_sqs must have one entry for each parameter");
    for (const Tensors* t : {&W, &MS, &VS}) want(!t->fast || t->n == n, "masters and scales must have one entry for each parameter");
    if (!n) return;
    std::vector<void*> p(n), m(n), v(n);
    std::vector<const void*> g(n);
    std::vector<float*> w(n), ms(n), vs(n);
    std::vector<int64_t> num(n);
    std::vector<int> pt(n), gt(n);
    std::vector<Tensor> keep;                                  // gradients in the layout of their parameters
    std::vector<const Tensor*> written;
    written.reserve(6 * n);
    const Tensor& first = *P.at(0, "params");
    on_gpu(first);
    c10::cuda::CUDAGuard dev(first.device());
    const auto device = first.device();
    for (Py_ssize_t i = 0; i < n; ++i) {
        const Tensor &pi = *P.at(i, "params"), &mi = *M.at(i, "exp_avgs"), &vi = *V.at(i, "exp_avg_sqs"), *gi = G.at(i, "grads");
        const Tensor *wi = W.at(i, "masters", true), *msi = MS.at(i, "exp_avg_scales", true), *vsi = VS.at(i, "exp_avg_sq_scales", true);
        for (const Tensor* t : {&pi, gi, &mi, &vi, wi, msi, vsi}) {
            if (!t) continue;
            on_gpu(*t);
            want(t->device() == device, "all tensors of a step must be on one device");
            want(t->layout() == at::kStrided, "sparse tensors are not supported");
        }
        pt[i] = code(pi); gt[i] = code(*gi);
        want(pi.is_non_overlapping_and_dense(), "a parameter must fill its memory without gaps or overlaps");
        want((msi != nullptr) == (vsi != nullptr), "a tensor has both scales or none");
        const auto st = msi ? at::kFloat8_e4m3fn : at::kFloat;
        want_type(mi.scalar_type() == st && vi.scalar_type() == st, "states are float32, or float8_e4m3fn with their scales");
        want(same_layout(mi, pi) && same_layout(vi, pi), "states must have their parameter's shape and strides");
        if (wi) {
            want_type(wi->scalar_type() == at::kFloat, "masters are float32");
            want(same_layout(*wi, pi), "a master must have its parameter's shape and strides");
        }
        num[i] = pi.numel();
        for (const Tensor* t : {msi, vsi}) if (t) {
            want_type(t->scalar_type() == at::kFloat, "scales are float32");
            want(t->is_contiguous() && t->numel() == (num[i] + 255) / 256, "scales have one value for every 256 values begun");
        }
        want(gi->sizes() == pi.sizes(), "a gradient must have its parameter's shape");
        if (!same_layout(*gi, pi)) {
            keep.push_back(at::empty_strided(pi.sizes(), pi.strides(), gi->options()));
            keep.back().copy_(gi->detach());
            g[i] = keep.back().data_ptr();
        } else {
            g[i] = gi->data_ptr();
        }
        p[i] = pi.data_ptr(); m[i] = mi.data_ptr(); v[i] = vi.data_ptr();
        w[i] = wi ? wi->data_ptr<float>() : nullptr;
        ms[i] = msi ? msi->data_ptr<float>() : nullptr;
        vs[i] = vsi ? vsi->data_ptr<float>() : nullptr;
        for (const Tensor* t : {&pi, &mi, &vi, wi, msi, vsi}) if (t) written.push_back(t);
    }
    for (const auto* t : {&grad_scale, &found_inf}) if (*t) {
        same_device(**t, first, "grad_scale / found_inf");
        want((*t)->scalar_type() == at::kFloat && (*t)->numel() == 1, "grad_scale and found_inf are float32 tensors of one value");
    }
    for (const Tensor* t : written) t->unsafeGetTensorImpl()->bump_version();     // what is derived from a parameter goes by its version
    ok(api.vig_adamw_step((int)n, p.data(), g.data(), m.data(), v.data(), w.data(), ms.data(), vs.data(), num.data(), pt.data(), gt.data(), step, lr, beta1, beta2, eps,
                          weight_decay, (const float*)ptr(get(grad_scale)), (const float*)ptr(get(found_inf)), stream()), "vig_adamw_step");
}

}  // namespace

void bind_train(py::module_& m) {
    m.def("gated_recurrence", &gated_recurrence);
    m.def("gated_recurrence_step", &gated_recurrence_step);
    m.def("add_rmsnorm_8bit", &add_rmsnorm_8bit);
    m.def("add_rmsnorm_train", &add_rmsnorm_train);
    m.def("add_rmsnorm_backward", &add_rmsnorm_backward);
    m.def("adamw_step", &adamw_step);
}

}  // namespace vig_host
