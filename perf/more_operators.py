"""Operators of blocks with a selective state space, as measurable cases: the scan over states (whole sequences, one token, forward with all
gradients), the short causal convolution in front of it (the same three), layer norm behind a residual add (forward with all gradients), and the
product of 8-bit integers that takes the rows of a quantizing norm.

``listed()`` names fixed cases, ``draw(rng)`` gives further ones of the same ranges; ``prepare`` makes what a program has in hand before
the call, ``run`` is one call: in its plain form of elementary torch operations, or, where ``own`` is true, through this package's entry
points.  ``exact`` is the definition in 64 bits, ``work`` the bytes and operations of a call."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EXACT_SUM = 1024                               # so many products of two 8-bit integers add up to less than 2^24, which fp32 holds exactly


def _scan(name, kind, B, L, D, N, dtype, G=1, z=True, state=False, ragged=False):
    return dict(name=name, kind=kind, B=B, L=L, D=D, N=N, G=G, dtype=dtype, z=z, state=state, ragged=ragged)


def _conv(name, kind, B, L, D, K, dtype, silu=True, state=False, ragged=False):
    return dict(name=name, kind=kind, B=B, L=L, D=D, K=K, dtype=dtype, silu=silu, state=state, ragged=ragged)


def _norm(name, M, N, dtype, residual=True):
    return dict(name=name, kind="norm_train", M=M, N=N, dtype=dtype, residual=residual)


def _int8(name, M, N, K, dtype, bias=False):
    return dict(name=name, kind="int8", M=M, N=N, K=K, dtype=dtype, bias=bias)


def listed():
    return [
        # ---- scan over states ----
        # one new token of a few streams that are being served: latency
        _scan("scan_step_b8_768", "scan_step", 8, 1, 768, 16, "bf16"),
        # two photos of other aspect ratios, padded to 14 x 14 patches, in full precision
        _scan("scan_196_f32", "scan", 2, 196, 384, 16, "f32", ragged=True),
        # one high-resolution image (128 x 128 patches) read in before a stream is continued: a long axis, few channels
        _scan("scan_16384_b1", "scan", 1, 16384, 768, 16, "bf16", state=True),
        # training on sequences of 64 x 64 patches
        _scan("scan_train_4096_b8", "scan_train", 8, 4096, 768, 16, "bf16"),
        # an odd length, two groups of channels with maps of their own, a small state
        _scan("scan_train_1021_f16", "scan_train", 3, 1021, 390, 8, "f16", G=2, z=False, state=True),
        # ---- short causal convolution ----
        # the prompt of the long image above
        _conv("conv_16384_b1", "conv", 1, 16384, 768, 4, "bf16", state=True),
        # one new token of a few streams
        _conv("conv_step_b8_768", "conv_step", 8, 1, 768, 4, "bf16"),
        # training on sequences of 64 x 64 patches
        _conv("conv_train_4096_b16", "conv_train", 16, 4096, 768, 4, "bf16"),
        # ---- layer norm behind a residual add ----
        # the first stage of the hierarchical model, 64 images of 56 x 56 patches
        _norm("norm_train_200704x96", 200704, 96, "bf16"),
        # its last stage in full precision, 32 images of 7 x 7 patches
        _norm("norm_train_1568x768_f32", 1568, 768, "f32", residual=False),
        # ---- product of 8-bit integers ----
        # the stacked projection of the widest block for a few streams, one token each: latency
        _int8("int8_8x2304x768", 8, 2304, 768, "bf16"),
        # the same for 16 sequences of 64 x 64 patches
        _int8("int8_65536x2304x768", 65536, 2304, 768, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["scan_step", "scan", "scan", "scan_train", "scan_train", "conv_step", "conv", "conv_train", "norm_train", "int8", "int8"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind.startswith("scan"):
        N, G = rng.choice([16, 16, 8, _log_int(rng, 1, 64)]), rng.choice([1, 1, 1, 2])
        D = G * rng.choice([_log_int(rng, 16, 512), 64 * rng.randint(1, 12)])
        L = 1 if kind == "scan_step" else _log_int(rng, 2, 16384)
        most = 8 * 4096 * 768 * 16 // (1 if kind == "scan_train" else 2) // (2 if dtype == "f32" else 1)
        B = _log_int(rng, 1, max(1, min(512 if L == 1 else 64, most // (L * D * N))))
        if B * L * D * N > most:
            L = max(2, most // (B * D * N))
        c = _scan("", kind, B, L, D, N, dtype, G, rng.random() < 0.6, L > 1 and rng.random() < 0.5, L > 1 and rng.random() < 0.3)
    elif kind.startswith("conv"):
        D, K = rng.choice([_log_int(rng, 16, 1024), 64 * rng.randint(1, 16)]), rng.choice([4, 4, 3, 2, rng.randint(1, 8)])
        L = 1 if kind == "conv_step" else _log_int(rng, 2, 16384)
        most = 16 * 4096 * 768 // (1 if kind == "conv_train" else 2) // (2 if dtype == "f32" else 1)
        B = _log_int(rng, 1, max(1, min(512 if L == 1 else 128, most // (L * D))))
        c = _conv("", kind, B, L, D, K, dtype, rng.random() < 0.7, L > 1 and rng.random() < 0.5, L > 1 and rng.random() < 0.3)
    elif kind == "norm_train":
        N = rng.choice([96, 192, 384, 768, _log_int(rng, 16, 4096)])
        most = 200704 * 96 // (2 if dtype == "f32" else 1)
        c = _norm("", _log_int(rng, 1, most // N), N, dtype, rng.random() < 0.7)
    else:
        N, K = rng.choice([192, 576, 1152, 2304, _log_int(rng, 16, 2304)]), rng.choice([192, 384, 768, _log_int(rng, 16, 4096)])
        most = 65536 * 2304 * 768 // (N * max(K, 512))
        c = _int8("", _log_int(rng, 1, min(65536, most)), N, K, dtype, rng.random() < 0.5)
    del c["name"]
    return c


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    s = dict(case=case)
    if case.get("ragged"):
        s["lengths"] = torch.randint(0, case["L"] + 1, (case["B"],), generator=gen, device="cuda", dtype=torch.int32)
    if kind.startswith("scan"):
        B, L, D, N = (case[n] for n in "BLDN")
        lead = (B,) if kind == "scan_step" else (B, L)
        maps = (*lead, N) if case["G"] == 1 else (*lead, case["G"], N)
        s["u"], s["dt"], s["B"], s["C"] = rand(*lead, D).to(dtype), (0.5 * rand(*lead, D)).to(dtype), rand(*maps).to(dtype), rand(*maps).to(dtype)
        s["z"] = rand(*lead, D).to(dtype) if case["z"] else None
        # rates 1 to N, steps between a thousandth and a tenth: how such a layer begins
        s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32).repeat(D, 1) * (1 + 0.1 * rand(D, N))
        step = torch.exp(torch.rand(D, generator=gen, device="cuda") * math.log(100) + math.log(1e-3))
        s["dt_bias"], s["D"] = torch.log(torch.expm1(step)), 1 + 0.1 * rand(D)
        s["state"] = rand(B, D, N) if case["state"] or kind == "scan_step" else None
        if kind == "scan_train":
            s["d_y"] = rand(*lead, D).to(dtype)
            s["d_final"] = rand(B, D, N) if case["state"] else None
            s["inputs"] = [s[n].requires_grad_(True) for n in ("u", "dt", "A", "B", "C", "D", "z", "dt_bias", "state") if s[n] is not None]
    elif kind.startswith("conv"):
        B, L, D, K = (case[n] for n in "BLDK")
        s["x"] = rand(*((B, D) if kind == "conv_step" else (B, L, D))).to(dtype)
        s["w"], s["bias"] = (rand(D, K) / math.sqrt(K)).to(dtype), (0.1 * rand(D)).to(dtype)
        s["state"] = rand(B, K - 1, D).to(dtype) if case["state"] or kind == "conv_step" else None
        if kind == "conv_train":
            s["d_y"] = rand(B, L, D).to(dtype)
            s["d_final"] = rand(B, K - 1, D).to(dtype) if case["state"] else None
            s["inputs"] = [s[n].requires_grad_(True) for n in ("x", "w", "bias", "state") if s[n] is not None]
    elif kind == "norm_train":
        M, N = case["M"], case["N"]
        s["x"] = (rand(M, N) + 0.5).to(dtype)
        s["residual"] = (2 * rand(M, N)).to(dtype) if case["residual"] else None
        s["w"], s["bias"] = (1 + 0.1 * rand(N)).to(dtype), (0.1 * rand(N)).to(dtype)
        s["d_y"], s["d_r"] = rand(M, N).to(dtype), rand(M, N).to(dtype)
        s["inputs"] = [s[n].requires_grad_(True) for n in ("x", "w", "bias", "residual") if s[n] is not None]
    else:
        M, N, K = (case[n] for n in "MNK")
        codes = lambda rows: (40 * rand(rows, K)).round().clamp(-127, 127).to(torch.int8)  # noqa: E731
        s["q"], s["w"] = codes(M), codes(N)
        s["q_scale"], s["w_scale"] = 0.02 + 0.01 * rand(M, 1).abs(), (0.5 + rand(N).abs()) / 127 / math.sqrt(K)
        s["bias"] = rand(N).to(dtype) if case["bias"] else None
    return s


# ---------------------------------------------------------------------------------------------------------------------
def _valid(s, L):
    """[B, L, 1]: whether a token lies within its sequence."""
    return (torch.arange(L, device="cuda") < s["lengths"][:, None])[..., None] if "lengths" in s else None


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _running(a, x, dim):
    """h_t = a_t h_{t-1} + x_t along dim 1 by doubling: after each step a row holds the sum over twice as many rows up to it."""
    reach = 1
    while reach < x.shape[dim]:
        x = torch.cat([x[:, :reach], x[:, reach:] + a[:, reach:] * x[:, :-reach]], dim)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], dim)
        reach *= 2
    return x


def _spread(maps, D):
    """[B, L, (G,) N] -> [B, L, D, N]: each channel with the values of its group."""
    maps = maps.float()
    return maps[:, :, None] if maps.dim() == 3 else maps.repeat_interleave(D // maps.shape[2], 2)


def _gather(x, maps):
    """The sum over the channels of each group, laid out like the maps."""
    return x.sum(2) if maps.dim() == 3 else x.unflatten(2, (maps.shape[2], -1)).sum(3)


def _plain_scan(s):
    case, dtype = s["case"], s["u"].dtype
    one = case["kind"] == "scan_step"
    wide = lambda n: None if s[n] is None else s[n][:, None] if one else s[n]  # noqa: E731
    u, x, Bm, Cm, z = wide("u").float(), wide("dt").float() + s["dt_bias"], wide("B"), wide("C"), wide("z")
    D = u.shape[2]
    delta = torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))
    mask = None if one else _valid(s, u.shape[1])
    if mask is not None:
        delta = delta * mask
    Bs, Cs = _spread(Bm, D), _spread(Cm, D)
    a = torch.exp(delta[..., None] * s["A"])
    h0 = s["state"] if s["state"] is not None else torch.zeros(u.shape[0], D, s["A"].shape[1], device="cuda")
    b = (delta * u)[..., None] * Bs
    b[:, 0] += a[:, 0] * h0
    h = _running(a, b, 1)
    y = (h * Cs).sum(-1) + s["D"] * u
    gate = z.float() * _sigmoid(z.float()) if z is not None else torch.ones_like(y)
    out = y * gate
    if mask is not None:
        out = out * mask
    out, final = out.to(dtype), h[:, -1].clone()
    if one:
        s["state"].copy_(final)
        return out[:, 0], s["state"]
    if case["kind"] == "scan":
        return out, final if case["state"] else None
    d_out = s["d_y"].float()
    if mask is not None:
        d_out = d_out * mask
    d_y = d_out * gate
    g = d_y[..., None] * Cs
    if s["d_final"] is not None:
        g[:, -1] += s["d_final"]
    # g_t = C_t d_y_t + a_{t+1} g_{t+1}: the same scan from the other end
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _running(later.flip(1), g.flip(1), 1).flip(1)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    through = g * a * before
    from_b = (g * Bs).sum(-1)
    d_delta = (through * s["A"]).sum(-1) + from_b * u
    d_x = d_delta * _sigmoid(x)
    if mask is not None:
        d_x = d_x * mask
    grads = [(from_b * delta + s["D"] * d_y).to(dtype), d_x.to(dtype), (through * delta[..., None]).sum((0, 1)),
             _gather(g * (delta * u)[..., None], Bm).to(dtype), _gather(h * d_y[..., None], Cm).to(dtype), (d_y * u).sum((0, 1))]
    if z is not None:
        p = _sigmoid(z.float())
        grads.append((d_out * y * p * (1 + z.float() * (1 - p))).to(dtype))
    grads.append(d_x.sum((0, 1)))
    if s["state"] is not None:
        grads.append(a[:, 0] * g[:, 0])
    return (out, *([final] if case["state"] else []), *grads)


def _plain_conv(s):
    case, dtype, K = s["case"], s["x"].dtype, s["case"]["K"]
    one = case["kind"] == "conv_step"
    x = s["x"][:, None] if one else s["x"]
    L, w = x.shape[1], s["w"].float()
    mask = None if one else _valid(s, L)
    x = x.float() if mask is None else x.float() * mask
    front = s["state"].float() if s["state"] is not None else torch.zeros(x.shape[0], K - 1, x.shape[2], device="cuda")
    whole = torch.cat([front, x], 1)
    # [B, L, D, K]: the window behind each token
    window = whole.unfold(1, K, 1)
    pre = (window * w).sum(-1) + s["bias"].float()
    out = pre * _sigmoid(pre) if case["silu"] else pre
    if mask is not None:
        out = out * mask
    ends = s["lengths"].long() if mask is not None else torch.full((x.shape[0],), L, device="cuda")
    rows = ends[:, None] + torch.arange(K - 1, device="cuda")
    final = whole.gather(1, rows[..., None].expand(-1, -1, x.shape[2])).to(dtype)
    if one:
        s["state"].copy_(final)
        return out[:, 0].to(dtype), s["state"]
    if case["kind"] == "conv":
        return out.to(dtype), final if case["state"] else None
    d = s["d_y"].float()
    if case["silu"]:
        p = _sigmoid(pre)
        d = d * p * (1 + pre * (1 - p))
    if mask is not None:
        d = d * mask
    # the window in front of each token, weights from the other end
    none = torch.zeros(x.shape[0], K - 1, x.shape[2], device="cuda")
    d_whole = (torch.cat([none, d, none], 1).unfold(1, K, 1) * w.flip(1)).sum(-1)
    if s["d_final"] is not None:
        d_whole = d_whole.scatter_add(1, rows[..., None].expand(-1, -1, x.shape[2]), s["d_final"].float())
    d_x = d_whole[:, K - 1:]
    if mask is not None:
        d_x = d_x * mask
    grads = [d_x.to(dtype), (window * d[..., None]).sum((0, 1)).to(dtype), d.sum((0, 1)).to(dtype)]
    if s["state"] is not None:
        grads.append(d_whole[:, :K - 1].to(dtype))
    return (out.to(dtype), *([final] if case["state"] else []), *grads)


def _plain_norm(s):
    dtype = s["x"].dtype
    r = s["x"].float() + s["residual"].float() if s["residual"] is not None else s["x"].float()
    w = s["w"].float()
    far = r - r.mean(-1, keepdim=True)
    rstd = torch.rsqrt((far * far).mean(-1, keepdim=True) + 1e-5)
    xh = far * rstd
    t = s["d_y"].float() * w
    d = (rstd * (t - t.mean(-1, keepdim=True) - xh * (t * xh).mean(-1, keepdim=True)) + s["d_r"].float()).to(dtype)
    return ((xh * w + s["bias"].float()).to(dtype), r.to(dtype), d, (s["d_y"].float() * xh).sum(0).to(dtype), s["d_y"].float().sum(0).to(dtype),
            *([d] if s["residual"] is not None else []))


def _plain_int8(s):
    q, w = s["q"].float(), s["w"].float()
    total = sum((q[:, k:k + EXACT_SUM] @ w[:, k:k + EXACT_SUM].t()).double() for k in range(0, q.shape[1], EXACT_SUM))
    y = total * s["q_scale"] * s["w_scale"]
    return (y + s["bias"].double() if s["bias"] is not None else y).to(DTYPES[s["case"]["dtype"]])


def _plain(s):
    kind = s["case"]["kind"]
    if kind.startswith("scan"):
        return _plain_scan(s)
    if kind.startswith("conv"):
        return _plain_conv(s)
    return _plain_norm(s) if kind == "norm_train" else _plain_int8(s)


def _ours(s):
    import vig_b200
    case = s["case"]
    kind = case["kind"]
    if kind == "scan_step":
        return vig_b200.selective_scan_step(s["u"], s["dt"], s["A"], s["B"], s["C"], s["state"], s["D"], s["z"], s["dt_bias"]), s["state"]
    if kind == "conv_step":
        return vig_b200.causal_conv_step(s["x"], s["state"], s["w"], s["bias"], activation="silu" if case["silu"] else None), s["state"]
    if kind == "int8":
        return vig_b200.linear_int8(s["q"], s["q_scale"], s["w"], s["w_scale"], s["bias"], dtype=DTYPES[case["dtype"]])
    if kind == "norm_train":
        outs = vig_b200.add_layernorm_train(s["x"], s["w"], s["bias"], s["residual"], eps=1e-5)
        return (*(t.detach() for t in outs), *torch.autograd.grad(outs, s["inputs"], [s["d_y"], s["d_r"]]))
    if kind.startswith("scan"):
        y, final = vig_b200.selective_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"], s["state"], case["state"],
                                           lengths=s.get("lengths"))
    else:
        y, final = vig_b200.causal_conv(s["x"], s["w"], s["bias"], s["state"], case["state"], activation="silu" if case["silu"] else None,
                                        lengths=s.get("lengths"))
    if not kind.endswith("_train"):
        return y, final
    outs, ds = ([y, final], [s["d_y"], s["d_final"]]) if case["state"] else ([y], [s["d_y"]])
    return (*(t.detach() for t in outs), *torch.autograd.grad(outs, s["inputs"], ds))


def run(state):
    if own:
        if state["case"]["kind"].endswith("_train"):
            return _ours(state)
        with torch.no_grad():
            return _ours(state)
    with torch.no_grad():
        return _plain(state)


# ---------------------------------------------------------------------------------------------------------------------
def _exact_scan(case, s, wide):
    """Token by token, and back."""
    B, L, D, N = (case[n] for n in "BLDN")
    u, x = wide["u"].view(B, L, D), wide["dt"].view(B, L, D) + wide["dt_bias"]
    pick = torch.arange(D, device="cuda") // (D // case["G"])
    Bs, Cs = (wide[n].view(B, L, case["G"], N) for n in "BC")
    A, skip, z = wide["A"], wide["D"], wide["z"].view(B, L, D) if case["z"] else None
    inside = (torch.arange(L, device="cuda") < s["lengths"][:, None]).double()[..., None] if case["ragged"] else torch.ones(B, L, 1, device="cuda").double()
    delta = torch.nn.functional.softplus(x, threshold=60.0) * inside
    train = case["kind"] == "scan_train"
    h = wide["state"] if s["state"] is not None else torch.zeros(B, D, N, device="cuda", dtype=torch.float64)
    ys, kept = torch.empty_like(u), []
    for t in range(L):
        if train:
            kept.append(h)
        h = torch.exp(delta[:, t, :, None] * A) * h + (delta[:, t] * u[:, t])[..., None] * Bs[:, t][:, pick]
        ys[:, t] = torch.einsum("bdn,bdn->bd", h, Cs[:, t][:, pick]) + skip * u[:, t]
    gate = torch.nn.functional.silu(z) if z is not None else 1.0
    out = ys * gate * inside
    if case["kind"] == "scan_step":
        return out[:, 0], h
    if not train:
        return out, h if case["state"] else None
    final = h
    d_out = wide["d_y"] * inside
    d_ys = d_out * gate
    g = wide["d_final"] if case["state"] else torch.zeros_like(final)
    d_u, d_x, dA = torch.empty_like(u), torch.empty_like(x), torch.zeros_like(A)
    dB, dC = torch.zeros_like(Bs), torch.zeros_like(Cs)
    for t in range(L - 1, -1, -1):
        a, before = torch.exp(delta[:, t, :, None] * A), kept.pop()
        b = (delta[:, t] * u[:, t])[..., None]
        now = a * before + b * Bs[:, t][:, pick]
        g = g + d_ys[:, t, :, None] * Cs[:, t][:, pick]
        dC[:, t].index_add_(1, pick, now * d_ys[:, t, :, None])
        dB[:, t].index_add_(1, pick, g * b)
        along = (g * Bs[:, t][:, pick]).sum(-1)
        flow = g * a * before
        dA += (flow * delta[:, t, :, None]).sum(0)
        d_x[:, t] = ((flow * A).sum(-1) + along * u[:, t]) * torch.sigmoid(x[:, t]) * inside[:, t]
        d_u[:, t] = along * delta[:, t] + skip * d_ys[:, t]
        g = g * a
    maps = wide["B"].shape
    d_z = [d_out * ys * torch.sigmoid(z) * (1 + z * torch.sigmoid(-z))] if z is not None else []
    return (out, *([final] if case["state"] else []), d_u, d_x, dA, dB.view(maps), dC.view(maps), (d_ys * u).sum((0, 1)), *d_z, d_x.sum((0, 1)),
            *([g] if case["state"] else []))


def _exact_conv(case, s, wide):
    """Tap by tap."""
    B, L, D, K = (case[n] for n in "BLDK")
    inside = (torch.arange(L, device="cuda") < s["lengths"][:, None]).double()[..., None] if case["ragged"] else torch.ones(B, L, 1, device="cuda").double()
    x = torch.zeros(B, K - 1 + L, D, device="cuda", dtype=torch.float64)
    x[:, K - 1:] = wide["x"].view(B, L, D) * inside
    if s["state"] is not None:
        x[:, :K - 1] = wide["state"]
    pre = wide["bias"].expand(B, L, D).clone()
    for k in range(K):
        pre += wide["w"][:, k] * x[:, k:k + L]
    act = torch.nn.functional.silu if case["silu"] else (lambda v: v)
    out = act(pre) * inside
    ends = s["lengths"].tolist() if case["ragged"] else [L] * B
    final = torch.stack([x[b, e:e + K - 1] for b, e in enumerate(ends)])
    if case["kind"] == "conv_step":
        return out[:, 0], final
    if case["kind"] == "conv":
        return out, final if case["state"] else None
    d = wide["d_y"] * inside
    if case["silu"]:
        d = d * torch.sigmoid(pre) * (1 + pre * torch.sigmoid(-pre))
    d_x, d_w = torch.zeros_like(x), torch.empty_like(wide["w"])
    for k in range(K):
        d_x[:, k:k + L] += wide["w"][:, k] * d
        d_w[:, k] = (d * x[:, k:k + L]).sum((0, 1))
    if case["state"]:
        for b, e in enumerate(ends):
            d_x[b, e:e + K - 1] += wide["d_final"][b]
    return (out, *([final] if case["state"] else []), d_x[:, K - 1:] * inside, d_w, d.sum((0, 1)), *([d_x[:, :K - 1]] if case["state"] else []))


def exact(case, seed):
    """The definitions in 64 bits, the scan token by token."""
    s = prepare(case, seed)
    wide = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["kind"].startswith("scan"):
        return _exact_scan(case, s, wide)
    if case["kind"].startswith("conv"):
        return _exact_conv(case, s, wide)
    if case["kind"] == "norm_train":
        r = wide["x"] + wide["residual"] if case["residual"] else wide["x"]
        inv = 1 / (r.var(1, keepdim=True, correction=0) + 1e-5).sqrt()
        far = (r - r.mean(1, keepdim=True)) * inv
        t = wide["d_y"] * wide["w"]
        d = inv * (t - t.mean(1, keepdim=True) - far * (far * t).mean(1, keepdim=True)) + wide["d_r"]
        return (far * wide["w"] + wide["bias"], r, d, (wide["d_y"] * far).sum(0), wide["d_y"].sum(0), *([d] if case["residual"] else []))
    y = wide["q_scale"] * (wide["q"] @ wide["w"].t()) * wide["w_scale"]
    return y + wide["bias"] if case["bias"] else y


def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"].startswith("scan"):
        n, states = case["B"] * case["L"] * case["D"], case["B"] * case["D"] * case["N"]
        maps = 2 * case["B"] * case["L"] * case["G"] * case["N"] * e
        train, through = case["kind"] == "scan_train", 4 if case["z"] else 3
        # forward u, dt, z in, y out, both maps in; training also d_y in and the gradients out; states in and out in 32 bits
        held = (4 if train else 2) * 4 * states if case["state"] or case["kind"] == "scan_step" else 0
        return dict(bytes=n * e * through * (2 if train else 1) + maps * (2 if train else 1) + 4 * case["D"] * case["N"] + held,
                    flops=n * case["N"] * (24 if train else 7))
    if case["kind"].startswith("conv"):
        n = case["B"] * case["L"] * case["D"]
        train = case["kind"] == "conv_train"
        held = case["B"] * (case["K"] - 1) * case["D"] * e * (4 if train else 2) if case["state"] or case["kind"] == "conv_step" else 0
        return dict(bytes=n * e * (4 if train else 2) + held, flops=n * (case["K"] * (6 if train else 2) + 5))
    if case["kind"] == "norm_train":
        n = case["M"] * case["N"]
        # x, residual, d_y, d_r in; y, r and the gradient of the sum out
        return dict(bytes=n * e * (7 if case["residual"] else 5) + 4 * case["N"] * e, flops=20 * n)
    M, N, K = (case[n] for n in "MNK")
    return dict(bytes=M * K + N * K + M * N * e + 4 * (M + N), flops=2 * M * N * K)
