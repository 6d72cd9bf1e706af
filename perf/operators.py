"""Operators that train and serve a block with a gated recurrence, as measurable cases: the recurrence itself (whole sequences, one
token, forward with all gradients), the RMS norm behind a residual add (8-bit rows with scales for serving, forward with all gradients
for training) and the AdamW step over many tensors.

``listed()`` names fixed cases, ``draw(rng)`` gives further ones of the same ranges; ``prepare`` makes what a program has in hand before
the call, ``run`` is one call: in its plain form of elementary torch operations, or, where ``own`` is true, through this package's entry
points.  ``exact`` is the definition in 64 bits, ``work`` the bytes and operations of a call."""
import itertools
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
TOP = {"e4m3": 448.0, "int8": 127.0}          # the largest value of an 8-bit type
BLOCK = 256                                    # elements that share the scales of 8-bit optimizer states
LR, BETA1, BETA2, EPS, DECAY = 2e-4, 0.9, 0.999, 1e-8, 0.05


def _rec(name, kind, B, L, D, dtype, norm=0.0, reverse=False, state=False):
    return dict(name=name, kind=kind, B=B, L=L, D=D, dtype=dtype, norm=norm, reverse=reverse, state=state)


def _norm(name, kind, M, N, dtype, out="", group=0, residual=True):
    return dict(name=name, kind=kind, M=M, N=N, dtype=dtype, out=out, group=group, residual=residual)


def _adamw(name, width, depth, dtype, bits, master=False, odd=0):
    return dict(name=name, kind="adamw", width=width, depth=depth, dtype=dtype, bits=bits, master=master, odd=odd)


def listed():
    return [
        # ---- gated recurrence ----
        # one new token of a few streams that are being served: latency
        _rec("step_b8_768", "step", 8, 1, 768, "bf16", 1.0),
        # a photo's 14 x 14 patches in full precision, log-space gates
        _rec("rec_196_f32", "rec", 2, 196, 192, "f32"),
        # one high-resolution image (128 x 128 patches) read in before a stream is continued: few channels, a long axis
        _rec("rec_16384_b1", "rec", 1, 16384, 768, "bf16", 16.0, state=True),
        # training on sequences of 64 x 64 patches
        _rec("rec_train_4096_b16", "rec_train", 16, 4096, 768, "bf16", 16.0),
        # an odd length and width, scanned from the end
        _rec("rec_train_1021_f16", "rec_train", 3, 1021, 193, "f16", 0.0, reverse=True),
        # ---- RMS norm behind a residual add ----
        # one token in front of an 8-bit product: latency
        _norm("norm8_1x768", "norm8", 1, 768, "bf16", "e4m3"),
        # eight images of 2048 x 2048 through a block of the widest model
        _norm("norm8_131072x768", "norm8", 131072, 768, "bf16", "e4m3"),
        # a few photos of another aspect ratio, scales for every 128 channels
        _norm("norm8_2508x384_g128", "norm8", 2508, 384, "f16", "e4m3", 128),
        # training on 64 images of 1024 x 1024, the narrowest model
        _norm("norm_train_262144x192", "norm_train", 262144, 192, "bf16"),
        # ---- AdamW ----
        # two blocks of the narrowest model in full precision, as a small fine-tuning job updates them
        _adamw("adamw_192x2_f32", 192, 2, "f32", 32),
        # all blocks of the middle model in full precision
        _adamw("adamw_384x12_f32", 384, 12, "f32", 32),
        # all blocks of the widest model: 16-bit weights with a full-precision copy, states in 8 bits
        _adamw("adamw_768x12_bf16_s8", 768, 12, "bf16", 8, master=True),
    ]


def _log_int(rng, lo, hi):
    n = max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))
    return n + 1 if n == 3 << 10 else n


def draw(rng):
    kind = rng.choice(["step", "rec", "rec_train", "norm8", "norm8", "norm_train", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "step":
        c = _rec("", kind, _log_int(rng, 1, 1024), 1, _log_int(rng, 64, 4096), dtype, rng.choice([0.0, 1.0, 16.0]))
    elif kind in ("rec", "rec_train"):
        L = _log_int(rng, 2, 16384)
        D = rng.choice([_log_int(rng, 32, 1024), 64 * rng.randint(1, 16)])
        most = (16 if kind == "rec_train" else 32) * 4096 * 768 // (2 if dtype == "f32" else 1)
        B = _log_int(rng, 1, max(1, min(256, most // (L * D))))
        c = _rec("", kind, B, L, D, dtype, rng.choice([0.0, 1.0, 16.0]), rng.random() < 0.3, rng.random() < 0.5)
    elif kind in ("norm8", "norm_train"):
        N = rng.choice([192, 384, 768, _log_int(rng, 32, 8192)])
        out, group = "", 0
        if kind == "norm8":
            out = rng.choice(["e4m3", "e4m3", "int8"])
            group = rng.choice([0, 0, 32, 64, 128])
            N = N if not group else max(group, N // group * group)
        most = 131072 * 768 // (2 if dtype == "f32" else 1) // (1 if kind == "norm8" else 2)
        c = _norm("", kind, _log_int(rng, 1, most // N), N, dtype, out, group, rng.random() < 0.8)
    else:
        bits = rng.choice([32, 8])
        width = rng.choice([96, 192, 384, 768])
        c = _adamw("", width, rng.randint(1, 6 if width == 768 else 12), dtype, bits, dtype != "f32" and rng.random() < 0.6, rng.randint(0, 999))
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------------
def _shapes(case):
    """Shapes of the tensors of ``depth`` blocks with a gated-linear-attention mixer and a gated MLP, and of an odd-sized head."""
    C, inter = case["width"], 256 * ((case["width"] * 8 // 3 + 255) // 256)
    block = [(C,), (C, 1, 3, 3), (2 * C, C), (16, C), (C, 16), (C,), (C, C), (64,), (64,), (C, C), (C,), (C,), (2 * inter, C), (C, inter)]
    return block * case["depth"] + ([(case["odd"], 7)] if case["odd"] else [])


def _to8(x):
    """8-bit codes and scales of blocks of 256 elements."""
    rows = x.view(-1, BLOCK)
    scale = rows.abs().amax(1) / TOP["e4m3"]
    return (rows / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]).to(torch.float8_e4m3fn).view(-1), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    dtype = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["kind"] in ("step", "rec", "rec_train"):
        shape = (case["B"], case["D"]) if case["kind"] == "step" else (case["B"], case["L"], case["D"])
        # raw gate logits of order one, or log-gates of a sigmoid of them
        z = rand(*shape) if case["norm"] else torch.nn.functional.logsigmoid(rand(*shape) + 1)
        s["x"], s["g"] = rand(*shape).to(dtype), z.to(dtype)
        s["state"] = rand(case["B"], case["D"]) if case["state"] or case["kind"] == "step" else None
        if case["kind"] == "rec_train":
            s["d_h"] = rand(*shape).to(dtype)
            s["d_final"] = rand(case["B"], case["D"]) if case["state"] else None
            s["inputs"] = [t.requires_grad_(True) for t in (s["x"], s["g"], s["state"]) if t is not None]
    elif case["kind"] in ("norm8", "norm_train"):
        M, N = case["M"], case["N"]
        s["x"] = rand(M, N).to(dtype)
        s["residual"] = (2 * rand(M, N)).to(dtype) if case["residual"] else None
        s["w"] = (1 + 0.1 * rand(N)).to(dtype)
        if case["kind"] == "norm_train":
            s["d_y"], s["d_r"] = rand(M, N).to(dtype), rand(M, N).to(dtype)
            s["inputs"] = [t.requires_grad_(True) for t in (s["x"], s["w"], s["residual"]) if t is not None]
    else:
        # every kind of tensor in one buffer, as a training program lays its parameters out; a tensor begins on a block of its own
        shapes = _shapes(case)
        sizes = [math.prod(shape) for shape in shapes]
        room = [-(-n // BLOCK) * BLOCK for n in sizes]
        *starts, total = itertools.accumulate(room, initial=0)
        used = torch.cat([torch.arange(r, device="cuda") < n for n, r in zip(sizes, room)])
        full = 0.05 * rand(total) * used
        s["p"] = full.to(dtype)
        s["master"] = full.clone() if case["master"] else None
        s["g"] = (1e-3 * rand(total) * used).to(dtype)
        m, root_v = 3e-4 * rand(total) * used, 1e-3 * (0.2 + rand(total).abs()) * used
        s["m"], s["m_scale"] = _to8(m) if case["bits"] == 8 else (m, None)
        s["v"], s["v_scale"] = _to8(root_v) if case["bits"] == 8 else (root_v * root_v, None)
        s["step"] = 1000 + seed % 1000

        for name in ("p", "master", "g", "m", "v"):
            s[name + "_list"] = None if s[name] is None else [s[name][a:a + n].view(shape) for a, n, shape in zip(starts, sizes, shapes)]
        for name in ("m_scale", "v_scale"):
            s[name + "_list"] = None if s[name] is None else [s[name][a // BLOCK:-(-(a + n) // BLOCK)] for a, n in zip(starts, sizes)]
    return s


# ---------------------------------------------------------------------------------------------------------------------
def _decay(g, norm):
    """exp of the log-gates, in 32 bits"""
    g = g.float()
    return torch.exp((torch.minimum(g, torch.zeros_like(g)) - torch.log1p(torch.exp(-g.abs()))) / norm) if norm else torch.exp(g)


def _scan(a, x):
    """h_t = a_t h_{t-1} + x_t along dim 1 by doubling: after each step a row holds the sum over twice as many rows up to it."""
    reach = 1
    while reach < x.shape[1]:
        x = torch.cat([x[:, :reach], x[:, reach:] + a[:, reach:] * x[:, :-reach]], 1)
        a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    return x


def _plain_rec(s):
    case = s["case"]
    turn = (lambda t: t.flip(1)) if case["reverse"] else (lambda t: t)
    x, g = turn(s["x"].float()), turn(s["g"].float())
    a = _decay(g, case["norm"])
    h0 = s["state"] if s["state"] is not None else torch.zeros_like(x[:, 0])
    h = _scan(a, torch.cat([x[:, :1] + a[:, :1] * h0[:, None], x[:, 1:]], 1))
    final = h[:, -1].clone()
    if case["kind"] == "rec":
        return turn(h).to(s["x"].dtype), final if case["state"] else None
    d_h = turn(s["d_h"].float())
    if s["d_final"] is not None:
        d_h = torch.cat([d_h[:, :-1], d_h[:, -1:] + s["d_final"][:, None]], 1)
    # d_x_t = d_h_t + a_{t+1} d_x_{t+1}: the same scan from the other end
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    d_x = _scan(later.flip(1), d_h.flip(1)).flip(1)
    d_g = d_x * a * torch.cat([h0[:, None], h[:, :-1]], 1)
    if case["norm"]:
        d_g = d_g / (1 + torch.exp(g)) / case["norm"]
    grads = [turn(d_x).to(s["x"].dtype), turn(d_g).to(s["x"].dtype)]
    return (turn(h).to(s["x"].dtype), *([final] if case["state"] else []), *grads, *([a[:, 0] * d_x[:, 0]] if case["state"] else []))


def _plain_norm(s):
    case, dtype = s["case"], s["x"].dtype
    r = s["x"].float() + s["residual"].float() if s["residual"] is not None else s["x"].float()
    w = s["w"].float()
    rstd = torch.rsqrt((r * r).mean(-1, keepdim=True) + 1e-6)
    y = r * rstd * w
    if case["kind"] == "norm8":
        rows = y.view(case["M"], -1, case["group"] or case["N"])
        scale = rows.abs().amax(-1) / TOP[case["out"]]
        q = rows / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
        q = q.to(torch.float8_e4m3fn) if case["out"] == "e4m3" else torch.round(q).to(torch.float16)
        return q.view(case["M"], case["N"]), scale, r.to(dtype)
    xh = r * rstd
    t = s["d_y"].float() * w
    d = (rstd * (t - xh * (t * xh).mean(-1, keepdim=True)) + s["d_r"].float()).to(dtype)
    d_w = (s["d_y"].float() * xh).sum(0).to(dtype)
    return (y.to(dtype), r.to(dtype), d, d_w, *([d] if s["residual"] is not None else []))


def _plain_adamw(s):
    g = s["g"].float()
    eight = s["case"]["bits"] == 8
    m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1) if eight else s["m"]
    v = (s["v"].float().view(-1, BLOCK) * s["v_scale"][:, None]).view(-1).square() if eight else s["v"]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * (g * g)
    p = s["master"] if s["master"] is not None else s["p"].float()
    step = s["step"]
    p = p * (1 - LR * DECAY) - LR / (1 - BETA1 ** step) * m / (torch.sqrt(v) / math.sqrt(1 - BETA2 ** step) + EPS)
    s["p"].copy_(p)
    if s["master"] is not None:
        s["master"].copy_(p)
    if eight:
        for name, x in (("m", m), ("v", torch.sqrt(v))):
            code, scale = _to8(x)
            if name == "v":         # a root that is not zero keeps a code that is not
                code = torch.where((x > 0) & (code.float() == 0), torch.full_like(x, 2.0 ** -9), code.float()).to(torch.float8_e4m3fn)
            s[name].copy_(code)
            s[name + "_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)


def _adamw_outputs(s):
    return [s[name] for name in ("p", "master", "m", "v", "m_scale", "v_scale") if s[name] is not None]


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "step":
        s["state"].copy_(_decay(s["g"], s["case"]["norm"]) * s["state"] + s["x"].float())
        return s["state"].to(s["x"].dtype), s["state"]
    if kind in ("rec", "rec_train"):
        return _plain_rec(s)
    if kind in ("norm8", "norm_train"):
        return _plain_norm(s)
    _plain_adamw(s)
    return _adamw_outputs(s)


def _ours(s):
    import vig_b200
    case = s["case"]
    if case["kind"] == "step":
        return vig_b200.gated_recurrence_step(s["x"], s["g"], s["state"], gate_logit_normalizer=case["norm"]), s["state"]
    if case["kind"] in ("rec", "rec_train"):
        h, final = vig_b200.gated_recurrence(s["x"], s["g"], s["state"], case["state"], reverse=case["reverse"], gate_logit_normalizer=case["norm"])
        if case["kind"] == "rec":
            return h, final
        outs, ds = ([h, final], [s["d_h"], s["d_final"]]) if case["state"] else ([h], [s["d_h"]])
        return (*(t.detach() for t in outs), *torch.autograd.grad(outs, s["inputs"], ds))
    if case["kind"] == "norm8":
        out = torch.float8_e4m3fn if case["out"] == "e4m3" else torch.int8
        q, scale, r = vig_b200.add_rmsnorm_8bit(s["x"], s["w"], s["residual"], eps=1e-6, dtype=out, group=case["group"] or None, prenorm=True)
        return q if out != torch.int8 else q.to(torch.float16), scale.view(case["M"], -1), r
    if case["kind"] == "norm_train":
        y, r = vig_b200.add_rmsnorm_train(s["x"], s["w"], s["residual"], eps=1e-6)
        return (y.detach(), r.detach(), *torch.autograd.grad([y, r], s["inputs"], [s["d_y"], s["d_r"]]))
    vig_b200.adamw_step(s["p_list"], s["g_list"], s["m_list"], s["v_list"], s["step"], LR, (BETA1, BETA2), EPS, DECAY, masters=s["master_list"],
                        exp_avg_scales=s["m_scale_list"], exp_avg_sq_scales=s["v_scale_list"])
    return _adamw_outputs(s)


def run(state):
    if own:
        if state["case"]["kind"] in ("rec_train", "norm_train"):
            return _ours(state)
        with torch.no_grad():
            return _ours(state)
    with torch.no_grad():
        return _plain(state)


# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    """The definitions in 64 bits, the recurrences token by token."""
    s = prepare(case, seed)
    wide = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["kind"] in ("step", "rec", "rec_train"):
        x, g = (wide[n].view(case["B"], case["L"], case["D"]) for n in ("x", "g"))
        a = torch.sigmoid(g).pow(1 / case["norm"]) if case["norm"] else g.exp()
        order = list(range(case["L"]))[::-1 if case["reverse"] else 1]
        state = wide.get("state", torch.zeros_like(x[:, 0]))
        h, before = torch.empty_like(x), torch.empty_like(x)
        for t in order:
            before[:, t] = state
            state = a[:, t] * state + x[:, t]
            h[:, t] = state
        if case["kind"] == "step":
            return h[:, 0], state
        if case["kind"] == "rec":
            return h, state if case["state"] else None
        u, d_x, d_g = wide.get("d_final", torch.zeros_like(state)), torch.empty_like(x), torch.empty_like(x)
        for t in order[::-1]:
            d_x[:, t] = wide["d_h"][:, t] + u
            u = a[:, t] * d_x[:, t]
            d_g[:, t] = u * before[:, t]
        if case["norm"]:
            d_g *= torch.sigmoid(-g) / case["norm"]
        return (h, *([state] if case["state"] else []), d_x, d_g, *([u] if case["state"] else []))
    if case["kind"] in ("norm8", "norm_train"):
        r = wide["x"] + wide["residual"] if case["residual"] else wide["x"]
        inv = 1 / (r.square().mean(1, keepdim=True) + 1e-6).sqrt()
        y = wide["w"] * r * inv
        if case["kind"] == "norm8":
            width = case["group"] or case["N"]
            scale = y.abs().unflatten(1, (-1, width)).amax(2) / TOP[case["out"]]
            return y / scale.repeat_interleave(width, 1), scale, r
        t = wide["d_y"] * wide["w"]
        d = inv * t - inv.pow(3) * r * (t * r).mean(1, keepdim=True) + wide["d_r"]
        return (y, r, d, (wide["d_y"] * r * inv).sum(0), *([d] if case["residual"] else []))
    eight = case["bits"] == 8
    per = (lambda name: wide[name + "_scale"].repeat_interleave(BLOCK)) if eight else (lambda name: 1.0)
    g, m = wide["g"], wide["m"] * per("m")
    v = (wide["v"] * per("v")) ** 2 if eight else wide["v"]
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g ** 2 - v)
    p = wide["master"] if case["master"] else wide["p"]
    p = p - LR * (DECAY * p + (m / (1 - BETA1 ** s["step"])) / ((v / (1 - BETA2 ** s["step"])) ** 0.5 + EPS))
    outs = [p] + ([p] if case["master"] else [])
    if not eight:
        return [*outs, m, v]
    v = v ** 0.5
    tops = [t.view(-1, BLOCK).abs().amax(1) / TOP["e4m3"] for t in (m, v)]
    codes = [t / c.clamp_min(1e-300).repeat_interleave(BLOCK) for t, c in zip((m, v), tops)]
    return [*outs, *codes, *tops]


def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "step":
        n = case["B"] * case["D"]
        return dict(bytes=n * (3 * e + 8), flops=4 * n)
    if case["kind"] in ("rec", "rec_train"):
        n, rows = case["B"] * case["L"] * case["D"], case["B"] * case["D"]
        train = case["kind"] == "rec_train"
        # forward x, g in, h out; training also d_h in, d_x and d_g out; states in and out in 32 bits
        return dict(bytes=n * e * (6 if train else 3) + (rows * 4 * (4 if train else 2) if case["state"] else 0), flops=n * (10 if train else 4))
    if case["kind"] == "norm8":
        n = case["M"] * case["N"]
        return dict(bytes=n * ((3 if case["residual"] else 1) * e + 1) + 4 * n // (case["group"] or case["N"]) + case["N"] * e, flops=8 * n)
    if case["kind"] == "norm_train":
        n = case["M"] * case["N"]
        # x, residual, d_y, d_r in; y, r and the gradient of the sum out
        return dict(bytes=n * e * (7 if case["residual"] else 5) + 2 * case["N"] * e, flops=18 * n)
    n = sum(math.prod(shape) for shape in _shapes(case))
    states = 4 + 16 / BLOCK if case["bits"] == 8 else 16
    return dict(bytes=n * (e * (2 if case["master"] else 3) + (8 if case["master"] else 0) + states), flops=16 * n)
