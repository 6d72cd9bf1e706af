"""AdamW over lists of tensors against the formula in 64 bits, and the optimizer class over many steps.

Tolerances: with u = 2^-24, m and v are two products and a sum each (4 u of the sum of their magnitudes), the step a root, two products and a
quotient (8 u of itself, and what m and v bring), the parameter one more sum; then the rounding of its type.  8-bit states are compared as the
values they stand for, within half a step of e4m3 (1/16 of the value, 2^-10 of the scale where codes are subnormal; a root that would get the
code 0 gets 2^-9, so up to 2^-9 of the scale)."""
import math

import pytest
import torch

import vig_b200

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
UNIT = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LR, B1, B2, EPS, WD = 3e-3, 0.9, 0.99, 1e-8, 0.1


def codes(x):
    """e4m3 codes and scales of blocks of 256 values in memory order"""
    flat = x.flatten()
    pad = torch.nn.functional.pad(flat, (0, -flat.numel() % 256)).view(-1, 256)
    scale = pad.abs().amax(1) / 448
    code = (pad / torch.where(scale > 0, scale, 1.0)[:, None]).to(torch.float8_e4m3fn).float()
    return code.flatten()[:flat.numel()].view(x.shape).to(torch.float8_e4m3fn), scale


def stood(code, scale):
    return (code.double().flatten() * scale.double().repeat_interleave(256)[:code.numel()]).view(code.shape)


def make(n, dtype, gdtype, eight, master, seed):
    gen = torch.Generator().manual_seed(seed)
    full = torch.randn(n, generator=gen)
    t = dict(p=full.to(dtype), g=(0.1 * torch.randn(n, generator=gen)).to(gdtype), master=full.clone() if master else None)
    m, root = 0.05 * torch.randn(n, generator=gen), 0.1 * torch.rand(n, generator=gen)
    if n > 3:
        root[1], m[2], t["g"][3] = 0, 0, 0
    if eight:
        (t["m"], t["ms"]), (t["v"], t["vs"]) = codes(m), codes(root)
    else:
        t.update(m=m, v=root * root, ms=None, vs=None)
    return t


def expected(t, step, scale=1.0):
    """(p, m, v) in 64 bits with bounds of their error"""
    eight = t["ms"] is not None
    m, v = (stood(t["m"], t["ms"]), stood(t["v"], t["vs"]) ** 2) if eight else (t["m"].double(), t["v"].double())
    g = t["g"].double() * scale
    em, ev = 6 * U * (B1 * m.abs() + (1 - B1) * g.abs()), 8 * U * (B2 * v + (1 - B2) * g * g) + 1e-40
    m, v = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    p = (t["p"] if t["master"] is None else t["master"]).double()
    den = (v / (1 - B2 ** step)).sqrt() + EPS
    rate = LR / (1 - B1 ** step)
    move = rate * m / den
    root = (v + ev).sqrt() - (v - ev).clamp_min(0).sqrt() + 2 * U * v.sqrt()
    emove = rate * em / den + move.abs() * (root / math.sqrt(1 - B2 ** step) / den + 8 * U)
    new = p * (1 - LR * WD) - move
    return new, emove + 4 * U * (p.abs() + move.abs()), m, em, v, ev


def compare(t, dev, step, scale=1.0):
    new, ep, m, em, v, ev = expected(t, step, scale)
    if t["master"] is not None:
        assert ((dev["master"].cpu().double() - new).abs() <= ep + U * new.abs()).all()
    assert ((dev["p"].cpu().double() - new).abs() <= ep + (U + 1.01 * UNIT[t["p"].dtype]) * (new.abs() + ep) + (2.0 ** -24 if t["p"].dtype == torch.float16 else 0)).all()
    if t["ms"] is None:
        assert ((dev["m"].cpu().double() - m).abs() <= em).all() and ((dev["v"].cpu().double() - v).abs() <= ev).all()
        return
    root, er = v.sqrt(), ev / (2 * v.sqrt()).clamp_min(1e-30) + 2 * U * v.sqrt()
    for name, x, e, floor in (("m", m, em, 2.0 ** -10), ("v", root, torch.minimum(er, ev.sqrt()), 2.0 ** -9)):
        scale_ = dev[name + "s"].cpu().double()
        top = torch.nn.functional.pad(x.flatten().abs(), (0, -x.numel() % 256)).view(-1, 256).amax(1)
        assert ((scale_ - top / 448).abs() <= 16 * U * top / 448 + 1e-37).all()
        unit = scale_.repeat_interleave(256)[:x.numel()].view(x.shape)
        got = stood(dev[name].cpu(), dev[name + "s"].cpu())
        assert ((got - x).abs() <= torch.maximum(x.abs() / 16, unit * floor) * 1.001 + 2 * e + 40 * U * unit * 448).all()
        if name == "v":
            assert ((got > 0) == (x > 0)).all()


def put(t):
    return {k: None if v is None else v.cuda() for k, v in t.items()}


def step_all(devs, step, **kw):
    col = lambda name: [d[name] for d in devs]  # noqa: E731
    vig_b200.adamw_step(col("p"), col("g"), col("m"), col("v"), step, LR, (B1, B2), EPS, WD, masters=col("master"), exp_avg_scales=col("ms"), exp_avg_sq_scales=col("vs"), **kw)


@pytest.mark.parametrize("step", [1, 1000])
@pytest.mark.parametrize("eight,master", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("dtype,gdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float32)])
def test_sizes(dtype, gdtype, eight, master, step):
    """One call over tensors of one value to several blocks, whole and ragged."""
    ts = [make(n, dtype, gdtype, eight, master, seed=n) for n in (1, 2, 7, 8, 255, 256, 257, 1000, 2047, 2048, 2049, 5000, 70001)]
    devs = [put(t) for t in ts]
    step_all(devs, step)
    for t, d in zip(ts, devs):
        compare(t, d, step)


def test_mixed_types_states_and_many_tensors():
    """More tensors than a launch holds, of all types in one call, with empty ones among them."""
    combos = [(p, g, e, m) for p, g in ((torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)) for e in (False, True) for m in (False, True)]
    ts = [make(0 if i % 50 == 3 else 1 + (i * 37) % 900, *combos[i % len(combos)], seed=i) for i in range(950)]
    devs = [put(t) for t in ts]
    step_all(devs, 3)
    for t, d in zip(ts, devs):
        if t["p"].numel():
            compare(t, d, 3)


@pytest.mark.parametrize("eight", [False, True])
def test_offsets_and_layouts(eight):
    """Values that begin off 16 bytes, a channels-last filter, a gradient in another layout than its parameter: same numbers as from plain ones."""
    t = make(3001, torch.bfloat16, torch.bfloat16, eight, True, seed=1)
    ref = put(t)
    step_all([ref], 5)
    d = put(t)
    off = {}
    for name in ("p", "g", "m", "v", "master"):
        room = torch.zeros(3010, dtype=d[name].dtype, device="cuda") if d[name].dtype != torch.float8_e4m3fn else torch.zeros(3010, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        off[name] = room[3:3004]
        off[name].copy_(d[name])
    off["ms"], off["vs"] = d["ms"], d["vs"]
    step_all([off], 5)
    for name in ("p", "m", "v", "master"):
        assert torch.equal(off[name].float(), ref[name].float()), name

    t = make(8 * 3 * 9, torch.float32, torch.float32, eight, False, seed=2)
    plain = put(t)
    step_all([plain], 5)
    last = {k: v if v is None or k in ("ms", "vs") else v.view(8, 9, 3).permute(0, 2, 1).view(8, 3, 3, 3) for k, v in put(t).items()}
    last["g"] = last["g"].contiguous()
    assert last["g"].stride() != last["p"].stride()
    step_all([last], 5)
    assert torch.equal(last["p"].view(8, 3, 9).permute(0, 2, 1).flatten(), plain["p"])


def test_gradient_scale_and_found_inf():
    t = make(1000, torch.float16, torch.float16, False, True, seed=3)
    d = put(t)
    step_all([d], 2, grad_scale=torch.tensor([0.125], device="cuda"), found_inf=torch.zeros(1, device="cuda"))
    compare(t, d, 2, scale=0.125)
    kept = {k: None if v is None else v.clone() for k, v in d.items()}
    d["g"][5] = float("inf")
    step_all([d], 3, found_inf=torch.ones(1, device="cuda"))
    for name in ("p", "m", "v", "master"):
        assert torch.equal(d[name], kept[name])


def test_nan_stays_where_it_is():
    for eight in (False, True):
        t = make(1024, torch.float32, torch.float32, eight, False, seed=4)
        clean, bad = put(t), put(t)
        bad["g"][300] = float("nan")
        for d in (clean, bad):
            step_all([d], 2)
        assert torch.isnan(bad["p"][300]) and torch.isnan(bad["m"].float()[300])
        rest = torch.arange(1024, device="cuda") != 300
        assert torch.equal(bad["p"][rest], clean["p"][rest])
        if eight:       # a block's scale is its largest value: the block is lost, and no other
            assert torch.isnan(bad["ms"]).tolist() == [False, True, False, False]
            out = (torch.arange(1024, device="cuda") // 256) != 1
            assert torch.equal(bad["m"].float()[out], clean["m"].float()[out])


def test_versions_of_what_is_written_rise():
    d = put(make(100, torch.float32, torch.float32, True, False, seed=5))
    before = {k: v._version for k, v in d.items() if v is not None}
    step_all([d], 1)
    assert all((d[k]._version > b) == (k != "g") for k, b in before.items())


@pytest.mark.parametrize("kw", [dict(), dict(state_bits=8, min_8bit_size=256), dict(master_weights=True)])
def test_optimizer_class(kw):
    """Thirty steps on a quadratic beside torch's own optimizer: the same path in 32 bits, the same place in 8; and a state that is saved and loaded
    goes on as the one that was not."""
    torch.manual_seed(0)
    dtype = torch.bfloat16 if "master_weights" in kw else torch.float32
    goal = [torch.randn(64, 48, device="cuda"), torch.randn(48, device="cuda")]
    ours = [torch.zeros_like(t, dtype=dtype).requires_grad_(True) for t in goal]
    theirs = [torch.zeros_like(t).requires_grad_(True) for t in goal]
    opt = vig_b200.AdamW([dict(params=ours[:1]), dict(params=ours[1:], weight_decay=0.0)], lr=0.05, weight_decay=0.02, **kw)
    ref = torch.optim.AdamW([dict(params=theirs[:1]), dict(params=theirs[1:], weight_decay=0.0)], lr=0.05, weight_decay=0.02)
    loss = lambda ps: sum(((p.float() - t) ** 2).sum() for p, t in zip(ps, goal))  # noqa: E731

    def go(o, ps):
        o.zero_grad()
        value = loss(ps)
        value.backward()
        o.step()
        return float(value.detach())

    first = go(opt, ours)
    go(ref, theirs)
    for _ in range(29):
        last = go(opt, ours)
        go(ref, theirs)
    assert last < 0.2 * first
    for a, b in zip(ours, theirs):
        # 32 bits: 30 steps of rounding; 16-bit gradients are taken at rounded weights; 8 bits: a step is off by up to 1/8 of itself (m and root
        # by 1/16 each), 30 steps of at most lr
        far = {"": 1e-4, "master_weights": 0.1, "state_bits": 30 * 0.05 / 8}[next((k for k in ("state_bits", "master_weights") if k in kw), "")]
        assert float((a.detach().float() - b.detach()).abs().max()) <= far
    if "state_bits" in kw:
        assert opt.state[ours[0]]["exp_avg"].dtype == torch.float8_e4m3fn and opt.state[ours[1]]["exp_avg"].dtype == torch.float32

    saved = opt.state_dict()
    copy = [p.detach().clone().requires_grad_(True) for p in ours]
    other = vig_b200.AdamW([dict(params=copy[:1]), dict(params=copy[1:], weight_decay=0.0)], lr=0.05, weight_decay=0.02, **kw)
    other.load_state_dict(saved)
    for _ in range(2):
        go(opt, ours)
        go(other, copy)
    assert all(torch.equal(a, b) for a, b in zip(ours, copy))


def test_steps_reach_derived_weights():
    """A layout that a module keeps of its weights goes by their version: it is made again after a step."""
    from vig_b200.modules import GatedLinearAttention
    attn = GatedLinearAttention(d_model=64, num_heads=1, expand_k=1.0, expand_v=1.0).cuda().bfloat16().eval()
    first = attn._pack(True)[1].clone()
    opt = vig_b200.AdamW(attn.parameters(), lr=0.1)
    for p in attn.parameters():
        p.grad = torch.ones_like(p)
    opt.step()
    assert not torch.equal(attn._pack(True)[1], first)


def test_refusals():
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    call = lambda p=None, g=None, m=None, v=None, step=1, **kw: vig_b200.adamw_step(  # noqa: E731
        [f(8)] if p is None else p, [f(8)] if g is None else g, [f(8)] if m is None else m, [f(8)] if v is None else v, step, **kw)
    call()
    vig_b200.adamw_step([], [], [], [], 1)
    eight = torch.zeros(8, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    for bad in (lambda: call(step=0), lambda: call(lr=-1.0), lambda: call(betas=(1.0, 0.9)), lambda: call(eps=-1.0), lambda: call(g=[]), lambda: call(g=[f(9)]),
                lambda: call(m=[f(9)]), lambda: call(masters=[f(8), f(8)]), lambda: call(p=[f(8, 2)[:, 0]]), lambda: call(m=[f(2, 4).t()], p=[f(4, 2)], g=[f(4, 2)], v=[f(4, 2)]),
                lambda: call(exp_avg_scales=[f(1)]), lambda: call(m=[eight], v=[eight], exp_avg_scales=[f(2)], exp_avg_sq_scales=[f(2)]),
                lambda: call(grad_scale=f(2))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: call(p=[f(8).double()]), lambda: call(m=[f(8).half()]), lambda: call(m=[eight], v=[eight]), lambda: call(masters=[f(8).half()]), lambda: call(g=[None]),
                lambda: call(p=5)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError):
        call(g=[torch.zeros(8)])
    with pytest.raises(ValueError):
        vig_b200.AdamW([f(8).requires_grad_(True)], state_bits=4)


def test_offsets_beyond_32_bits():
    """A tensor of more than 2^31 values: its last blocks as a call on them alone gives them, bit for bit."""
    n, k = (1 << 31) + 1000, 256 * 40 + 1000                  # the tail begins on a block
    gen = torch.Generator(device="cuda").manual_seed(8)
    p, g = (torch.empty(n, dtype=torch.bfloat16, device="cuda").normal_(generator=gen) for _ in range(2))
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    scales = [torch.zeros((n + 255) // 256, device="cuda") for _ in range(2)]
    tail = [t[-k:].clone() for t in (p, g, m.view(torch.uint8), v.view(torch.uint8))]
    tail[2], tail[3] = (t.view(torch.float8_e4m3fn) for t in tail[2:])
    small = [torch.zeros((k + 255) // 256, device="cuda") for _ in range(2)]
    for step in (1, 2):
        vig_b200.adamw_step([p], [g], [m], [v], step, exp_avg_scales=scales[:1], exp_avg_sq_scales=scales[1:])
        vig_b200.adamw_step(*[[t] for t in tail], step, exp_avg_scales=small[:1], exp_avg_sq_scales=small[1:])
    assert torch.equal(p[-k:], tail[0])
    assert torch.equal(m[-k:].view(torch.uint8), tail[2].view(torch.uint8)) and torch.equal(v[-k:].view(torch.uint8), tail[3].view(torch.uint8))
    assert torch.equal(scales[0][-len(small[0]):], small[0]) and torch.equal(scales[1][-len(small[1]):], small[1])
