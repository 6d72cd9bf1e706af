"""Every form of the recurrence's kernels against 64 bits, forward and all gradients: strips of 8, 16 and 32 lanes with one CTA and in clusters, over
several steps with a ragged last one, rows off 16 bytes, few tokens by single channels and by several.

Tolerances as in test_gated_recurrence_gpu.py (4 u of the sum of magnitudes a token; a decay that is off by E of itself adds E a S), but a raw logit's decay
is off by a part of its logarithm (7 terms of a polynomial: 2^-19 of it; 9 terms: 8 u) and 8 u for the exponential, and gate gradients are taken at
states in fp32: no rounding of h to 16 bits is allowed for."""
import pytest
import torch

import vig_b200
from test_gated_recurrence_gpu import TINY, U, UNIT, decay, scan

pytestmark = pytest.mark.gpu


def decay_error(g, norm, dtype):
    if not norm:
        return 8 * U + 2 * U * g.abs().clamp_max(200)
    return 8 * U + (8 * U if dtype == torch.float32 else 2.0 ** -19) * torch.nn.functional.logsigmoid(g).abs().clamp_max(200 * norm) / norm


def make(B, L, D, dtype, norm, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, z, d_h = (rand(B, L, D) for _ in range(3))
    g = 2 * z if norm else -0.3 * torch.rand(B, L, D, generator=gen, device="cuda")
    return x.to(dtype), g.to(dtype), d_h.to(dtype), rand(B, D), rand(B, D)


def truth(x, g, d_h, h0, d_f, norm, reverse, dtype, rounded=0.0):
    """(value, bound) of h, final, dx, dg, d(h0); ``rounded``: what h is off by, of itself, where the gate gradient is taken at it"""
    turn = (lambda t: t.flip(1)) if reverse else (lambda t: t)
    xd, gd, dd = (turn(t.double()) for t in (x, g, d_h))
    a, ea = decay(gd, norm), decay_error(gd, norm, dtype)
    before, h, eh, final, ef = scan(a, xd, h0.double(), ea=ea)
    # u_t = a_t (dh_t + u_{t+1}), dx_t = dh_t + u_{t+1}: carried as d_x_t = dh_t + a_{t+1} d_x_{t+1}
    later, elater = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1), torch.cat([ea[:, 1:], torch.zeros_like(a[:, :1])], 1)
    _, dx, edx, _, _ = scan(later.flip(1), dd.flip(1), d_f.double(), ea=elater.flip(1))
    dx, edx = dx.flip(1), edx.flip(1)
    u, eu = a * dx, a * edx + (ea + 2 * U) * a * dx.abs()
    ebefore = torch.cat([torch.zeros_like(eh[:, :1]), eh[:, :-1] + rounded * (h[:, :-1].abs() + eh[:, :-1])], 1)
    dg = u * before
    edg = eu * before.abs() + u.abs() * ebefore + eu * ebefore + 4 * U * dg.abs()
    if norm:
        s = torch.sigmoid(-gd) / norm
        dg, edg = dg * s, edg * s + dg.abs() * s * (16 * U + 4 * ea)      # 1 - sigmoid comes from the same logarithm
    return (turn(h), turn(eh)), (final, ef), (turn(dx), turn(edx)), (turn(dg), turn(edg)), (u[:, 0], eu[:, 0])


def check(got, ref, dtype, name):
    value, bound = ref
    off = (got.double() - value).abs()
    most = bound + UNIT[dtype] * (value.abs() + bound) + TINY[dtype]
    assert torch.isfinite(got).all(), name
    assert (off <= most).all(), f"{name}: worst {float((off / most).max()):.2f} of the bound"


def check_all(B, L, D, dtype, norm, reverse, slices=None):
    x, g, d_h, h0, d_f = make(B, L, D, dtype, norm, seed=B + L + D)
    leaf = [t.clone().requires_grad_(True) for t in (x, g, h0)]
    h, final = vig_b200.gated_recurrence(*leaf, True, reverse=reverse, gate_logit_normalizer=norm)
    got = (h.detach(), final.detach(), *torch.autograd.grad([h, final], leaf, [d_h, d_f]))
    for s in slices or [slice(None)]:
        ref = truth(*(t[s] for t in (x, g, d_h, h0, d_f)), norm, reverse, dtype)
        for name, r, i in (("h", ref[0], 0), ("final", ref[1], 1), ("dx", ref[2], 2), ("dg", ref[3], 3), ("dh0", ref[4], 4)):
            check(got[i][s], r, torch.float32 if i in (1, 4) else dtype, name)
    # a third of a unit more than its own rounding is already too much for the gate gradient as a whole
    if dtype != torch.float32:
        value, _ = truth(x[:1], g[:1], d_h[:1], h0[:1], d_f[:1], norm, reverse, dtype)[3]
        near = value.to(dtype).double()
        assert float((got[3][:1].double() - value).norm()) <= 1.1 * float((near - value).norm())


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


# (sequences at 148 SMs, tokens, channels, type, lanes of a strip forward and backward; 0: not the form of whole 16-byte pieces)
FORMS = [
    (60, 210, 384, torch.bfloat16, 32, 32),          # one CTA each
    (24, 300, 1024, torch.float16, 32, 32),
    (48, 300, 1000, torch.bfloat16, 32, 16),         # backward in halves
    (16, 301, 768, torch.bfloat16, 16, 16),          # strips of 16 lanes, one CTA, several steps
    (24, 300, 768, torch.float16, 16, 16),
    (17, 300, 1024, torch.bfloat16, 16, 16),
    (12, 300, 768, torch.float32, 16, 32),           # backward: clusters of two
    (8, 701, 384, torch.bfloat16, 32, 32),           # clusters of eight
    (4, 1101, 384, torch.float16, 16, 16),
    (1, 3001, 192, torch.bfloat16, 8, 8),            # clusters of eight or sixteen, several steps
    (30, 201, 768, torch.float32, 32, 16),
    (40, 260, 1024, torch.float32, 32, 32),
    (16, 201, 384, torch.float32, 16, 16),
    (3, 600, 96, torch.float32, 8, 8),
    (50, 300, 193, torch.bfloat16, 0, 0),            # rows off 16 bytes: one CTA, and clusters
    (2, 1500, 97, torch.float16, 0, 0),
    (2, 1500, 97, torch.float32, 0, 0),
    (320, 5, 1024, torch.bfloat16, 0, 0),            # few tokens, several channels a thread
    (330, 17, 1024, torch.float16, 0, 0),
    (330, 45, 512, torch.float32, 0, 0),
    (3, 15, 100, torch.bfloat16, 0, 0),              # ... and one
    (400, 41, 101, torch.float16, 0, 0),
]


@pytest.mark.parametrize("norm,reverse", [(16.0, False), (1.0, True), (0.0, False)])
@pytest.mark.parametrize("B,L,D,dtype,fwd,bwd", FORMS)
def test_forms(B, L, D, dtype, fwd, bwd, norm, reverse):
    B = max(1, B * sms() // 148)
    check_all(B, L, D, dtype, norm, reverse, [slice(0, 3), slice(B - 1, B)])


def test_forms_are_reached(tmp_path):
    """The shapes above take the strips that they are meant to take (three times, the profiler may lose one)."""
    import json
    import re
    for n, (B, L, D, dtype, fwd, bwd) in enumerate(FORMS):
        B = max(1, B * sms() // 148)
        x, g, d_h, _, _ = make(B, L, D, dtype, 16.0, seed=1)
        leaf = [x.requires_grad_(True), g.requires_grad_(True)]
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
            for _ in range(3):
                torch.autograd.grad(vig_b200.gated_recurrence(*leaf, gate_logit_normalizer=16.0)[0], leaf, d_h)
                torch.cuda.synchronize()
        prof.export_chrome_trace(str(tmp_path / f"{n}.json"))
        names = {e["name"] for e in json.load(open(tmp_path / f"{n}.json"))["traceEvents"] if e.get("cat") == "kernel"}
        lanes = {int(m[2]): int(m[3]) for m in (re.search(r"rec_tile_kernel<[^,]*, \(?(?:bool\)?)?(\w+), \(?(?:bool\)?)?(\w+), \(?(?:bool\)?)?\w+, \(?(?:int\)?)?(\d+)>", s.replace("true", "1").replace("false", "0")) for s in names) if m}
        assert lanes == ({0: fwd, 1: bwd} if fwd else {}), (B, L, D, dtype, names)


@pytest.mark.parametrize("L", [1, 2, 7, 8, 9, 15, 16, 17, 24, 25, 31, 33, 63, 64, 65, 72, 73, 127, 128, 129, 137])
@pytest.mark.parametrize("D,dtype", [(8, torch.bfloat16), (40, torch.float16), (33, torch.bfloat16)])
def test_states_at_every_remainder(L, D, dtype):
    """Groups of eight tokens are counted from the end: every length around a group, a thread's tokens and a step, both directions."""
    for reverse in (False, True):
        check_all(2, L, D, dtype, 1.0, reverse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_thirds_of_a_projection(dtype):
    """x and g as column slices of one tensor, and without an initial state: the bits of copies."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    z = torch.randn(3, 200, 3 * 64, generator=gen, device="cuda").to(dtype)
    d = torch.randn(3, 200, 64, generator=gen, device="cuda").to(dtype)
    views = [t.detach().requires_grad_(True) for t in z.chunk(3, -1)[:2]]
    copies = [t.detach().contiguous().requires_grad_(True) for t in z.chunk(3, -1)[:2]]
    assert not views[0].is_contiguous()
    (a, _), (b, _) = (vig_b200.gated_recurrence(*t, gate_logit_normalizer=16.0) for t in (views, copies))
    assert torch.equal(a, b)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(a, views, d), torch.autograd.grad(b, copies, d)))


@pytest.mark.parametrize("B,L,D", [(2, 5, 24), (2, 300, 64), (2, 300, 33), (320, 9, 1024)])
@pytest.mark.parametrize("reverse", [False, True])
def test_c_backward_at_the_rounded_output(B, L, D, reverse):
    """The C entry that takes h in the place of x and states: its gate gradient may be off by h's rounding."""
    from vig_b200 import _lib
    lib, dtype, norm = _lib.lib(), torch.bfloat16, 16.0
    x, g, d_h, h0, d_f = make(B, L, D, dtype, norm, seed=3)
    with torch.no_grad():
        h, _ = vig_b200.gated_recurrence(x, g, h0, reverse=reverse, gate_logit_normalizer=norm)
    dx, dg, d0 = torch.empty_like(x), torch.empty_like(x), torch.empty_like(h0)
    p = _lib.ptr
    assert lib.vig_gated_recurrence_bwd(p(g), p(h), p(h0), p(d_h), p(d_f), p(dx), p(dg), p(d0), B, L, D, None, None, None, norm, int(reverse), 1, None, _lib.stream_ptr()) == 0
    s = slice(0, 2)
    ref = truth(*(t[s] for t in (x, g, d_h, h0, d_f)), norm, reverse, dtype, rounded=UNIT[dtype])
    for name, got, r, t in (("dx", dx, ref[2], dtype), ("dg", dg, ref[3], dtype), ("dh0", d0, ref[4], torch.float32)):
        check(got[s], r, t, name)


def test_states_refusals():
    from vig_b200 import _lib
    lib = _lib.lib()
    assert lib.vig_gated_recurrence_states_bytes(2, 8, 16) == 0 and lib.vig_gated_recurrence_states_bytes(2, 9, 16) == 2 * 16 * 4
    assert lib.vig_gated_recurrence_states_bytes(3, 25, 10) == 3 * 3 * 10 * 4 and lib.vig_gated_recurrence_states_bytes(0, 25, 10) == 0
    x = torch.zeros(1, 20, 8, dtype=torch.bfloat16, device="cuda")
    st = torch.zeros(64, device="cuda")
    p = _lib.ptr
    fwd = lambda states, dtype=1: lib.vig_gated_recurrence_train_fwd(p(x), p(x), None, 0, p(x), None, 0, states, 1, 20, 8, None, None, None, 0.0, 0, dtype, None, _lib.stream_ptr())  # noqa: E731
    bwd = lambda states, dtype=1: lib.vig_gated_recurrence_train_bwd(p(x), p(x), states, None, p(x), None, p(x), p(x), None, 1, 20, 8, None, None, None, 0.0, 0, dtype, None, _lib.stream_ptr())  # noqa: E731
    for call in (fwd, bwd):
        assert call(None) == -1 and call(st.data_ptr() + 4) == -4 and call(st.data_ptr(), 0) == -3


@pytest.mark.parametrize("B,L,D,dtype", [(3, 1, 64, 1), (2, 9, 100, 2), (1, 20000, 96, 1), (2, 5000, 97, 2), (4, 1101, 384, 1), (40, 300, 768, 0), (3, 700, 96, 0)])
@pytest.mark.parametrize("reverse", [0, 1])
def test_c_state_in_place(B, L, D, dtype, reverse):
    """The final state where the initial one was, over one CTA and over clusters of which one writes it: the bits of two buffers."""
    from vig_b200 import _lib
    lib, p = _lib.lib(), _lib.ptr
    t = (torch.float32, torch.bfloat16, torch.float16)[dtype]
    x, g, _, h0, _ = make(B, L, D, t, 1.0, seed=L)
    h, h2, final, state = torch.empty_like(x), torch.empty_like(x), torch.empty_like(h0), h0.clone()
    for out, s0, s1 in ((h, h0, final), (h2, state, state)):
        assert lib.vig_gated_recurrence_fwd(p(x), p(g), p(s0), D, p(out), p(s1), D, B, L, D, None, None, None, 1.0, reverse, dtype, None, _lib.stream_ptr()) == 0
    assert torch.equal(h, h2) and torch.equal(final, state) and not torch.equal(final, h0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm", [1.0, 16.0])
def test_long_memories(norm, dtype):
    """Logits of 7 to 10: states that decay by 1e-4 a token and less.  The logarithm is right to a part in 10^6 of itself, and a decay is rounded to 2^-25
    at random: some 1e-5 of the state over 6000 tokens.  A logarithm right to 2^-22 absolute would be off by 1e-3."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(1, 6000, 64, generator=gen, device="cuda").to(dtype)
    z = (8.5 + 0.5 * torch.randn(1, 6000, 64, generator=gen, device="cuda")).to(dtype)
    _, final = vig_b200.gated_recurrence(x, z, None, True, gate_logit_normalizer=norm)
    a, s = decay(z.double(), norm), torch.zeros(1, 64, dtype=torch.float64, device="cuda")
    for t in range(6000):
        s = a[:, t] * s + x[:, t].double()
    assert float((final.double() - s).norm() / s.norm()) < 1e-4


@pytest.mark.parametrize("D,reverse", [(1024, False), (1001, True)])
def test_gradients_beyond_32_bits(D, reverse):
    """Tensors of more than 2^31 values: gradients at both ends against calls on those ends alone.  4000 tokens forget what is beyond them; both calls then
    round values that agree to 1e-6."""
    L, n = 2_200_000, 3000
    gen = torch.Generator(device="cuda").manual_seed(8)
    x, g, d = (torch.empty(1, L, D, dtype=torch.bfloat16, device="cuda").normal_(generator=gen) for _ in range(3))
    kw = dict(gate_logit_normalizer=1.0, reverse=reverse)

    def grads(part):
        leaf = [t[:, part].detach().requires_grad_(True) for t in (x, g)]
        return torch.autograd.grad(vig_b200.gated_recurrence(*leaf, **kw)[0], leaf, d[:, part])

    whole = grads(slice(None))
    for end, keep in ((slice(0, n + 4000), slice(0, n)), (slice(L - n - 4000, L), slice(4000, n + 4000))):
        for got, want in zip(whole, grads(end)):
            got, want = got[:, end][:, keep].float(), want[:, keep].float()
            assert ((got - want).abs() <= 2 * UNIT[torch.bfloat16] * want.abs() + 1e-5).all()
