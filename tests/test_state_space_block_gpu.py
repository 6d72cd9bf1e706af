"""The block on the selective scan: all of its operators together, against the same block written with torch in 64 bits; trained, read in and served."""
import pytest
import torch
import torch.nn.functional as F

import vig_b200

pytestmark = pytest.mark.gpu


def plain(block, x, residual=None):
    """[B, L, d_model] in 64 bits on the CPU"""
    p = {k: v.detach().double().cpu() for k, v in block.named_parameters()}
    x = x.double().cpu()
    r = x if residual is None else x + residual.double().cpu()
    y = F.layer_norm(r, (block.d_model,), p["norm.weight"], p["norm.bias"], block.norm.eps)
    u, z = (y @ p["in_proj.weight"].t()).chunk(2, -1)
    K, L = block.d_conv, x.shape[1]
    padded = F.pad(u, (0, 0, K - 1, 0))
    u = F.silu(sum(p["conv_weight"][:, k] * padded[:, k:k + L] for k in range(K)) + p["conv_bias"])
    t, B, C = (u @ p["x_proj.weight"].t()).split([block.dt_rank, block.d_state, block.d_state], -1)
    delta = F.softplus(t @ p["dt_proj.weight"].t() + p["dt_bias"])
    A, h, out = -torch.exp(p["A_log"]), torch.zeros(x.shape[0], block.d_inner, block.d_state).double(), []
    for i in range(L):
        h = torch.exp(delta[:, i, :, None] * A) * h + (delta[:, i] * u[:, i])[..., None] * B[:, i, None]
        out.append((h * C[:, i, None]).sum(-1) + p["D"] * u[:, i])
    return (torch.stack(out, 1) * F.silu(z)) @ p["out_proj.weight"].t(), r


def far(a, b):
    return float((a.detach().double().cpu() - b).norm() / b.norm())


@pytest.mark.parametrize("dtype,limit", [(torch.float32, 1e-5), (torch.bfloat16, 3e-2)])
def test_forward(dtype, limit):
    """fp32: products of width up to 192 in fp32, sums of 192 u.  bf16: five roundings of 2^-8 in a row (norm, two projections, convolution, gate) and those of the weights stay
    below eight of them."""
    torch.manual_seed(0)
    block = vig_b200.SelectiveStateSpace(96).cuda().to(dtype)
    x, r = torch.randn(2, 130, 96, device="cuda").to(dtype), torch.randn(2, 130, 96, device="cuda").to(dtype)
    for residual in (None, r):
        y, out_r, state = block(x, residual)
        ref, ref_r = plain(block, x, residual)
        assert state is None and far(y, ref) < limit and far(out_r, ref_r) < limit


def test_gradients_against_differences():
    torch.manual_seed(1)
    block = vig_b200.SelectiveStateSpace(16, d_state=5, d_conv=3).cuda()
    x = torch.randn(2, 12, 16, device="cuda", requires_grad=True)
    w = torch.randn(2, 12, 16, device="cuda")
    y, r, _ = block(x)
    grads = dict(zip([n for n, _ in block.named_parameters()], torch.autograd.grad((y * w).sum() + (r * w).sum(), [*block.parameters(), x])))
    loss = lambda: float((plain(block, x.detach())[0] * w.double().cpu()).sum())  # noqa: E731
    gen = torch.Generator().manual_seed(0)
    for name, p in block.named_parameters():
        at = tuple(int(torch.randint(0, n, (), generator=gen)) for n in p.shape)
        with torch.no_grad():
            was = p[at].clone()
            p[at] = was + 2 ** -10
            up = loss()
            p[at] = was - 2 ** -10
            diff = (up - loss()) * 2 ** 9
            p[at] = was
        # second-order differences: 2^-20 of a third derivative of order one to ten
        assert abs(float(grads[name][at]) - diff) <= 1e-3 * (1 + abs(diff)), name


@pytest.mark.parametrize("dtype,limit", [(torch.float32, 1e-5), (torch.bfloat16, 3e-2)])
def test_prefix_then_steps(dtype, limit):
    """A ragged batch of prompts is read in and continued token by token: what the whole sequences give."""
    torch.manual_seed(2)
    block = vig_b200.SelectiveStateSpace(64).cuda().to(dtype)
    x = torch.randn(3, 80, 64, device="cuda").to(dtype)
    n = torch.tensor([70, 1, 33], device="cuda")
    with torch.no_grad():
        whole, whole_r, _ = block(x)
        prompt = torch.where(torch.arange(80, device="cuda")[:, None] < n[:, None, None], x, torch.full_like(x, 7.0))
        y, _, state = block(prompt, output_final_state=True, lengths=n)
        for b in range(3):
            assert far(y[b, :n[b]], whole[b, :n[b]].double().cpu()) < limit
        for i in range(5):
            tokens = x[torch.arange(3, device="cuda"), n + i]
            out, r = block.step(tokens, None, state)
            ref = whole[torch.arange(3, device="cuda"), n + i]
            assert far(out, ref.double().cpu()) < limit and torch.equal(r, tokens)
        state = block.empty_state(3)
        outs = [block.step(x[:, i], None, state)[0] for i in range(80)]
    assert far(torch.stack(outs, 1), whole.double().cpu()) < limit


def test_trains_with_adamw_and_autocast():
    torch.manual_seed(3)
    block = vig_b200.SelectiveStateSpace(64).cuda()
    opt = vig_b200.AdamW(block.parameters(), lr=1e-3)
    x = torch.randn(4, 100, 64, device="cuda")
    before = [p.detach().clone() for p in block.parameters()]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y, r, _ = block(x)
        y, r, _ = block(y, r)
    assert y.dtype == torch.bfloat16 and r.dtype == torch.float32
    (y.float() + r).square().mean().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in block.parameters())
    opt.step()
    assert all(not torch.equal(a, p) for a, p in zip(before, block.parameters()))
    vig_b200.check_status()


def test_recurrence_in_whole_numbers():
    """GatedRecurrence serves with int8 products as near to its 16-bit ones as with e4m3 ones (codes of 127 steps against 3 bits of mantissa)."""
    torch.manual_seed(4)
    block = vig_b200.GatedRecurrence(64).cuda().bfloat16()
    x, zero = torch.randn(8, 64, device="cuda").bfloat16(), torch.zeros(8, 64, device="cuda")
    plain16, _ = block.step(x, None, zero.clone())
    off = {}
    for dtype in (torch.float8_e4m3fn, torch.int8):
        assert block.quantize(dtype) is block and block._codes()[0].dtype == dtype
        off[dtype] = far(block.step(x, None, zero.clone())[0], plain16.double().cpu())
    assert off[torch.int8] < off[torch.float8_e4m3fn] < 0.2
    with torch.no_grad():
        block.in_proj.weight.mul_(2)
    assert torch.equal(block._codes()[0], block.quantize(torch.int8)._codes()[0])
    with pytest.raises(TypeError):
        block.quantize(torch.float16)


def test_many_streams():
    """Two blocks' calls on two streams at once, with their backward passes: the same bits as alone."""
    torch.manual_seed(5)
    blocks = [vig_b200.SelectiveStateSpace(64).cuda().bfloat16() for _ in range(2)]
    xs = [torch.randn(4, 300, 64, device="cuda").bfloat16() for _ in range(2)]

    def run(block, x):
        y, _, _ = block(x)
        return torch.autograd.grad(y.float().square().sum(), list(block.parameters()))

    alone = [run(b, x) for b, x in zip(blocks, xs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        together = []
        for b, x, s in zip(blocks, xs, streams):
            with torch.cuda.stream(s):
                together.append(run(b, x))
        torch.cuda.synchronize()
        for a, t in zip(alone, together):
            assert all(torch.equal(p, q) for p, q in zip(a, t))
