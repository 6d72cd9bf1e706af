"""The trainable layer norm without a residual: what comes back through ``r`` is added to the norm's share of dx before that is rounded, as ``add_layernorm_backward`` does it."""
import pytest
import torch

import vig_b200
from test_layernorm_rows_gpu import EPS, check, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N", [(1, 1), (40, 96), (75, 333), (9, 4096), (3, 16392)])
def test_one_rounding(M, N, dtype):
    t, d_y, d_r = make(M, N, dtype, seed=M, residual=False)
    g = {k: None if v is None else v.cuda().requires_grad_(True) for k, v in t.items()}
    y, r = vig_b200.add_layernorm_train(g["x"], g["weight"], g["bias"], eps=EPS)
    dx, dw, db = torch.autograd.grad([y, r], [g["x"], g["weight"], g["bias"]], [d_y.cuda(), d_r.cuda()])
    with torch.no_grad():
        plain = vig_b200.add_layernorm_backward(d_y.cuda(), g["x"], g["weight"], EPS, d_r.cuda())
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), plain))
    # the bound of a call whose residual is zeros knows one rounding
    check(dx, reference(dict(t, residual=torch.zeros_like(t["x"])), d_y, d_r)[2], "dx")


def test_the_sum_is_the_input():
    """Its values, in its memory; in a chain of norms, through one result or the other, and where x wants no gradient."""
    t, d_y, d_r = make(20, 64, torch.bfloat16, seed=0, residual=False)
    x, w, b, d_y, d_r = (v.cuda() for v in (t["x"], t["weight"], t["bias"], d_y, d_r))
    w.requires_grad_(True)
    y, r = vig_b200.add_layernorm_train(x, w, b)
    assert r is x and not r.requires_grad
    torch.autograd.grad(y, w, d_y)
    with torch.no_grad():
        assert vig_b200.add_layernorm_train(x, w, b)[1] is x
    leaf = x.clone().requires_grad_(True)
    y, r = vig_b200.add_layernorm_train(leaf, w, b)
    assert torch.equal(r, x) and r.data_ptr() == leaf.data_ptr() and r.requires_grad
    only_r, = torch.autograd.grad(r, leaf, d_r, retain_graph=True)
    only_y, = torch.autograd.grad(y, leaf, d_y, retain_graph=True)
    assert torch.equal(only_r, d_r) and torch.equal(only_y, vig_b200.add_layernorm_backward(d_y, x, w.detach(), 1e-5)[0])
    # the next norm's residual is r: its gradient comes back through both
    y2, r2 = vig_b200.add_layernorm_train(y, w, b, r)
    both, = torch.autograd.grad([y2, r2], leaf, [d_y, d_r])
    with torch.no_grad():
        d_sum = vig_b200.add_layernorm_backward(d_y, y, w, 1e-5, d_r, r)[0]
        want = vig_b200.add_layernorm_backward(d_sum, x, w, 1e-5, d_sum)[0]
    assert torch.equal(both, want)
    leaf.grad = None
    (vig_b200.add_layernorm_train(leaf, w, b)[1].float().sum()).backward()
    assert torch.equal(leaf.grad, torch.ones_like(leaf))
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(vig_b200.add_layernorm_train(leaf, w, b)[1].sum(), leaf, create_graph=True)
