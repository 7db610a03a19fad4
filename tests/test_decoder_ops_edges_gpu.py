"""Calls of the decoder operators at the edge of what their documentation allows, on the GPU."""
import pytest
import torch

from llm_training_amd import ops
from test_attention_mod_gpu import MODS
from test_attention_mod_gpu import run as attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("added", [False, True])
@pytest.mark.parametrize("roles", ["w1=w2", "w1=gate", "w2=gate", "all"])
def test_norm_add_norm_one_parameter_in_two_roles(roles, added):
    """One parameter as two or three of the weights, with a gradient buffer: the buffer gets the sum of the roles'
    gradients. fp32 throughout: sums of 40 products of three factors and means over 64 columns, each off by a few units
    of the terms' magnitudes; 2^-16 of the sum of their sizes holds 2^8 roundings."""
    torch.manual_seed(4)
    T, H = 40, 64
    x, res, dh, ds = (torch.randn(T, H, device=DEV) for _ in range(4))
    w, v = (torch.rand(H, device=DEV).add_(0.5).requires_grad_(True) for _ in range(2))
    pick = {"w1=w2": (w, w, v), "w1=gate": (w, v, w), "w2=gate": (v, w, w), "all": (w, w, w)}[roles]
    d = {id(t): t.detach().double().requires_grad_(True) for t in (w, v)}

    def norm(t, m):
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-5) * m

    s = res.double() + norm(x.double(), d[id(pick[0])]) * d[id(pick[2])]
    want = torch.autograd.grad((norm(s, d[id(pick[1])]), s), d[id(w)], (dh.double(), ds.double()))[0]
    # size of what is summed: d (dres) and dh stay below 4 (|dh| + |ds|) for these inputs, the normalised rows below |n|
    size = 16 * (dh.abs() + ds.abs()).double().sum(0) * 4
    w.main_grad, w.grad_added = torch.full((H,), 3.0, device=DEV), added
    y = ops.norm_add_norm(x.requires_grad_(True), res, pick[0], pick[1], 1e-5, gate=pick[2])
    torch.autograd.backward(y, (dh, ds))
    want = want + (3.0 if added else 0.0)
    assert ((w.main_grad.double() - want).abs() <= 2.0 ** -16 * size).all()
    assert w.grad_added and w.grad is None


@pytest.mark.parametrize("mod", list(MODS))
@pytest.mark.parametrize("scale", [-0.125, 0.0])
@pytest.mark.parametrize("kw", [dict(), dict(ndocs=3), dict(window=40)])
def test_modified_scores_with_a_scale_of_zero_or_below(mod, scale, kw):
    """Masked scores stay masked whatever the sign that a product of -inf would take."""
    got = attention(2, 200, 4, 2, 64, scale=scale, **kw, **MODS[mod])
    assert all(t.isfinite().all() for t in got)
