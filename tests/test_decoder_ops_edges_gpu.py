"""Calls of the decoder operators at the edge of what their documentation allows, on the GPU."""
from types import SimpleNamespace

import pytest
import torch

from llm_training_amd import ops
from llm_training_amd.models.hf_causal_lm import hf_attention
from llm_training_amd.ops import fused
from llm_training_amd.ops.embedding import vocab_embedding
from test_attention_mod_gpu import MODS, compare, oracle
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


@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("softcap", [60.0, 50.0, 100.0])
@pytest.mark.parametrize("size", [1e-30, 1e10, 1e30])
def test_capped_scores_at_both_ends_and_values_of_any_size(D, softcap, size):
    """Rows whose scores are saturated at the cap, at its negative, and at both: the probabilities are taken against the
    row's maximum, so neither they nor their products with V leave fp32's range. dO is scaled so that dP stays of the
    order of 1."""
    torch.manual_seed(5)
    S = 700
    end = torch.tensor([1.0, -1.0, 0.0], device=DEV)[torch.arange(S, device=DEV) % 3]  # of the query's scores
    mix = torch.where(torch.rand(S, device=DEV) < 0.5, 1.0, -1.0)                      # of the key
    q, k = (torch.randn(1, S, 2, D, device=DEV) for _ in range(2))
    q[..., 0], q[..., 1] = 400.0 * end[None, :, None], 400.0 * (1 - end.abs())[None, :, None]
    k[..., 0], k[..., 1] = 40.0, 40.0 * mix[None, :, None]
    v = torch.randn(1, S, 2, D, device=DEV) * size
    q, k, v = (t.bfloat16().requires_grad_(True) for t in (q, k, v))
    do = (torch.randn(1, S, 2, D, device=DEV) / size).bfloat16()
    o = ops.flash_attention(q, k, v, softcap=softcap)
    got = [o, *torch.autograd.grad(o, (q, k, v), do)]
    with torch.no_grad():
        want, lim = oracle(q, k, v, do, True, None, -1, D ** -0.5, softcap, None, None)
        # The oracle's 1 - tanh^2 is 0 where the derivative is below 2^-52 (4e-24 here), and with it the bound's share of
        # delta's and dP's errors, p dx (e_delta + 2^-11 mag). Up to 2^-52 of that share is added back: e_delta <=
        # 2^-8 (max dP + max delta) <= 2^-8 mag, so 2^-52 (2^-8 + 2^-11) mag a score, and p sums to 1 over a row's keys.
        mag = 2 * (do.double().abs().sum(-1).max() * v.double().abs().max())
        share = D ** -0.5 * 2.0 ** -52 * (2.0 ** -8 + 2.0 ** -11) * mag
        lim[1] += share * k.double().abs().max()
        lim[2] += share * S * q.double().abs().max()
        compare(got, want, lim)
        plain = ops.flash_attention(q, k, v, softcap=softcap)
    assert plain.isfinite().all() and torch.equal(o == 0, plain == 0)


@pytest.mark.parametrize("dtype,eps", [(torch.float16, 2.0 ** -11), (torch.float32, 2.0 ** -24)])
def test_capped_attention_of_other_types_keeps_the_dense_path(dtype, eps, monkeypatch):
    """fp16 / fp32 layers of a capped model hold the scores in their own type: flash_attention's torch form would take
    twice the memory for fp16."""
    monkeypatch.setattr(fused, "flash_attention", None)
    torch.manual_seed(6)
    B, H, S, D, cap, scale = 2, 4, 90, 64, 20.0, 0.125
    q, k, v = (torch.randn(B, h, S, D, device=DEV).to(dtype) for h in (H, 2, 2))
    m = SimpleNamespace(is_causal=True, training=False)
    o, _ = hf_attention(m, q, k, v, None, scaling=scale, softcap=cap)
    assert o.dtype == dtype
    kd, vd = k.double().repeat_interleave(2, 1), v.double().repeat_interleave(2, 1)
    i = torch.arange(S, device=DEV)
    x = torch.matmul(q.double(), kd.transpose(-1, -2).contiguous()) * scale
    s = (cap * torch.tanh(x / cap)).masked_fill(i[None] > i[:, None], float("-inf"))
    p = torch.softmax(s, -1)
    # scores: product, scale, quotient, tanh and cap rounded to the type, each half a step of at most |x|, beside fp32 sums
    # over D; a score off by t changes p by a factor of up to 1 +- 2 t; p and the output are rounded once each
    mag = torch.matmul(q.double().abs(), kd.abs().transpose(-1, -2).contiguous()).max() * scale
    t = 5 * eps * x.abs().max() + (D + 1) * 2.0 ** -24 * mag
    lim = (2.5 * t + 2 * eps + S * 2.0 ** -24) * torch.matmul(p, vd.abs()).transpose(1, 2) + 2.0 ** -24
    assert ((o.double() - torch.matmul(p, vd).transpose(1, 2)).abs() <= lim).all()


@pytest.mark.parametrize("buffer", [None, torch.bfloat16, torch.float32])
def test_linear_token_stats_of_no_rows(buffer):
    """No rows: the weight's gradient is zero (nothing is added to a buffer), whatever its memory held."""
    w = torch.randn(96, 64, device=DEV).bfloat16().requires_grad_(True)
    h = torch.randn(0, 64, device=DEV).bfloat16().requires_grad_(True)
    labels = torch.zeros(0, device=DEV, dtype=torch.long)
    junk = [torch.full(w.shape, 7.0, device=DEV, dtype=t) for t in (torch.bfloat16, torch.float32)]
    del junk
    if buffer is None:
        r = ops.linear_token_stats(h, w, labels, top_k=2)
        gh, gw = torch.autograd.grad(r.logps.sum() + r.entropy.sum(), (h, w))
        assert gh.shape == (0, 64) and not gw.any()
        return
    w.main_grad = torch.full(w.shape, 3.0, device=DEV, dtype=buffer)
    for added, value in ((True, 3.0), (False, 0.0)):
        w.grad_added = added
        ops.linear_token_stats(h, w, labels).logps.sum().backward()
        assert (w.main_grad == value).all() and w.grad_added


def test_embedding_of_a_model_keeps_its_second_derivative():
    """Linear in the table: the gradient is differentiable in dY, as it was in front of the kernels."""
    torch.manual_seed(7)
    w = torch.randn(9, 8, device=DEV).requires_grad_(True)
    g = torch.randn(5, 8, device=DEV).requires_grad_(True)
    ids = torch.tensor([1, 1, 2, 8, 1], device=DEV)
    dw, = torch.autograd.grad(vocab_embedding(ids, w, 0, 9, False, 0.5), w, g, create_graph=True)
    dg, = torch.autograd.grad(dw.square().sum(), g)
    # (three summands at most and a factor that is a power of two: a few roundings of values up to 8)
    assert torch.allclose(dw.detach(), torch.zeros_like(w).index_add(0, ids, 0.5 * g.detach()), atol=1e-5)
    assert torch.allclose(dg, 2 * 0.5 * dw.detach()[ids], atol=1e-5)


def test_second_derivatives_of_the_python_nodes_are_refused():
    """The nodes for gradient buffers and the linear head's say so instead of leaving terms out."""
    x = torch.randn(4, 8, device=DEV).requires_grad_(True)
    v = torch.rand(8, device=DEV).requires_grad_(True)
    v.main_grad = torch.zeros(8, device=DEV)
    h = torch.randn(4, 64, device=DEV).bfloat16().requires_grad_(True)
    t = torch.randn(96, 64, device=DEV).bfloat16()
    labels = torch.zeros(4, dtype=torch.long, device=DEV)
    for y, z in ((ops.norm_add_norm(x, x.detach(), v, None, 1e-6)[1], x),
                 (ops.linear_token_stats(h, t, labels).logps, h)):
        d, = torch.autograd.grad(y.float().square().sum(), z, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            d.float().square().sum().backward()


@pytest.mark.parametrize("N", [5, 700])
def test_embedding_shard_behind_the_vocabulary(N):
    """A vocabulary smaller than the shards' rows: the last ranks' shards begin behind it and hold nothing."""
    w = torch.randn(2, 8, device=DEV).requires_grad_(True)
    ids = torch.arange(N, device=DEV) % 10
    y = vocab_embedding(ids, w, 12, 10, True)
    assert y.shape == (N, 8) and not y.any()
    assert not torch.autograd.grad(y, w, torch.ones_like(y))[0].any()
