"""Calls of the decoder operators at the edge of what their documentation allows, as far as the host decides them."""
from types import SimpleNamespace

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from llm_training_amd import ops
from llm_training_amd.models.hf_causal_lm import hf_attention
from llm_training_amd.ops import block_norm as bn
from llm_training_amd.ops import reference as ref


class _TorchKernels:
    """Stand-in for the block-norm kernels with their contract: every target is written (or added to) from its state
    before the launch, in an order nobody promises (here the last role first)."""

    def block_norm_fwd(self, x, res, w1, w2, gate, eps, alpha, offset):
        h, s = ref.norm_add_norm(x, res, w1, w2, eps, gate, alpha, offset)
        self.cfg = (eps, alpha, offset)
        return h, s, torch.empty(0), torch.empty(0)

    def block_norm_bwd(self, dh, ds, x, res, w1, w2, gate, r1, r2, alpha, offset, dw1, dgate, dw2, add):
        with torch.enable_grad():
            ins = [None if t is None else t.detach().requires_grad_(True) for t in (x, res, w1, gate, w2)]
            h, s = ref.norm_add_norm(ins[0], ins[1], ins[2], ins[4], self.cfg[0], ins[3], alpha, offset)
            ys, gs = zip(*((y, g) for y, g in ((h, dh), (s, ds)) if g is not None))
            used = [t for t in ins if t is not None]
            got = dict(zip(map(id, used), torch.autograd.grad(ys, used, gs, allow_unused=True)))
        before = [None if t is None else t.clone() for t in (dw1, dgate, dw2)]
        for i, (t, w) in reversed(list(enumerate(zip((dw1, dgate, dw2), ins[2:])))):
            if t is not None:
                t.copy_(got[id(w)] + (before[i] if add >> i & 1 else 0))
        return got[id(ins[0])], got[id(ins[1])]


def test_norm_add_norm_one_parameter_in_two_roles(monkeypatch):
    """One parameter as two or three of the weights, with a gradient buffer: the buffer gets the sum of the roles'."""
    monkeypatch.setattr(bn, "on_kernels", lambda t: True)
    fake = _TorchKernels()
    monkeypatch.setattr(bn, "lib", lambda: fake)
    torch.manual_seed(0)
    x, res, dh, ds = (torch.randn(5, 16) for _ in range(4))
    for roles in ("w1=w2", "w1=gate", "w2=gate", "all"):
        w = torch.rand(16).requires_grad_(True)
        v = torch.rand(16).requires_grad_(True)
        w1, w2, gate = {"w1=w2": (w, w, v), "w1=gate": (w, v, w), "w2=gate": (v, w, w), "all": (w, w, w)}[roles]
        plain = torch.autograd.grad(ref.norm_add_norm(x, res, w1, w2, 1e-5, gate), w, (dh, ds))[0]
        for added in (False, True):
            w.main_grad, w.grad_added = torch.full((16,), 3.0), added
            y = ops.norm_add_norm(x.clone().requires_grad_(True), res, w1, w2, 1e-5, gate=gate)
            torch.autograd.backward(y, (dh, ds))
            assert torch.allclose(w.main_grad, plain + (3.0 if added else 0.0), atol=1e-5), (roles, added)
            assert w.grad_added and w.grad is None


def _capped64(q, k, v, scale, cap, window=None):
    """Causal capped attention of [B, H, S, D] in 64 bits, [B, S, H, D]."""
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    i = torch.arange(q.shape[2])
    s = cap * torch.tanh(q @ k.transpose(-1, -2) * scale / cap)
    see = i[None] <= i[:, None]
    if window is not None:
        see &= i[:, None] - i[None] < window
    return (torch.softmax(s.masked_fill(~see, float("-inf")), -1) @ v).transpose(1, 2)


def test_dense_capped_attention_multiplies_by_contiguous_operands():
    """The dense path of capped attention (here: a cap beyond the kernels' range): no product, forward or backward, has a
    transposed view on its right, and the gradients are those of the formula."""
    m = SimpleNamespace(is_causal=True, training=False)
    seen = []

    class Products(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if func in (torch.ops.aten.bmm.default, torch.ops.aten.baddbmm.default):
                seen.append(args[-1].is_contiguous())
            return func(*args, **(kwargs or {}))

    torch.manual_seed(0)
    q = torch.randn(2, 7, 4, 6, dtype=torch.float64).transpose(1, 2).requires_grad_(True)
    k, v = (torch.randn(2, 7, 2, 6, dtype=torch.float64).transpose(1, 2).requires_grad_(True) for _ in range(2))
    do = torch.randn(2, 7, 4, 6, dtype=torch.float64)
    with Products():
        o, _ = hf_attention(m, q, k, v, None, scaling=0.4, softcap=5e3)
        got = torch.autograd.grad(o, (q, k, v), do)
    assert len(seen) == 6 and all(seen), seen
    want = _capped64(q, k, v, 0.4, 5e3)
    assert torch.allclose(o, want, atol=1e-6)  # (the probabilities are taken in fp32)
    for a, b in zip(got, torch.autograd.grad(want, (q, k, v), do)):
        assert torch.allclose(a, b, atol=1e-5)


def test_dense_attention_keeps_a_window_without_segments():
    """A sliding window narrower than the sequence, no segment ids: capped (a cap beyond the kernels' range)."""
    m = SimpleNamespace(is_causal=True, training=False)
    torch.manual_seed(1)
    q = torch.randn(2, 4, 9, 6)
    k, v = (torch.randn(2, 2, 9, 6) for _ in range(2))
    for window in (1, 4, 8, 9, 30):
        o, _ = hf_attention(m, q, k, v, None, scaling=0.4, softcap=5e3, sliding_window=window)
        want = _capped64(q.double(), k.double(), v.double(), 0.4, 5e3, window)
        assert torch.allclose(o.double(), want, atol=1e-5), window  # (fp32: some dozen roundings of values up to 4)


def test_norm_add_norm_refuses_a_second_derivative():
    """Its backward has no graph: differentiating it says so instead of leaving terms out."""
    x, res, w = torch.randn(3, 8).requires_grad_(True), torch.randn(3, 8), torch.rand(8)
    _, s = ops.norm_add_norm(x, res, w, None, 1e-5)
    g, = torch.autograd.grad(s.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.square().sum().backward()


def test_dense_attention_of_a_module_without_a_causal_mask():
    """No causal mask comes with the window there: SDPA over all keys, as without one."""
    m = SimpleNamespace(is_causal=False, training=False)
    torch.manual_seed(2)
    q, k, v = (torch.randn(1, 2, 6, 8) for _ in range(3))
    o, _ = hf_attention(m, q, k, v, None, scaling=0.3, sliding_window=2)
    want = torch.softmax(q @ k.transpose(-1, -2) * 0.3, -1) @ v
    assert torch.allclose(o, want.transpose(1, 2), atol=1e-5)


def test_dense_capped_attention_under_autocast():
    """fp32 tensors, products in bf16: the gradients come back in fp32, as near as bf16 operands leave them."""
    m = SimpleNamespace(is_causal=True, training=False)
    torch.manual_seed(3)
    q, k, v = (torch.randn(1, 2, 6, 8).requires_grad_(True) for _ in range(3))
    with torch.autocast("cpu", dtype=torch.bfloat16):
        o, _ = hf_attention(m, q, k, v, None, scaling=0.3, softcap=5e3)
    got = torch.autograd.grad(o.float().sum(), (q, k, v))
    want = torch.autograd.grad(_capped64(*(t.double() for t in (q, k, v)), 0.3, 5e3).sum(), (q, k, v))
    for a, b in zip(got, want):
        # a dozen bf16 roundings on the way, 2^-8 each of values up to 4, in sums of up to 8
        assert a.dtype == torch.float32 and (a - b).abs().max() < 12 * 2.0 ** -8 * 4 * 8 ** 0.5
