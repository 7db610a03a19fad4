"""Calls of the decoder operators at the edge of what their documentation allows, as far as the host decides them."""
import torch

from llm_training_amd import ops
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
