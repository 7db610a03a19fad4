"""The norms around a block, its gate, its residual scale and the residual sum as one operator.

GPU tensors (bf16, fp16, fp32) run csrc/block_norm.hip, one kernel each way (and one for the weights' gradients);
CPU tensors run :func:`reference.norm_add_norm`.
"""
from __future__ import annotations

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import reference as ref
from .native import lib, on_kernels


def _target(w):
    """(buffer, add, returned gradient) of a weight gradient: the engine's flat buffer where there is one."""
    mg = getattr(w, "main_grad", None)
    if mg is not None:
        return mg.view(-1), bool(getattr(w, "grad_added", False)), None
    g = torch.empty_like(w)
    return g, False, g


def _packed(t):
    """``t`` contiguous and 16-byte aligned (a gradient can be a slice of a larger one)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _NormAddNormFn(Function):
    """The node for weights with a gradient buffer (others: csrc/decoder_ops.cpp)."""

    @staticmethod
    def forward(ctx, x, res, w1, w2, gate, eps, alpha, offset):
        x, res = _packed(x), _packed(res)
        h, s, r1, r2 = lib().block_norm_fwd(x, res, w1, w2, gate, eps, alpha, offset)
        ctx.save_for_backward(x, res, r1, r2)
        ctx.w = (w1, w2, gate)
        ctx.cfg = (alpha, offset)
        ctx.set_materialize_grads(False)
        return (s,) if w2 is None else (h, s)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x, res, r1, r2 = ctx.saved_tensors
        w1, w2, gate = ctx.w
        alpha, offset = ctx.cfg
        dh, ds = (None, grads[0]) if w2 is None else grads
        if dh is None and ds is None:
            return (None,) * 8
        dh = None if dh is None else _packed(dh)
        ds = None if ds is None else _packed(ds)
        bufs, rets, add, used, again = [None] * 3, [None] * 3, 0, [], []
        for i, (w, need) in enumerate(((w1, ctx.needs_input_grad[2]), (gate, ctx.needs_input_grad[4]),
                                       (w2, ctx.needs_input_grad[3]))):
            if w is None or not need:
                continue
            buf, more, rets[i] = _target(w)
            if any(b is not None and b.data_ptr() == buf.data_ptr() for b in bufs):
                # one parameter in two roles: the kernel writes its targets independently of each other
                again.append((buf, torch.empty_like(buf, dtype=torch.float32)))
                bufs[i] = again[-1][1]
                continue
            bufs[i] = buf
            add |= int(more) << i
            used.append(w)
        dx, dres = lib().block_norm_bwd(dh, ds, x, res, w1, w2, gate, r1, r2, alpha, offset, *bufs, add)
        for buf, part in again:
            buf.add_(part)
        for w in used:
            if getattr(w, "main_grad", None) is not None:
                w.grad_added = True
        return dx, dres, rets[0], rets[2], rets[1], None, None, None


class _RefNormAddNormFn(Function):
    """Torch math with gradient-buffer support."""

    @staticmethod
    def forward(ctx, x, res, w1, w2, gate, eps, alpha, offset):
        ctx.save_for_backward(x, res)
        ctx.w = (w1, w2, gate)
        ctx.cfg = (eps, alpha, offset)
        ctx.set_materialize_grads(False)
        h, s = ref.norm_add_norm(x, res, w1, w2, eps, gate, alpha, offset)
        return (s,) if w2 is None else (h, s)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        from .fused import _wgrad_vec
        x, res = ctx.saved_tensors
        ws = ctx.w
        if all(g is None for g in grads):
            return (None,) * 8
        with torch.enable_grad():
            leaves = [x.detach().requires_grad_(True), res.detach().requires_grad_(True)]
            wl = [None if w is None else w.detach().requires_grad_(True) for w in ws]
            h, s = ref.norm_add_norm(leaves[0], leaves[1], wl[0], wl[1], ctx.cfg[0], wl[2], *ctx.cfg[1:])
            ys = [s] if ws[1] is None else [h, s]
            ys, gs = zip(*((y, g) for y, g in zip(ys, grads) if g is not None))
            ins = leaves + [w for w in wl if w is not None]
            got = list(torch.autograd.grad(ys, ins, gs, allow_unused=True))
        dx, dres = got[:2]
        it, dws = iter(got[2:]), []
        for i, w in enumerate(ws):
            g = next(it) if w is not None else None
            if w is None or not ctx.needs_input_grad[2 + i]:
                dws.append(None)
            else:
                dws.append(_wgrad_vec(w, torch.zeros_like(w) if g is None else g))
        return dx, dres, *dws, None, None, None


def norm_add_norm(x: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor,
                  pre_weight: torch.Tensor | None, eps: float, gate: torch.Tensor | None = None,
                  residual_scale: float = 1.0, weight_offset: float = 0.0):
    """``s = residual + residual_scale * gate * rmsnorm(x; post_weight)`` and ``h = rmsnorm(s; pre_weight)`` ->
    ``(h, s)``: what lies between the output ``x`` of one block of a decoder layer and the input ``h`` of the next in
    layers with norms on both sides of a block. ``pre_weight=None``: no block follows, h is None. ``gate``: learned
    factors per channel [H]. ``weight_offset`` 1 for weights stored around zero (norms that multiply by 1 + w).

    x, residual: [..., H], H a multiple of 8 up to 8192, with weights of their dtype. Statistics, the sum and both
    norms are held in fp32, and h is normalised from the unrounded sum: each output is rounded once."""
    if x.shape != residual.shape:
        raise ValueError(f"norm_add_norm: x {tuple(x.shape)} and residual {tuple(residual.shape)} differ")
    for n, t in (("residual", residual), ("post_weight", post_weight), ("pre_weight", pre_weight), ("gate", gate)):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"norm_add_norm: {n} is {t.dtype}, x is {x.dtype}")
    for n, t in (("post_weight", post_weight), ("pre_weight", pre_weight), ("gate", gate)):
        if t is not None and tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"norm_add_norm: {n} must be [{x.shape[-1]}], is {tuple(t.shape)}")
    native = on_kernels(x)
    if native and not any(hasattr(w, "main_grad") for w in (post_weight, pre_weight, gate)):
        out = lib().block_norm(x, residual, post_weight, pre_weight, gate, eps, residual_scale, weight_offset)
        return (None, out[0]) if pre_weight is None else (out[0], out[1])
    fn = _NormAddNormFn if native else _RefNormAddNormFn
    out = fn.apply(x, residual, post_weight, pre_weight, gate, float(eps), float(residual_scale), float(weight_offset))
    return (None, out[0]) if pre_weight is None else out
