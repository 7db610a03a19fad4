"""Embedding lookup with scaling, and its weight gradient by sorted tokens.

GPU tensors (bf16, fp16, fp32) run csrc/embedding.hip: the gradient of a row is summed in fp32 over its tokens in
ascending order and rounded once, so it is the same bits in every run. CPU tensors run torch ops.
"""
from __future__ import annotations

import torch
from torch.autograd import Function

from .native import lib, on_kernels


def _rows(v0, v1, shape):
    """Rows of the table that hold ids (a shard wholly behind a small vocabulary has none: v1 < v0)."""
    return max(0, min(v1 - v0, shape[0]))


class _EmbeddingFn(Function):
    @staticmethod
    def forward(ctx, ids, w, v0, v1, sharded, scale):
        ctx.save_for_backward(ids)
        ctx.w = w  # (the parameter itself: saved tensors are unpacked as aliases without main_grad)
        ctx.wshape = w.shape
        ctx.cfg = (v0, v1, sharded, scale)
        if on_kernels(w):
            return lib().embedding_fwd(ids.contiguous(), w.contiguous(), v0, _rows(v0, v1, w.shape), scale, sharded)
        local = ids - v0
        if sharded:  # vocab-sharded: rows owned by other ranks contribute zeros
            mask = (ids >= v0) & (ids < v1)
            local = torch.where(mask, local, torch.zeros_like(local))
            out = torch.nn.functional.embedding(local, w)
            out = out * mask.unsqueeze(-1).to(out.dtype)
        else:
            out = torch.nn.functional.embedding(local, w)
        return out if scale == 1.0 else (out.float() * scale).to(out.dtype)

    @staticmethod
    def backward(ctx, g):
        (ids,) = ctx.saved_tensors
        w = ctx.w
        v0, v1, sharded, scale = ctx.cfg
        if not ctx.needs_input_grad[1]:
            return None, None, None, None, None, None
        mg = getattr(w, "main_grad", None)
        # (a backward that is differentiated itself, create_graph=True, takes the torch form below)
        if on_kernels(g) and not (mg is None and torch.is_grad_enabled() and g.requires_grad):
            fresh = mg is None
            dw = torch.empty(ctx.wshape, dtype=w.dtype, device=g.device) if fresh else mg.view(ctx.wshape)
            lib().embedding_bwd_(ids.contiguous(), g.contiguous(), dw, v0, _rows(v0, v1, ctx.wshape), scale,
                                 not fresh and bool(getattr(w, "grad_added", False)), sharded)
            if fresh:
                return None, dw, None, None, None, None
            w.grad_added = True
            return None, None, None, None, None, None
        if scale != 1.0:
            g = g.float() * scale
        mask = (ids >= v0) & (ids < v1)
        local = (ids - v0).masked_fill(~mask, 0).reshape(-1)
        g2 = (g * mask.unsqueeze(-1).to(g.dtype)).reshape(-1, g.shape[-1])
        if mg is None:
            dw = torch.zeros(ctx.wshape, dtype=g.dtype, device=g.device)
            dw.index_add_(0, local, g2)
            return None, dw.to(w.dtype), None, None, None, None
        if not getattr(w, "grad_added", False):
            mg.zero_()
        mg.view(ctx.wshape).index_add_(0, local, g2.to(mg.dtype))
        w.grad_added = True
        return None, None, None, None, None, None


def vocab_embedding(ids: torch.Tensor, w: torch.Tensor, v0: int, v1: int, sharded: bool, scale: float = 1.0):
    """Rows ``ids - v0`` of ``w`` (a table or, ``sharded``, one rank's rows [v0, v1) of it, whose foreign ids give
    zeros) times ``scale``."""
    return _EmbeddingFn.apply(ids, w, int(v0), int(v1), bool(sharded), float(scale))


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[ids]``: ids int32 / int64 of any shape, weight [V, H] -> [..., H] in the weight's dtype.

    The product is taken in fp32 and rounded once. The gradient goes to ``weight.main_grad`` where the engine keeps
    one. On the GPU an id outside the table gives a row of zeros and is reported by ``check_kernel_errors``."""
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"embedding: ids must be int32 or int64, are {ids.dtype}")
    if weight.dim() != 2:
        raise ValueError(f"embedding: weight must be [V, H], is {tuple(weight.shape)}")
    if on_kernels(weight) and not hasattr(weight, "main_grad"):
        return lib().embedding(ids, weight, scale)
    return vocab_embedding(ids, weight, 0, weight.shape[0], False, scale)
