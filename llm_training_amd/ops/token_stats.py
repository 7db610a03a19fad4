"""Log probabilities of given tokens with the entropy and the likeliest alternatives of every position.

GPU logits (bf16, fp16, fp32) run csrc/token_stats.hip: one pass over the logits forward, one backward for the
gradients of all the outputs, and no [N, V] log-softmax. CPU logits run :func:`reference.token_stats`.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import reference as ref
from .native import lib, on_kernels, use_native

MAX_TOP_K = 32


class TokenStats(NamedTuple):
    logps: torch.Tensor      # [...] fp32: log p(label)
    entropy: torch.Tensor    # [...] fp32: -sum p log p, in nats
    top_logps: torch.Tensor  # [..., K] fp32: log p of the K likeliest tokens, descending
    top_ids: torch.Tensor    # [..., K] int64


def _f32(g, n):
    return None if g is None else g.reshape(n).float().contiguous()


class _LinearTokenStatsFn(Function):
    """Statistics of h @ W^T in row chunks, as :class:`fused._LinearLogpsFn`: the backward recomputes each chunk's
    logits and overwrites them with their gradient, so one [chunk, V] buffer lives at a time."""

    @staticmethod
    def forward(ctx, h, w, labels, ignore_index, top_k, chunk):
        from .fused import mm_nt
        N = h.shape[0]
        f = dict(device=h.device, dtype=torch.float32)
        logps, ent, norm = torch.empty(N, **f), torch.empty(N, **f), torch.empty(N, 2, **f)
        top, ids = torch.empty(N, top_k, **f), torch.empty(N, top_k, device=h.device, dtype=torch.int64)
        for s0 in range(0, N, chunk):
            s = slice(s0, min(N, s0 + chunk))
            got = lib().token_stats_fwd(mm_nt(h[s], w), labels[s], ignore_index, top_k)
            for dst, src in zip((logps, ent, norm, top, ids), got):
                dst[s] = src
        ctx.save_for_backward(h, labels, norm, ent, ids)
        ctx.w = w
        ctx.cfg = (ignore_index, chunk)
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return logps, ent, top, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logp, g_ent, g_top, _):
        from .fused import _apply_weight_grad, dw_accumulator, dw_add_chunk, mm_nn, mm_nt, weight_t
        h, labels, norm, ent, ids = ctx.saved_tensors
        w = ctx.w
        ignore_index, chunk = ctx.cfg
        if g_logp is None and g_ent is None and g_top is None:
            return (None,) * 6
        N = h.shape[0]
        g_logp, g_ent = _f32(g_logp, N), _f32(g_ent, N)
        g_top = None if g_top is None else g_top.float().contiguous()
        need_h, need_w = ctx.needs_input_grad[:2]
        dh = torch.empty_like(h) if need_h else None
        dw = dw_accumulator(w, N, chunk) if need_w else None
        if need_w and N == 0:  # (no chunk writes it)
            dw.zero_()
        wt = weight_t(w, N) if need_h and N > chunk else None
        for s0 in range(0, N, chunk):
            s = slice(s0, min(N, s0 + chunk))
            lg = mm_nt(h[s], w)
            lib().token_stats_bwd_(lg, labels[s], ignore_index, norm[s], ent[s], ids[s],
                                   None if g_logp is None else g_logp[s], None if g_ent is None else g_ent[s],
                                   None if g_top is None else g_top[s], lg)
            if need_h:
                mm_nn(lg, w, out=dh[s], wt=wt)
            if need_w:
                dw_add_chunk(dw, lg, h[s], s0 == 0)
        dwr = None
        if need_w:
            dwr = _apply_weight_grad(w, dw, torch.ones((), device=dw.device, dtype=torch.float32))
        return dh, dwr, None, None, None, None


def _check(labels, rows, top_k, vocab):
    if labels.numel() != rows:
        raise ValueError(f"token_stats: {labels.numel()} labels for {rows} rows")
    if not 0 <= top_k <= min(MAX_TOP_K, vocab):
        raise ValueError(f"token_stats: top_k must be between 0 and min({MAX_TOP_K}, vocabulary {vocab}), is {top_k}")


def token_stats(logits: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100, top_k: int = 0) -> TokenStats:
    """:class:`TokenStats` of ``logits`` [..., V] at ``labels`` [...] (int64), differentiable in the logits.

    Positions labelled ``ignore_index`` give zeros, ids of -1 and no gradient. Equal logits are ranked by the lower
    id. Logits of -inf have probability zero; a row without a finite logit, with a NaN or with +inf gives NaN. ``top_k``
    up to 32 (GPU vocabularies up to 229376 tokens at 32, more at fewer)."""
    V = logits.shape[-1]
    # (views are nodes of the graph: none where the shapes are already [N, V] and [N])
    lg = logits if logits.dim() == 2 else logits.reshape(-1, V)
    lab = labels if labels.dim() == 1 else labels.reshape(-1)
    _check(lab, lg.shape[0], top_k, V)
    if on_kernels(lg):
        if (V > 1 and lg.stride(1) != 1) or (lg.shape[0] > 1 and lg.stride(0) < V):  # (or one row, expanded)
            lg = lg.contiguous()
        out = lib().token_stats(lg, lab.long().contiguous(), ignore_index, top_k)
    else:
        out = ref.token_stats(lg, lab.long(), ignore_index, top_k)
    if labels.dim() == 1:
        return TokenStats(*out)
    sh = labels.shape
    return TokenStats(out[0].view(sh), out[1].view(sh), out[2].view(*sh, top_k), out[3].view(*sh, top_k))


def linear_token_stats(h: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100,
                       top_k: int = 0, chunk_size: int = 8192) -> TokenStats:
    """:func:`token_stats` of ``h @ w.T`` (h [..., H], w [V, H]) without the whole [N, V] logits."""
    h2, lab = h.reshape(-1, h.shape[-1]), labels.reshape(-1)
    _check(lab, h2.shape[0], top_k, w.shape[0])
    if h2.shape[1] != w.shape[1] or chunk_size < 1:
        raise ValueError(f"linear_token_stats: h [..., {h2.shape[1]}], w {tuple(w.shape)}, chunk_size {chunk_size}")
    if use_native(h2):
        out = _LinearTokenStatsFn.apply(h2.contiguous(), w, lab.long().contiguous(), int(ignore_index), int(top_k),
                                        int(chunk_size))
        sh = labels.shape
        return TokenStats(out[0].view(sh), out[1].view(sh), out[2].view(*sh, top_k), out[3].view(*sh, top_k))
    from .fused import linear
    return token_stats(linear(h2, w).view(*labels.shape, w.shape[0]), labels, ignore_index, top_k)
