"""Sequence operators with gradients: attention over ragged token sequences with a learned relative position bias by buckets, and the norm - gate -
residual - norm join around a block.  Forward and backward are libstgcma_hip.so launches on torch's current stream (relattn.hip, normjoin.hip);
torch supplies memory only.  No state is kept between calls, so the calls may be captured, replayed and issued from several streams.
"""
import contextlib

import torch
from torch.autograd.function import once_differentiable

from . import kernels as K
from .kernels import BF16


def _on(t):
    """The device of the call's tensors as the current one (a kernel launch goes to the current device)."""
    if t.is_cuda and t.device.index != torch.cuda.current_device():
        return torch.cuda.device(t.device)
    return contextlib.nullcontext()


def _grad(dy, dtype):
    """An incoming gradient as the kernels read it: its own type, dense rows, 16-byte aligned."""
    dy = dy.to(dtype).contiguous()
    return dy.clone() if dy.data_ptr() % 16 else dy


class RelAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, geom, cu_q, cu_k, max_q, max_k, key_mask):
        need = ctx.needs_input_grad
        train = any(need[:4])
        o, lse = K.relattn_fwd(geom, q, k, v, table, cu_q, cu_k, max_q=max_q, max_k=max_k, key_mask=key_mask, want_lse=train)
        if train:
            ctx.save_for_backward(q, k, v, table, cu_q, cu_k, key_mask, o, lse)
            ctx.how = (geom, max_q, max_k)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, table, cu_q, cu_k, key_mask, o, lse = ctx.saved_tensors
        geom, max_q, max_k = ctx.how
        need = ctx.needs_input_grad
        with _on(q):
            grads = K.relattn_bwd(geom, q, k, v, table, cu_q, cu_k, o, lse, _grad(do, BF16), max_q=max_q, max_k=max_k, key_mask=key_mask,
                                  want_table=need[3])
        return tuple(g if n else None for g, n in zip(grads, need)) + (None,) * 6


def rel_attention(q, k, v, table, geom, cu_q, cu_k=None, *, max_q=None, max_k=None, key_mask=None):
    """softmax(scale q k^T + table[bucket(distance)]) v over ragged sequences, differentiable in q, k, v and table (kernels.relattn_fwd has the
    arguments; geom: kernels.RelGeom).  Returns o bf16 [Tq, H * D]."""
    with _on(q):
        return RelAttentionFn.apply(q, k, v, table, geom, cu_q, cu_k, max_q, max_k, key_mask)


class NormJoinFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, gate, post_w, post_b, pre_w, pre_b, how):
        train = any(ctx.needs_input_grad[:7])
        x_new, y, stats = K.norm_join_fwd(x, h, gate, post_w, post_b, pre_w, pre_b, want_stats=train, **how)
        if train:
            ctx.save_for_backward(x_new, h, gate, post_w, post_b, pre_w, pre_b, stats)
            ctx.how = how
            ctx.set_materialize_grads(False)
        return x_new, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dx_new, dy):
        x_new, h, gate, post_w, post_b, pre_w, pre_b, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dx_new is None and dy is None:
            return (None,) * 8
        with _on(h):
            dy = torch.zeros_like(h) if dy is None else _grad(dy, BF16)
            dx_new = None if dx_new is None else _grad(dx_new, x_new.dtype)
            g = K.norm_join_bwd(x_new, h, gate, post_w, post_b, pre_w, pre_b, stats, dy, dx_new, want_params=any(need[3:7]), want_gate=need[2], **ctx.how)
        names = ("dx", "dh", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b")
        return tuple(g[n] if w else None for n, w in zip(names, need)) + (None,)


def norm_join(x, h, gate, post_w, post_b, pre_w, pre_b, *, kind="layer", alpha=1.0, eps=1e-5, rows_per_group=None):
    """(x_new, y): x_new = alpha x + gate * Norm(h), y = Norm(x_new), each norm with its own weight and bias -- the norm after a block, its gate, the
    residual sum and the norm before the next block (kernels.norm_join_fwd has the arguments).  Differentiable in every tensor."""
    with _on(x):
        return NormJoinFn.apply(x, h, gate, post_w, post_b, pre_w, pre_b, dict(kind=kind, alpha=alpha, eps=eps, rows_per_group=rows_per_group))
