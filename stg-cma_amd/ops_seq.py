"""Sequence operators with gradients: attention over ragged token sequences with a learned relative position bias by buckets, and the norm - gate -
residual - norm join around a block.  Forward and backward are libstgcma_hip.so launches on torch's current stream (relattn.hip, normjoin.hip);
torch supplies memory only.  No state is kept between calls, so the calls may be captured, replayed and issued from several streams.  (As for any
captured backward: drop eager autograd graphs of the same leaves first, their accumulation nodes belong to the eager stream.)
"""
import torch
from torch.autograd.function import once_differentiable

from . import kernels as K
from .kernels import BF16


def _ready(dy, dtype):
    """An incoming gradient as the kernels read it: its own type, dense rows, 16-byte aligned."""
    if dy.dtype != dtype:
        dy = dy.to(dtype)
    if not dy.is_contiguous():
        dy = dy.contiguous()
    return dy.clone() if dy.data_ptr() % 16 else dy


def _apply(fn, device, *args):
    """fn.apply with the tensors' device as the current one (a kernel launch goes to the current device)."""
    if device.type == "cuda" and device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return fn.apply(*args)
    return fn.apply(*args)


class RelAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, geom, cu_q, cu_k, max_q, max_k, key_mask):
        train = any(ctx.needs_input_grad[:4])
        o, lse, a = K._relattn_fwd(geom, q, k, v, table, cu_q, cu_k, max_q, max_k, key_mask, None, train)
        if train:
            plan = geom.plan(q.device)
            ctx.save_for_backward(q, k, v, o, lse, table, cu_q, cu_k, key_mask, plan)
            ctx.call = a                                       # the checked sizes and strides; its pointers are taken again from the saved tensors
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, table, cu_q, cu_k, key_mask, plan = ctx.saved_tensors
        need = ctx.needs_input_grad
        a = type(ctx.call).from_buffer_copy(ctx.call)
        a.Q, a.K, a.V, a.O = q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr()
        a.ldq, a.ldk, a.ldv, a.ldo = K._rel_ld(q), K._rel_ld(k), K._rel_ld(v), K._rel_ld(o)      # (hooks may have stored a dense copy)
        a.lse, a.table, a.cu_q, a.plan = lse.data_ptr(), table.data_ptr(), cu_q.data_ptr(), plan.data_ptr()
        a.cu_k = a.cu_q if cu_k is None else cu_k.data_ptr()
        a.key_mask = None if key_mask is None else key_mask.data_ptr()
        grads = K._relattn_bwd(a, q.device, _ready(do, BF16), need[3])
        return tuple(g if n else None for g, n in zip(grads, need)) + (None,) * 6


def rel_attention(q, k, v, table, geom, cu_q, cu_k=None, *, max_q=None, max_k=None, key_mask=None):
    """softmax(scale q k^T + table[bucket(distance)]) v over ragged sequences, differentiable in q, k, v and table (kernels.relattn_fwd has the
    arguments; geom: kernels.RelGeom).  Returns o bf16 [Tq, H * D]."""
    return _apply(RelAttentionFn, q.device, q, k, v, table, geom, cu_q, cu_k, max_q, max_k, key_mask)


class NormJoinFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, gate, post_w, post_b, pre_w, pre_b, kind, alpha, eps, rows_per_group):
        train = any(ctx.needs_input_grad[:7])
        x_new, y, stats, a = K._norm_join_fwd(x, h, gate, (post_w, post_b, pre_w, pre_b), kind, alpha, eps, rows_per_group, train)
        if train:
            ctx.save_for_backward(x_new, h, stats, gate, post_w, post_b, pre_w, pre_b)
            ctx.call = a                                       # the checked sizes and strides; its pointers are taken again from the saved tensors
            ctx.set_materialize_grads(False)
        return x_new, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dx_new, dy):
        if dx_new is None and dy is None:
            return (None,) * 11
        x_new, h, stats, gate, post_w, post_b, pre_w, pre_b = ctx.saved_tensors
        need = ctx.needs_input_grad
        a = type(ctx.call).from_buffer_copy(ctx.call)
        a.xo, a.h, a.stats, a.w1, a.w2 = x_new.data_ptr(), h.data_ptr(), stats.data_ptr(), post_w.data_ptr(), pre_w.data_ptr()
        a.ldxo, a.ldh = K._rel_ld(x_new), K._rel_ld(h)
        if gate is not None:
            a.gate = gate.data_ptr()
        if post_b is not None:
            a.b1 = post_b.data_ptr()
        if pre_b is not None:
            a.b2 = pre_b.data_ptr()
        dy = torch.zeros(h.shape, dtype=BF16, device=h.device) if dy is None else _ready(dy, BF16)
        if dx_new is not None:
            dx_new = _ready(dx_new, x_new.dtype)
        dx, dh, dw1, db1, dw2, db2, dg = K._norm_join_bwd(a, h.device, x_new.dtype, dy, dx_new, (post_w, post_b, pre_w, pre_b), gate, any(need[3:7]), need[2])
        if not all(need[:7]):
            dx, dh, dg, dw1, db1, dw2, db2 = (g if n else None for g, n in zip((dx, dh, dg, dw1, db1, dw2, db2), need))
        return dx, dh, dg, dw1, db1, dw2, db2, None, None, None, None


def norm_join(x, h, gate, post_w, post_b, pre_w, pre_b, *, kind="layer", alpha=1.0, eps=1e-5, rows_per_group=None):
    """(x_new, y): x_new = alpha x + gate * Norm(h), y = Norm(x_new), each norm with its own weight and bias -- the norm after a block, its gate, the
    residual sum and the norm before the next block (kernels.norm_join_fwd has the arguments).  Differentiable in every tensor."""
    return _apply(NormJoinFn, x.device, x, h, gate, post_w, post_b, pre_w, pre_b, kind, alpha, eps, rows_per_group)
