"""The join's column sums (gradients of weights, biases and gate) against 64-bit sums, within bounds that a missing row or a zero does not meet."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import join_ref as J
from test_norm_join_gpu import CASES, _make

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
LEAVES = ("x", "h", "gate", "w1", "b1", "w2", "b2")
NAMES = {"gate": "gate", "w1": "post_w", "b1": "post_b", "w2": "pre_w", "b2": "pre_b"}

MORE = [
    (2000, 64, "layer", F32, "one", None, True, True, 1.0, True),
    (2001, 72, "rms", BF16, "one", None, False, False, 1.0, True),
    (9, 512, "layer", F32, "one", None, True, True, 1.0, True),           # three blocks: the few-rows join of their sums
    (4500, 768, "rms", BF16, "group", 197, False, False, 1.0, True),      # groups in pieces
]


@pytest.mark.parametrize("case", range(len(CASES) + len(MORE)))
def test_column_sums(stg, gpu, case):
    from stgcma import ops_seq
    rows, C, kind, stream, gate, rpg, pb, qb, alpha, with_dx = (CASES + MORE)[case]
    t = _make(gpu, rows, C, kind, stream, gate, rpg, pb, qb, 500 + case)
    leaf = {n: t[n].detach().requires_grad_(True) for n in LEAVES if t[n] is not None}
    xn, y = ops_seq.norm_join(*[leaf.get(n) for n in LEAVES], kind=kind, alpha=alpha, rows_per_group=rpg)
    grads = torch.autograd.grad([xn, y] if with_dx else [y], list(leaf.values()), [t["dxn"], t["dy"]] if with_dx else [t["dy"]])
    got = dict(zip(leaf, grads))
    for n, (val, bound, _) in J.column_sums(t, kind, alpha, 1e-5, rpg, xn.detach(), with_dx).items():
        name = next(k for k, v in NAMES.items() if v == n)
        d = (got[name].double() - val).abs()
        assert got[name].shape == val.shape and bool((d <= bound + 1e-30).all()), (n, float((d / bound).max()), float(d.max()), float(val.abs().max()))


@pytest.mark.parametrize("rows,C", [(12, 512), (40, 128), (30, 1024), (7, 8192)])
def test_partial_sums_that_cancel(stg, gpu, rows, C):
    """2^24, then 1, then -2^24 far apart in the rows: the blocks' sums are these numbers, and added in 64 bits they make exactly 1."""
    from stgcma import kernels as K
    x = torch.randn(rows, C, device=gpu)
    h = torch.randn(rows, C, device=gpu).to(BF16)
    w1, b1, w2, b2 = torch.zeros(C, device=gpu), torch.ones(C, device=gpu), torch.ones(C, device=gpu), torch.zeros(C, device=gpu)     # n = 1
    gate = torch.tensor([0.5], device=gpu)
    xn, y, st = K.norm_join_fwd(x, h, gate, w1, b1, w2, b2)
    big = torch.zeros(rows, C, device=gpu)
    big[0, 3], big[rows // 2, 3], big[rows - 1, 3] = 2.0 ** 24, 1.0, -2.0 ** 24
    zero = torch.zeros(rows, C, dtype=BF16, device=gpu)
    g = K.norm_join_bwd(xn, h, gate, w1, b1, w2, b2, st, zero, big)
    assert float(g["dgate"]) == 1.0
    assert float(g["dpost_b"][3]) == 0.5
    g = K.norm_join_bwd(xn, h, gate, w1, b1, w2, b2, st, big.to(BF16))
    assert float(g["dpre_b"][3]) == 1.0
