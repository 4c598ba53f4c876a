"""The join's bounds catch what they are for (on the CPU, with 64-bit sums in the kernel's place), and the size of its gradient buffer."""
import ctypes as C
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import join_ref as J
import seq_ref as R
from test_norm_join_gpu import CASES, _make
from test_norm_join_sums_gpu import MORE


@pytest.mark.parametrize("case", range(len(CASES) + len(MORE)))
def test_bounds_see_a_missing_row_and_a_zero(case):
    rows, Cw, kind, stream, gate, rpg, pb, qb, alpha, with_dx = (CASES + MORE)[case]
    t = _make(torch.device("cpu"), rows, Cw, kind, stream, gate, rpg, pb, qb, 900 + case)
    a = [t[n] for n in ("x", "h", "gate", "w1", "b1", "w2", "b2")]
    xn = R.norm_join(*a, kind, alpha, 1e-5, rpg)["x_new"].to(stream)
    want = R.norm_join(*a, kind, alpha, 1e-5, rpg, t["dy"], t["dxn"] if with_dx else None, x_new=xn)
    for name, (val, bound, terms) in J.column_sums(t, kind, alpha, 1e-5, rpg, xn, with_dx).items():
        ref = want["d" + name]
        assert val.shape == ref.shape and bool(((val - ref).abs() <= 1e-9 * (1 + ref.abs())).all()), name        # two ways to the same value
        if rows == 1 and kind == "layer" and Cw == 8:
            continue
        assert bool((val.abs() > bound).any()), (name, "zero passes")
        last = terms[rows - 1:]                               # the last row left out
        if name == "gate" and gate == "group":
            gone, b = last[0].abs(), bound[-1]
        elif name == "gate" and gate == "one":
            gone, b = last.sum().abs().view(1), bound.view(1)
        else:
            gone, b = last[0].abs(), bound
        assert bool((gone > b).any()), (name, "a missing row passes", float((gone / b).max()))


@pytest.mark.parametrize("kind,biases,want", [(0, 2, 4 * 64), (0, 0, 2 * 64), (1, 2, 4 * 64 + 4), (1, 1, 3 * 64 + 4), (2, 2, 5 * 64), (3, 1, 3 * 64)])
def test_size_of_the_gradient_buffer(stg, kind, biases, want):
    """stg_norm_join_param_floats is the number of floats that the backward writes: the sums, padded to whole 16-byte pieces."""
    from stgcma import _lib
    a = _lib.NormJoinArgs()
    for n in ("x", "h", "w1", "w2", "xo", "y", "stats"):
        setattr(a, n, 4096)
    a.gate = 4096 if kind else None
    a.b1, a.b2 = (4096 if biases > 0 else None), (4096 if biases > 1 else None)
    a.x_dtype, a.gate_kind, a.rows_per_group, a.rows, a.C = _lib.STG_F32, kind, 4, 10, 64
    assert _lib.lib().stg_norm_join_param_floats(C.byref(a)) == want
