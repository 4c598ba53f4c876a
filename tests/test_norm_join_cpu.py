"""The size of the join's gradient buffer."""
import ctypes as C

import pytest


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
