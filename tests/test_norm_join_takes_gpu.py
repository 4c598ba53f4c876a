"""What the join takes: single rows of wide buffers, a gate of one value at any element of a buffer."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_norm_join_gpu import _make

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
LEAVES = ("x", "h", "gate", "w1", "b1", "w2", "b2")


def test_single_rows_of_wide_buffers(stg, gpu):
    """One row has no leading dimension to be misaligned, in the backward either."""
    from stgcma import kernels as K, ops_seq
    t = _make(gpu, 1, 96, "layer", F32, "channel", None, True, True, 550)
    odd = dict(t)
    for n, v in (("x", t["x"]), ("h", t["h"]), ("dy", t["dy"]), ("dxn", t["dxn"])):
        wide = torch.zeros(1, 101, dtype=v.dtype, device=gpu)
        wide[:, :96] = v
        odd[n] = wide[:, :96]
    outs = []
    for s in (t, odd):
        leaf = [s[n].detach().requires_grad_(True) for n in LEAVES]
        xn, y = ops_seq.norm_join(*leaf)
        outs.append([xn.detach(), y.detach()] + list(torch.autograd.grad([xn, y], leaf, [s["dxn"], s["dy"]])))
        xn, y, st = K.norm_join_fwd(*[s[n] for n in LEAVES])
        if s is odd:
            wide = torch.zeros(1, 101, device=gpu)
            wide[:, :96] = xn
            xn = wide[:, :96]
        outs[-1] += list(K.norm_join_bwd(xn, *[s[n] for n in LEAVES[1:]], st, s["dy"], s["dxn"]).values())
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_single_gate_anywhere_in_a_buffer(stg, gpu):
    """A gate of one value is read as one value: a view into a flat buffer of parameters at any element."""
    from stgcma import ops_seq
    t = _make(gpu, 70, 96, "layer", F32, "one", None, True, True, 540)
    flat = torch.randn(9, device=gpu)
    outs = []
    for i in range(4):
        flat[i:i + 1] = t["gate"]
        for g in (flat[i:i + 1], flat[i]):
            leaf = [(g if n == "gate" else t[n]).detach().requires_grad_(True) for n in LEAVES]
            xn, y = ops_seq.norm_join(*leaf)
            grads = torch.autograd.grad([xn, y], leaf, [t["dxn"], t["dy"]])
            assert grads[2].shape == g.shape
            outs.append([xn.detach(), y.detach()] + [v.reshape(-1) for v in grads])
    assert all(torch.equal(a, b) for o in outs[1:] for a, b in zip(outs[0], o))
