"""The join's column sums (gradients of weights, biases and gate)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


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
