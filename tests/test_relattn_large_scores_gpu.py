"""Rows whose scores are large in magnitude: every probability still belongs to a distribution (the rows' sum is one), forward and backward.

The softmax does not see a number added to every entry of the table.  The inputs are made so that fp32 does not either: queries and keys hold
0, +-s, and table = shift + small, with s^2 and small / scale multiples of the spacing of fp32 numbers at shift / scale, so that scale q.k + table
is exact.  The oracle then takes `small` alone, and its bounds (tests/seq_ref.py) hold: what the shift leaves in an exponent is one rounding
per row, which the row's sum takes out again, plus roundings of differences of scores (2^-24 of less than 2^7, where the oracle's e allows (D + 8) 2^-24 of as much)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import seq_ref as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _cu(lens, dev):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=dev)


# shift, size of a query's and key's elements, step of the table's entries, range of those steps
SHIFTS = [(1e6, 1, 0.0625, 16), (-1e6, 1, 0.0625, 16), (5e7, 8, 4.0, 2), (-5e7, 8, 4.0, 2), (-9e7, 8, 8.0, 1), (-1e9, 8, 0.0, 1)]
SHAPES = [
    # lens, H, Hkv, D, buckets, far, causal
    ([50], 2, 2, 64, 32, 128, False),
    ([200, 3, 64], 4, 2, 64, 16, 40, True),
    ([300, 33], 2, 1, 128, 8, 20, False),                     # most tiles behind the last border, on both sides
    ([150, 70], 2, 1, 128, 8, 20, True),
    ([130], 2, 2, 96, 8, 20, False),
    ([40, 100], 2, 2, 32, 8, 20, True),
]


def _both(K, geom, q, k, v, table, cu, do, ref, frozen, what):
    o, lse = K.relattn_fwd(geom, q, k, v, table, cu)
    R.within(o, ref["o"], what + " o", 1e-6)
    got = K.relattn_bwd(geom, q, k, v, table, cu, None, o, lse, do)
    for name, g in zip(("dv", "dq", "dk", "dtable"), (got[2], got[0], got[1], got[3])):
        R.within(g, ref[name], f"{what} {name}", 1e-6)
    got = K.relattn_bwd(geom, q, k, v, table, cu, None, o, lse, do, want_table=False)
    for name, g in zip(("dv", "dq", "dk"), (got[2], got[0], got[1])):
        R.within(g, frozen[name], f"{what} {name} (frozen table)", 1e-6)


@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("shift", range(len(SHIFTS)))
def test_a_shift_of_every_entry(stg, gpu, shift, shape):
    from stgcma import kernels as K
    base, s, step, most = SHIFTS[shift]
    lens, H, Hkv, D, nb, far, causal = SHAPES[shape]
    n = sum(lens)
    g = torch.Generator(device=gpu)
    g.manual_seed(700 + 10 * shift + shape)
    ints = lambda lo, hi, *size: torch.randint(lo, hi + 1, size, generator=g, device=gpu).float()
    few = (torch.rand(n, H * D, generator=g, device=gpu) < 4.0 / D).float()              # about four elements to a query's head
    q, k = (s * few * ints(-1, 1, n, H * D)).to(BF16), (s * ints(-1, 1, n, Hkv * D)).to(BF16)
    v = torch.randn(n, Hkv * D, generator=g, device=gpu).to(BF16)
    small = step * ints(-most, most, nb, H)
    table = (small.double() + base).float()
    assert torch.equal(table.double() - base, small.double()) or base == -1e9
    geom = K.RelGeom(H, D, kv_heads=Hkv, num_buckets=nb, max_distance=far, causal=causal, scale=0.125, device=gpu)
    for do in (torch.ones(n, H * D, dtype=BF16, device=gpu), torch.randn(n, H * D, generator=g, device=gpu).to(BF16)):
        refs = [R.attention(q, k, v, small, lens, lens, H, Hkv, D, nb, far, causal, 0.125, None, do, table_grad=t) for t in (True, False)]
        _both(K, geom, q, k, v, table, _cu(lens, gpu), do, *refs, f"shift {base:g}")


@pytest.mark.parametrize("D", [64, 128])
def test_first_causal_rows_in_a_hidden_bucket(stg, gpu, D):
    """The bucket of distance 0 at -1e9: the first row of a causal sequence sees nothing else, every other row sees everything but itself.  (For the oracle
    the entry is -60: e^-60 is far below every bound.)"""
    from stgcma import kernels as K
    lens, H, Hkv, nb, far = [150, 1, 40], 4, 2, 16, 40
    n = sum(lens)
    g = torch.Generator(device=gpu)
    g.manual_seed(790)
    rn = lambda *size: torch.randn(*size, generator=g, device=gpu)
    q, k, v, do = (rn(n, h * D).to(BF16) for h in (H, Hkv, Hkv, H))
    table = rn(nb, H)
    table[0] = -1e9
    oracle = table.clone()
    oracle[0] = -60.0
    geom = K.RelGeom(H, D, kv_heads=Hkv, num_buckets=nb, max_distance=far, causal=True, device=gpu)
    refs = [R.attention(q, k, v, oracle, lens, lens, H, Hkv, D, nb, far, True, D ** -0.5, None, do, table_grad=t) for t in (True, False)]
    _both(K, geom, q, k, v, table, _cu(lens, gpu), do, *refs, "hidden diagonal")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("base", [-9e7, 1e6])
def test_a_shift_with_masks_and_unequal_lengths(stg, gpu, base, causal):
    """The same with masked keys, more keys than queries or fewer, a sequence without a visible key, and rows behind the last one."""
    from stgcma import kernels as K
    lens_q, lens_k, H, Hkv, D, nb, far = [70, 130, 5, 200, 33], [200, 60, 90, 200, 33], 4, 2, 64, 8, 20
    s, step, most = (8, 8.0, 1) if base == -9e7 else (1, 0.0625, 16)
    g = torch.Generator(device=gpu)
    g.manual_seed(771)
    ints = lambda lo, hi, *size: torch.randint(lo, hi + 1, size, generator=g, device=gpu).float()
    nq, nk = sum(lens_q) + 3, sum(lens_k) + 3
    few = (torch.rand(nq, H * D, generator=g, device=gpu) < 4.0 / D).float()
    q, k = (s * few * ints(-1, 1, nq, H * D)).to(BF16), (s * ints(-1, 1, nk, Hkv * D)).to(BF16)
    v, do = torch.randn(nk, Hkv * D, generator=g, device=gpu).to(BF16), torch.randn(nq, H * D, generator=g, device=gpu).to(BF16)
    mask = torch.rand(nk, generator=g, device=gpu) >= 0.4
    mask[sum(lens_k[:4]):] = False
    small = step * ints(-most, most, nb, H)
    table = (small.double() + base).float()
    geom = K.RelGeom(H, D, kv_heads=Hkv, num_buckets=nb, max_distance=far, causal=causal, scale=0.125, device=gpu)
    cu_q, cu_k = _cu(lens_q, gpu), _cu(lens_k, gpu)
    ref = R.attention(q, k, v, small, lens_q, lens_k, H, Hkv, D, nb, far, causal, 0.125, mask, do)
    o, lse = K.relattn_fwd(geom, q, k, v, table, cu_q, cu_k, key_mask=mask)
    R.within(o, ref["o"], "o", 1e-6)
    for hint in (None, 64):
        got = K.relattn_bwd(geom, q, k, v, table, cu_q, cu_k, o, lse, do, key_mask=mask, max_q=hint, max_k=hint)
        for name, t in zip(("dq", "dk", "dv", "dtable"), got):
            R.within(t, ref[name], name, 1e-6)


def test_many_short_sequences_and_one_long_with_a_shift(stg, gpu):
    """Fewer blocks than tiles (20 000 sequences without a length hint): a block that strides over tiles keeps account of rows far out in any of them."""
    from stgcma import kernels as K
    S, H, Hkv, D, nb, far = 20000, 2, 1, 32, 8, 20
    lens = [0] * S
    lens[17], lens[4000], lens[19998] = 33, 1500, 129
    n = sum(lens)
    g = torch.Generator(device=gpu)
    g.manual_seed(772)
    ints = lambda lo, hi, *size: torch.randint(lo, hi + 1, size, generator=g, device=gpu).float()
    few = (torch.rand(n, H * D, generator=g, device=gpu) < 4.0 / D).float()
    q, k = (few * ints(-1, 1, n, H * D)).to(BF16), ints(-1, 1, n, Hkv * D).to(BF16)
    v, do = torch.randn(n, Hkv * D, generator=g, device=gpu).to(BF16), torch.randn(n, H * D, generator=g, device=gpu).to(BF16)
    small = 0.0625 * ints(-16, 16, nb, H)
    table = (small.double() - 1e6).float()
    for causal in (False, True):
        geom = K.RelGeom(H, D, kv_heads=Hkv, num_buckets=nb, max_distance=far, causal=causal, scale=0.125, device=gpu)
        ref = R.attention(q, k, v, small, lens, lens, H, Hkv, D, nb, far, causal, 0.125, None, do)
        o, lse = K.relattn_fwd(geom, q, k, v, table, _cu(lens, gpu))
        for name, t in zip(("dq", "dk", "dv", "dtable"), K.relattn_bwd(geom, q, k, v, table, _cu(lens, gpu), None, o, lse, do)):
            R.within(t, ref[name], name, 1e-6)


def test_a_replayed_graph_between_large_and_ordinary_scores(stg, gpu):
    """Inputs that need the rows' sums and inputs that do not take turns in one graph: every replay gives the eager bits."""
    from stgcma import kernels as K
    lens, H, Hkv, D = [150, 41], 4, 2, 64
    n = sum(lens)
    g = torch.Generator(device=gpu)
    g.manual_seed(773)
    rn = lambda *size: torch.randn(*size, generator=g, device=gpu)
    geom = K.RelGeom(H, D, kv_heads=Hkv, causal=True, device=gpu)
    cu = _cu(lens, gpu)
    sets = [[rn(n, h * D).to(BF16) for h in (H, Hkv, Hkv, H)] + [rn(32, H) + shift] for shift in (0.0, -3e5, 7e7)]

    def step(q, k, v, do, table):
        o, lse = K.relattn_fwd(geom, q, k, v, table, cu, max_q=150)
        return (o, lse) + K.relattn_bwd(geom, q, k, v, table, cu, None, o, lse, do, max_q=150)
    want = [step(*s) for s in sets]
    buf = [t.clone() for t in sets[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*buf)
    for i in (1, 0, 2, 0, 1, 2, 0):
        for b, s in zip(buf, sets[i]):
            b.copy_(s)
        graph.replay()
        _ = step(*sets[(i + 1) % 3])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))
