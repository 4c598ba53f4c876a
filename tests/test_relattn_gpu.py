"""Attention over ragged sequences with a learned relative position bias by buckets, on the GPU, against 64-bit references (tests/seq_ref.py derives
the bounds): lengths from nothing to several tiles, grouped heads, masks that leave a row empty, strides, refused calls, streams and graphs."""
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


def _make(gpu, lens_q, lens_k, H, Hkv, D, buckets, seed, tail=0, fused=True):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    rn = lambda *s, dtype=BF16: torch.randn(*s, generator=g, device=gpu, dtype=F32).to(dtype)
    Tq, Tk = sum(lens_q) + tail, sum(lens_k) + tail
    if fused and lens_q == lens_k:
        qkv = rn(Tq, (H + 2 * Hkv) * D)
        q, k, v = qkv[:, :H * D], qkv[:, H * D:(H + Hkv) * D], qkv[:, (H + Hkv) * D:]
    else:
        q, k, v = rn(Tq, H * D), rn(Tk, Hkv * D), rn(Tk, Hkv * D)
    return q, k, v, rn(buckets, H, dtype=F32), rn(Tq, H * D)


CASES = [
    # lens_q, lens_k (None: the same), H, Hkv, D, buckets, far, causal, mask, tail
    ([1], None, 1, 1, 32, 4, 2, False, None, 0),
    ([1], None, 2, 1, 64, 2, 2, True, None, 0),
    ([3, 14, 7, 11], None, 8, 8, 64, 32, 128, False, None, 0),
    ([31, 32, 33, 0, 63, 64, 65, 1], None, 4, 2, 32, 16, 40, False, None, 5),
    ([127, 128, 129], None, 3, 3, 96, 12, 100, False, "random", 0),
    ([127, 5, 193], None, 6, 2, 128, 32, 128, True, None, 0),
    ([300], None, 2, 2, 64, 8, 20, False, None, 3),                   # most tiles behind the last border
    ([257, 70], None, 4, 1, 64, 64, 800, True, "random", 0),
    ([40, 90, 17], None, 4, 4, 64, 32, 128, False, "last", 0),           # a sequence without a key
    ([40, 90, 17], None, 7, 1, 32, 32, 128, True, "first", 2),           # causal rows before the first visible key are empty
    ([5, 64, 100], [70, 64, 130], 4, 2, 64, 16, 40, False, None, 0),     # queries at the end of a longer key sequence
    ([1, 130, 3, 9], [200, 100, 0, 1], 4, 4, 96, 16, 40, True, None, 0),  # more queries than keys: the first see nothing; no key at all
    ([700], None, 1, 1, 128, 32, 128, False, None, 0),
    ([0, 0, 2], None, 2, 2, 64, 32, 128, False, None, 1),
]


def _mask(kind, lens, gpu, seed, tail):
    n = sum(lens) + tail
    if kind is None:
        return None
    g = torch.Generator(device=gpu)
    g.manual_seed(seed + 1)
    m = torch.rand(n, generator=g, device=gpu) >= 0.3
    if kind == "last":
        m[sum(lens[:-1]):] = False
    if kind == "first":
        at = 0
        for x in lens:
            m[at:at + x // 3] = False
            at += x
    return m


@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward_and_gradients(stg, gpu, case):
    from stgcma import kernels as K, ops_seq
    lens_q, lens_k, H, Hkv, D, nb, far, causal, mk, tail = CASES[case]
    lens_k = lens_q if lens_k is None else lens_k
    q, k, v, table, do = _make(gpu, lens_q, lens_k, H, Hkv, D, nb, 100 + case, tail)
    mask = _mask(mk, lens_k, gpu, case, tail)
    geom = K.RelGeom(H, D, kv_heads=Hkv, num_buckets=nb, max_distance=far, causal=causal, device=gpu)
    cu_q = _cu(lens_q, gpu)
    cu_k = None if lens_k == lens_q else _cu(lens_k, gpu)
    ref = R.attention(q, k, v, table, lens_q, lens_k, H, Hkv, D, nb, far, causal, D ** -0.5, mask, do)
    o, lse = K.relattn_fwd(geom, q, k, v, table, cu_q, cu_k, max_q=max(lens_q), max_k=max(lens_k), key_mask=mask)
    R.within(o, ref["o"], "o")
    R.within(lse, ref["lse"], "lse", 1e-6)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    o2 = ops_seq.rel_attention(*leaves, geom, cu_q, cu_k, max_q=max(lens_q), max_k=max(lens_k), key_mask=mask)
    R.within(o2, ref["o"], "o (training)")
    for name, g in zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(o2, leaves, do)):
        R.within(g, ref[name], name, 1e-6)
    # frozen table: delta from the rounded o alone
    o3 = ops_seq.rel_attention(*leaves[:3], table, geom, cu_q, cu_k, key_mask=mask)          # (and no length hint)
    assert torch.equal(o3, o)
    ref = R.attention(q, k, v, table, lens_q, lens_k, H, Hkv, D, nb, far, causal, D ** -0.5, mask, do, table_grad=False)
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o3, leaves[:3], do)):
        R.within(g, ref[name], name + " (frozen table)", 1e-6)


@pytest.mark.parametrize("causal", [False, True])
def test_table_gradient_against_differences(stg, gpu, causal):
    """<dtable, direction> against a central difference of the 64-bit forward: the difference's own error is h^2 / 6 of a third derivative that
    softmax bounds by ~10 sum |do o|-sized terms; with h = 1e-4 it stays far below the gradient's bound, which is what is asserted."""
    from stgcma import kernels as K, ops_seq
    lens, H, Hkv, D, nb, far = [50, 97], 4, 2, 64, 16, 40
    q, k, v, table, do = _make(gpu, lens, lens, H, Hkv, D, nb, 7)
    geom = K.RelGeom(H, D, kv_heads=Hkv, num_buckets=nb, max_distance=far, causal=causal, device=gpu)
    t = table.detach().requires_grad_(True)
    o = ops_seq.rel_attention(q, k, v, t, geom, _cu(lens, gpu), max_q=97)
    (dt,) = torch.autograd.grad(o, [t], do)
    way = torch.randn(table.shape, generator=torch.Generator().manual_seed(3)).to(gpu).double()
    ref = R.attention(q, k, v, table, lens, lens, H, Hkv, D, nb, far, causal, D ** -0.5, None, do)

    def loss(s):
        r = R.attention(q, k, v, table.double() + s * way, lens, lens, H, Hkv, D, nb, far, causal, D ** -0.5)
        return (r["o"][0] * do.double()).sum()
    h = 1e-4
    diff = float((loss(h) - loss(-h)) / (2 * h))
    got = float((dt.double() * way).sum())
    bound = float((ref["dtable"][1] * way.abs()).sum())
    assert abs(got - diff) <= bound + 1e-5 * float(ref["o"][0].abs().mul(do.double().abs()).sum()), (got, diff, bound)


def test_rows_outside_and_masked_rows_are_not_read(stg, gpu):
    """NaN and infinities behind the last sequence, in masked keys and around the tensors' columns leave no trace, and a given output keeps its rows."""
    from stgcma import kernels as K
    lens, H, Hkv, D = [70, 33], 4, 2, 64
    q, k, v, table, do = _make(gpu, lens, lens, H, Hkv, D, 32, 5, tail=9)
    mask = _mask("random", lens, gpu, 3, 9)
    geom = K.RelGeom(H, D, kv_heads=Hkv, device=gpu)
    cu = _cu(lens, gpu)
    o, lse = K.relattn_fwd(geom, q, k, v, table, cu, max_q=70, key_mask=mask)
    g0 = K.relattn_bwd(geom, q, k, v, table, cu, None, o, lse, do, max_q=70, key_mask=mask)
    bad = ~mask
    bad[103:] = True
    q2, k2, v2, do2 = q.clone(), k.clone(), v.clone(), do.clone()
    k2[bad], v2[bad] = float("nan"), float("inf")
    q2[103:], do2[103:] = float("nan"), float("nan")
    mine = torch.full_like(o, 7.0)
    o2, lse2 = K.relattn_fwd(geom, q2, k2, v2, table, cu, max_q=70, key_mask=mask, out=mine)
    assert o2 is mine and torch.equal(o2[:103], o[:103]) and bool((o2[103:] == 7.0).all()) and torch.equal(lse2[:, :103], lse[:, :103])
    assert bool((o[103:] == 0).all())
    o3 = o.clone()
    o3[103:] = float("nan")
    g1 = K.relattn_bwd(geom, q2, k2, v2, table, cu, None, o3, lse, do2, max_q=70, key_mask=mask)
    for a, b in zip(g0, g1):
        assert torch.equal(a, b)
    assert all(bool((t[103:] == 0).all()) for t in g1[:3])
    assert bool((g1[1][bad] == 0).all()) and bool((g1[2][bad] == 0).all())


def test_lowest_and_infinite_bias_entries(stg, gpu):
    """-inf in the table hides its distances, and so does any entry at or below -1e30 (a mask by the type's lowest value): a query with nothing else is an
    empty row with no gradient; very large finite entries stay scores."""
    from stgcma import kernels as K
    n, H, D = 40, 2, 64
    q, k, v, table, do = _make(gpu, [n], [n], H, H, D, 8, 11)
    geom = K.RelGeom(H, D, num_buckets=8, max_distance=16, device=gpu)
    cu = _cu([n], gpu)
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    for scale in (D ** -0.5, 1.0, 4.0):
        geom.scale = scale
        for low in (torch.finfo(F32).min, -1e30, -float("inf")):
            hidden = torch.full_like(table, low)
            o, lse = K.relattn_fwd(geom, q, k, v, hidden, cu)
            assert bool((o == 0).all()) and bool((lse == -float("inf")).all())
            assert all(bool((t == 0).all()) for t in K.relattn_bwd(geom, q, k, v, hidden, cu, None, o, lse, do))
            assert bool((K.relattn_decode(geom, q[:1], k[None], v[None], hidden, lens) == 0).all())
        for shift in (-5e7, 5e7):                              # one number added to every entry: the same probabilities, up to the fp32 sum
            o, _ = K.relattn_fwd(geom, q, k, v, torch.full_like(table, shift), cu)
            assert bool(torch.isfinite(o).all()) and float(o.double().abs().max()) <= float(v.double().abs().max()) * (1 + 2.0 ** -7)
    geom.scale = D ** -0.5
    t2 = table.clone()
    t2[4:] = -float("inf")                                    # every key behind the query is hidden: the causal rule by the bias alone
    o, lse = K.relattn_fwd(geom, q, k, v, t2, cu)
    x = torch.einsum("qhd,khd->hqk", q.double().view(n, H, D), k.double().view(n, H, D)) * D ** -0.5
    rel = torch.arange(n, device=gpu)[None] - torch.arange(n, device=gpu)[:, None]
    ids = torch.tensor([[geom.bucket(int(r)) for r in row] for row in rel.cpu()], device=gpu)
    x = x + t2.double().t()[:, ids]
    assert bool(torch.isinf(x[:, rel > 0]).all())
    p = torch.softmax(x, -1)
    want = torch.einsum("hqk,khd->qhd", p, v.double().view(n, H, D)).reshape(n, H * D)
    size = torch.einsum("hqk,khd->qhd", p, v.double().abs().view(n, H, D)).reshape(n, H * D)
    assert bool(((o.double() - want).abs() <= 2.0 ** -8 * (want.abs() + 1.1 * size)).all())


def test_same_call_same_bits_and_length_hints(stg, gpu):
    from stgcma import kernels as K
    lens, H, Hkv, D = [200, 1, 333, 64], 8, 2, 64
    q, k, v, table, do = _make(gpu, lens, lens, H, Hkv, D, 32, 21)
    for causal in (False, True):
        geom = K.RelGeom(H, D, kv_heads=Hkv, causal=causal, device=gpu)
        cu = _cu(lens, gpu)
        first = None
        for hint in (333, 333, 333, 64, 1, None, 10 ** 6):        # a hint below the longest still computes every row
            o, lse = K.relattn_fwd(geom, q, k, v, table, cu, max_q=hint)
            dq, dk, dv, dt = K.relattn_bwd(geom, q, k, v, table, cu, None, o, lse, do, max_q=hint)
            if first is None:
                first = (o, lse, dq, dk, dv, dt)
                continue
            for a, b in zip(first[:5], (o, lse, dq, dk, dv)):
                assert torch.equal(a, b)
            if hint == 333:
                assert torch.equal(first[5], dt)
            else:                                              # other blocks, another order of the fp32 sums
                assert float((first[5] - dt).abs().max()) <= 1e-4 * float(first[5].abs().max())


def test_bad_offsets_stay_inside(stg, gpu):
    """Offsets that decrease, are negative or pass the tensors' ends are clamped: the calls return and write nothing outside."""
    from stgcma import kernels as K
    H, D, n = 2, 64, 100
    q, k, v, table, do = _make(gpu, [n], [n], H, H, D, 32, 31)
    geom = K.RelGeom(H, D, device=gpu)
    guard = torch.full((n + 64, H * D), 3.0, dtype=BF16, device=gpu)
    for offs in ([0, 60, 40, 100], [-5, 50, 100], [0, 30, 10 ** 9], [0, -1, 100], [7, 100]):
        cu = torch.tensor(offs, dtype=torch.int32, device=gpu)
        o, lse = K.relattn_fwd(geom, q, k, v, table, cu, out=guard[:n])
        K.relattn_bwd(geom, q, k, v, table, cu, None, o, lse, do)
        torch.cuda.synchronize()
        assert bool((guard[n:] == 3.0).all())
    cu = _cu([n], gpu)
    want = K.relattn_fwd(geom, q, k, v, table, cu)[0]
    assert torch.equal(K.relattn_fwd(geom, q, k, v, table, torch.tensor([7, 10 ** 9], dtype=torch.int32, device=gpu))[0], want)


def test_capture_and_streams(stg, gpu):
    """Forward and backward in one graph, replayed with new inputs between eager work, and on a side stream, give the eager bits."""
    from stgcma import kernels as K, ops_seq
    lens, H, Hkv, D = [90, 41], 4, 2, 64
    geom = K.RelGeom(H, D, kv_heads=Hkv, device=gpu)
    cu = _cu(lens, gpu)
    sets = [_make(gpu, lens, lens, H, Hkv, D, 32, 40 + i) for i in range(3)]

    def step(q, k, v, table, do):
        a = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
        o = ops_seq.rel_attention(*a, geom, cu, max_q=90)
        return (o.detach(),) + torch.autograd.grad(o, a, do)
    want = [step(*s) for s in sets]
    buf = [t.clone() for t in sets[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = step(*buf)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*buf)
    for i in (1, 2, 0, 2):
        for b, s in zip(buf, sets[i]):
            b.copy_(s)
        graph.replay()
        _ = step(*sets[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


DECODE = [
    # lens, cap, H, Hkv, D, buckets, far, causal table
    ([1], 1, 1, 1, 64, 32, 128, True),
    ([701], 701, 12, 12, 64, 32, 128, True),
    ([0, 1, 31, 32, 33, 127, 128, 129, 500], 512, 8, 2, 128, 32, 128, True),
    ([1000, 0, 3], 1024, 7, 1, 32, 16, 40, True),
    ([260, 90], 300, 40, 1, 96, 64, 800, True),              # more query heads to a group than an MFMA tile has columns
    ([3000, 2999, 17, 1500], 3000, 16, 4, 96, 12, 100, False),   # the table of a two-sided model
]


@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode(stg, gpu, case):
    from stgcma import kernels as K
    lens, cap, H, Hkv, D, nb, far, causal = DECODE[case]
    S = len(lens)
    g = torch.Generator(device=gpu)
    g.manual_seed(200 + case)
    rn = lambda *s, dtype=BF16: torch.randn(*s, generator=g, device=gpu, dtype=F32).to(dtype)
    q, kv, table = rn(S, H * D), rn(S, cap + 3, 2 * Hkv * D), rn(nb, H, dtype=F32)
    kc, vc = kv[:, 1:cap + 1, :Hkv * D], kv[:, 1:cap + 1, Hkv * D:]     # slices of one larger cache
    geom = K.RelGeom(H, D, kv_heads=Hkv, num_buckets=nb, max_distance=far, causal=causal, device=gpu)
    o = K.relattn_decode(geom, q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=gpu))
    flat = lambda c: torch.cat([c[s, :n] for s, n in enumerate(lens)])
    live = [s for s, n in enumerate(lens) if n]
    ref = R.attention(q[live], flat(kc), flat(vc), table, [1] * len(live), [n for n in lens if n], H, Hkv, D, nb, far, causal, D ** -0.5)
    R.within(o[live], ref["o"], "o", 1e-6)
    for s, n in enumerate(lens):
        if n == 0:
            assert bool((o[s] == 0).all())
        kc[s, n:] = float("nan")                               # what stands behind a sequence's end is not read
        vc[s, n:] = float("inf")
    again = K.relattn_decode(geom, q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=gpu))
    assert torch.equal(o, again)
    over = K.relattn_decode(geom, q, kc[:, :1], vc[:, :1], table, torch.tensor([10 ** 9] * S, dtype=torch.int32, device=gpu))   # clamped to the capacity
    one = K.relattn_decode(geom, q, kc[:, :1], vc[:, :1], table, torch.ones(S, dtype=torch.int32, device=gpu))
    assert torch.equal(torch.nan_to_num(over, 9.0, 9.0, 9.0), torch.nan_to_num(one, 9.0, 9.0, 9.0))


def test_decode_equals_last_row_of_forward(stg, gpu):
    """A sequence decoded token by token gives the causal forward's rows (each within its own bound of the common value: twice the rounding)."""
    from stgcma import kernels as K
    n, H, Hkv, D = 150, 8, 2, 64
    q, k, v, table, _ = _make(gpu, [n], [n], H, Hkv, D, 32, 77, fused=False)
    geom = K.RelGeom(H, D, kv_heads=Hkv, causal=True, device=gpu)
    o, _ = K.relattn_fwd(geom, q, k, v, table, _cu([n], gpu))
    ref = R.attention(q, k, v, table, [n], [n], H, Hkv, D, 32, 128, True, D ** -0.5)["o"]
    kc, vc = torch.zeros_like(k)[None], torch.zeros_like(v)[None]
    lens = torch.zeros(1, dtype=torch.int32, device=gpu)
    rows = []
    for t in range(n):
        kc[0, t], vc[0, t] = k[t], v[t]
        lens += 1
        rows.append(K.relattn_decode(geom, q[t:t + 1], kc, vc, table, lens))
    R.within(torch.cat(rows), ref, "decoded", 1e-6)
    R.within(o, ref, "forward", 1e-6)


def test_decode_capture(stg, gpu):
    from stgcma import kernels as K
    S, cap, H, Hkv, D = 3, 600, 8, 2, 64
    g = torch.Generator(device=gpu)
    g.manual_seed(5)
    rn = lambda *s: torch.randn(*s, generator=g, device=gpu, dtype=F32).to(BF16)
    geom = K.RelGeom(H, D, kv_heads=Hkv, causal=True, device=gpu)
    q, kc, vc, table = rn(S, H * D), rn(S, cap, Hkv * D), rn(S, cap, Hkv * D), rn(32, H).float()
    lens = torch.tensor([600, 20, 333], dtype=torch.int32, device=gpu)
    K.relattn_decode(geom, q, kc, vc, table, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.relattn_decode(geom, q, kc, vc, table, lens)
    for new in ([1, 2, 3], [600, 600, 600], [599, 0, 128]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        q.copy_(rn(S, H * D))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, K.relattn_decode(geom, q, kc, vc, table, lens))


def _all(K, geom, q, k, v, table, cu_q, cu_k, do, **kw):
    """Forward and every gradient through the direct calls."""
    o, lse = K.relattn_fwd(geom, q, k, v, table, cu_q, cu_k, **kw)
    return (o, lse) + K.relattn_bwd(geom, q, k, v, table, cu_q, cu_k, o, lse, do, **kw)


@pytest.mark.parametrize("causal", [False, True])
def test_empty_tensors(stg, gpu, causal):
    from stgcma import kernels as K
    H, Hkv, D = 4, 2, 64
    geom = K.RelGeom(H, D, kv_heads=Hkv, causal=causal, device=gpu)
    table = torch.randn(32, H, device=gpu)
    e = lambda n, h: torch.randn(n, h * D, device=gpu).to(BF16)
    for tq, tk, offs_q, offs_k in ((0, 0, [0, 0], None), (5, 5, [0], None), (4, 0, [0, 4], [0, 0]), (0, 6, [0, 0], [0, 6]), (0, 0, [0], None)):
        cu_q = torch.tensor(offs_q, dtype=torch.int32, device=gpu)
        cu_k = None if offs_k is None else torch.tensor(offs_k, dtype=torch.int32, device=gpu)
        got = _all(K, geom, e(tq, H), e(tk, Hkv), e(tk, Hkv), table, cu_q, cu_k, e(tq, H))
        assert [tuple(t.shape) for t in got] == [(tq, H * D), (H, tq), (tq, H * D), (tk, Hkv * D), (tk, Hkv * D), (32, H)]
        assert all(bool((t == 0).all()) for i, t in enumerate(got) if i != 1) and bool((got[1] == -float("inf")).all())
    none = K.relattn_decode(geom, e(3, H), e(3, Hkv).view(3, 1, -1)[:, :0], e(3, Hkv).view(3, 1, -1)[:, :0], table, torch.ones(3, dtype=torch.int32, device=gpu))
    assert bool((none == 0).all())
    assert K.relattn_decode(geom, e(0, H), e(0, Hkv).view(0, 1, Hkv * D), e(0, Hkv).view(0, 1, Hkv * D), table, torch.ones(0, dtype=torch.int32, device=gpu)).shape == (0, H * D)


@pytest.mark.parametrize("causal", [False, True])
def test_offsets_beyond_32_bits(stg, gpu, causal):
    """Rows 2^24 elements apart: the last of 200 stands 3.3 * 10^9 elements behind the first, and everything equals the dense call."""
    from stgcma import kernels as K
    n, H, D = 200, 2, 64
    q, k, v, table, do = _make(gpu, [n], [n], H, H, D, 32, 61)
    geom = K.RelGeom(H, D, causal=causal, device=gpu)
    big = torch.empty(n, 1 << 24, dtype=BF16, device=gpu)
    wide = [big[:, i * H * D:(i + 1) * H * D] for i in range(4)]
    for w, t in zip(wide, (q, k, v, do)):
        w.copy_(t)
    cu = _cu([n], gpu)
    want, got = (_all(K, geom, a, b, c, table, cu, None, d) for a, b, c, d in ((q, k, v, do), wide))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    assert torch.equal(K.relattn_decode(geom, q[:1], k[None], v[None], table, lens), K.relattn_decode(geom, q[:1], wide[1][None], wide[2][None], table, lens))
    two = big.view(2, n // 2, 1 << 24)                          # sequences 1.7 * 10^9 elements apart
    lens = torch.tensor([n // 2, 37], dtype=torch.int32, device=gpu)
    dense = [t.reshape(2, n // 2, H * D) for t in (k, v)]
    assert torch.equal(K.relattn_decode(geom, q[:2], *dense, table, lens), K.relattn_decode(geom, q[:2], two[:, :, H * D:2 * H * D], two[:, :, 2 * H * D:3 * H * D], table, lens))


MORE = [
    # lens_q, lens_k, H, Hkv, D, buckets, far, causal, mask
    ([130, 3, 64], [40, 200, 0], 2, 1, 64, 32, 128, False, None),        # more queries than keys without the causal rule
    ([2300], [2300], 1, 1, 128, 256, 2048, True, None),                  # the widest table and LDS arrays
    ([2300], [2300], 1, 1, 128, 256, 2048, False, "random"),
    ([2100, 1], [2101, 300], 2, 2, 32, 250, 2040, False, None),
    ([400, 129], [400, 129], 65, 5, 32, 4, 3, True, None),               # many heads, thirteen to a group
    ([513], [513], 2, 2, 96, 32, 128, True, "first"),
]


@pytest.mark.parametrize("case", range(len(MORE)))
def test_wide_tables_and_lengths(stg, gpu, case):
    from stgcma import kernels as K
    lens_q, lens_k, H, Hkv, D, nb, far, causal, mk = MORE[case]
    q, k, v, table, do = _make(gpu, lens_q, lens_k, H, Hkv, D, nb, 400 + case, fused=False)
    mask = _mask(mk, lens_k, gpu, case, 0)
    geom = K.RelGeom(H, D, kv_heads=Hkv, num_buckets=nb, max_distance=far, causal=causal, device=gpu)
    ref = R.attention(q, k, v, table, lens_q, lens_k, H, Hkv, D, nb, far, causal, D ** -0.5, mask, do)
    got = _all(K, geom, q, k, v, table, _cu(lens_q, gpu), _cu(lens_k, gpu), do, max_q=max(lens_q), max_k=max(lens_k), key_mask=mask)
    for name, t in zip(("o", "lse", "dq", "dk", "dv", "dtable"), got):
        R.within(t, ref[name], name, 1e-6)


@pytest.mark.parametrize("Hkv", [2, 1])
@pytest.mark.parametrize("causal", [False, True])
def test_many_sequences_without_a_hint(stg, gpu, causal, Hkv):
    """20 000 sequences, nearly all empty, one of 1500 rows: fewer blocks than the longest sequence has tiles, each striding over several; a shared head's
    query heads stay in one block (elsewhere in this file they are split over several)."""
    from stgcma import kernels as K
    S, H, D = 20000, 2, 32
    lens = [0] * S
    lens[17], lens[4000], lens[4001], lens[19998] = 33, 1500, 700, 129
    q, k, v, table, do = _make(gpu, lens, lens, H, Hkv, D, 32, 71, tail=3)
    geom = K.RelGeom(H, D, kv_heads=Hkv, causal=causal, device=gpu)
    ref = R.attention(q, k, v, table, lens, lens, H, Hkv, D, 32, 128, causal, D ** -0.5, None, do)
    got = _all(K, geom, q, k, v, table, _cu(lens, gpu), None, do)
    for name, t in zip(("o", "lse", "dq", "dk", "dv", "dtable"), got):
        R.within(t, ref[name], name, 1e-6)


def test_autograd_corners(stg, gpu):
    """Saved tensors that hooks move and pack densely, single wanted gradients, a strided incoming gradient, and no second derivative."""
    from stgcma import kernels as K, ops_seq
    lens, H, Hkv, D = [70, 41], 4, 2, 64
    q, k, v, table, do = _make(gpu, lens, lens, H, Hkv, D, 32, 81)
    geom = K.RelGeom(H, D, kv_heads=Hkv, device=gpu)
    cu, mask = _cu(lens, gpu), _mask("random", lens, gpu, 2, 0)
    run = lambda *a: ops_seq.rel_attention(*a, geom, cu, max_q=70, key_mask=mask)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
    want = torch.autograd.grad(run(*leaves), leaves, do)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu().contiguous(), lambda t: t.to(gpu)):
        o = run(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(o, leaves, do)))
    for i in (0, 1, 3):
        a = [t.detach().requires_grad_(i == j) for j, t in enumerate((q, k, v, table))]
        got, = torch.autograd.grad(run(*a), [a[i]], do)
        name = ("dq", "dk", "dv", "dtable")[i]
        R.within(got, R.attention(q, k, v, table, lens, lens, H, Hkv, D, 32, 128, False, D ** -0.5, mask, do, table_grad=i == 3)[name], name, 1e-6)
    o = run(*leaves)
    turned = do.t().contiguous().t()
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(o, leaves, turned)))
    o = run(*leaves)
    (dq,) = torch.autograd.grad(o, leaves[:1], do, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.float().sum().backward()
    with torch.no_grad():
        assert torch.equal(run(*leaves), o)
    leaves[0].data.fill_(1.0)                                  # .data escapes the version check; an in-place change does not
    o = run(*leaves)
    with torch.no_grad():
        leaves[3].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(o, leaves, do)


def test_refusals_on_the_gpu(stg, gpu):
    from stgcma import kernels as K
    lens, H, Hkv, D = [9, 4], 4, 2, 64
    q, k, v, table, do = _make(gpu, lens, lens, H, Hkv, D, 32, 91, fused=False)
    geom = K.RelGeom(H, D, kv_heads=Hkv, device=gpu)
    cu = _cu(lens, gpu)
    o, lse = K.relattn_fwd(geom, q, k, v, table, cu)
    shifted = torch.zeros(q.numel() + 1, dtype=BF16, device=gpu)[1:].view(q.shape)
    odd = torch.zeros(13, H * D + 4, dtype=BF16, device=gpu)[:, :H * D]
    fwd = [(q.half(), k, v, table, cu), (q.float(), k, v, table, cu), (q[:, :-64], k, v, table, cu), (q, k[:-1], v, table, cu), (q, k, v.t(), table, cu),
           (shifted, k, v, table, cu), (odd, k, v, table, cu), (q, k, v, table.half(), cu), (q, k, v, table[:-1], cu), (q, k, v, table.t(), cu), (q, k, v, table, cu.long()),
           (q, k, v, table, cu.cpu()), (q, k, v, table.cpu(), cu), (q, k, v, table, cu[:0]), (q, k, v, table, cu, cu[:2].clone()), (q, q, q, table, cu)]
    for bad in fwd:
        with pytest.raises(RuntimeError):
            K.relattn_fwd(geom, *bad)
    for mask in (torch.ones(12, dtype=torch.bool, device=gpu), torch.ones(13, device=gpu), torch.ones(13, dtype=torch.bool), torch.ones(26, dtype=torch.bool, device=gpu)[::2]):
        with pytest.raises(RuntimeError):
            K.relattn_fwd(geom, q, k, v, table, cu, key_mask=mask)
    with pytest.raises(RuntimeError):
        K.relattn_fwd(geom, q, k, v, table, cu, out=torch.empty_like(q, dtype=F32))
    with pytest.raises(RuntimeError):
        K.relattn_fwd(geom, q, k, v, table, cu, max_q=-1)
    for bad in ((o, lse, do.float()), (o, lse[:, :-1], do), (o, None, do), (o, lse, do[:-1]), (o.float(), lse, do)):
        with pytest.raises(RuntimeError):
            K.relattn_bwd(geom, q, k, v, table, cu, None, *bad)
    kc, vc = k[None].expand(3, -1, -1), v[None].expand(3, -1, -1)
    n3 = torch.tensor([13, 5, 1], dtype=torch.int32, device=gpu)
    shared = K.relattn_decode(geom, q[:3], kc, vc, table, n3)   # one cache for every sequence
    assert torch.equal(shared, K.relattn_decode(geom, q[:3], kc.contiguous(), vc.contiguous(), table, n3))
    wide = torch.full((3, 2 * H * D), 5.0, dtype=BF16, device=gpu)
    assert torch.equal(K.relattn_decode(geom, q[:3], kc, vc, table, n3, out=wide[:, :H * D]), shared) and bool((wide[:, H * D:] == 5.0).all())
    for bad in ((q[:3].float(), kc, vc, table, n3), (q[:2], kc, vc, table, n3), (q[:3], kc[:, :-1], vc, table, n3), (q[:3], kc, vc.half(), table, n3), (q[:3], kc, vc, table, n3[:2]),
                (q[:3], kc, vc, table, n3.cpu()), (q[:3], k, v, table, n3), (q[:3], kc, vc.contiguous().flatten()[:-1], table, n3)):
        with pytest.raises(RuntimeError):
            K.relattn_decode(geom, *bad)


def test_two_streams_at_once(stg, gpu):
    """Calls in flight on two streams together keep their own workspaces."""
    from stgcma import kernels as K
    lens, H, Hkv, D = [700, 300], 8, 2, 64
    geom = K.RelGeom(H, D, kv_heads=Hkv, device=gpu)
    cu = _cu(lens, gpu)
    sets = [_make(gpu, lens, lens, H, Hkv, D, 32, 95 + i) for i in range(2)]
    n = torch.tensor([1000, 1], dtype=torch.int32, device=gpu)
    decode = lambda s: K.relattn_decode(geom, s[0][:2], s[1][None].expand(2, -1, -1), s[2][None].expand(2, -1, -1), s[3], n)
    want = [_all(K, geom, *s[:4], cu, None, s[4], max_q=700) + (decode(s),) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(3):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(_all(K, geom, *s[:4], cu, None, s[4], max_q=700) + (decode(s),))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_of_one_key_have_no_score_gradient(stg, gpu, causal, D):
    """A softmax over one key is constant: dq, dk and dtable are zero, not the roundings of dP - delta, and dv is do."""
    from stgcma import kernels as K
    H, Hkv = 4, 2
    geom = K.RelGeom(H, D, kv_heads=Hkv, causal=causal, device=gpu)
    for lens, shown in (([1, 0, 1, 1], None), ([40, 1, 64], (7, 40, 60))):
        q, k, v, table, do = _make(gpu, lens, lens, H, Hkv, D, 32, 131)
        mask = None
        if shown:
            mask = torch.zeros(sum(lens), dtype=torch.bool, device=gpu)
            mask[list(shown)] = True
        for want_table in (True, False):
            o, lse = K.relattn_fwd(geom, q, k, v, table, _cu(lens, gpu), max_q=max(lens), key_mask=mask)
            dq, dk, dv, dt = K.relattn_bwd(geom, q, k, v, table, _cu(lens, gpu), None, o, lse, do, max_q=max(lens), key_mask=mask, want_table=want_table)
            assert not dq.any() and not dk.any() and (dt is None or not dt.any())
            ref = R.attention(q, k, v, table, lens, lens, H, Hkv, D, 32, 128, causal, D ** -0.5, mask, do)
            R.within(dv, ref["dv"], "dv", 1e-6)
    lens = [200]                                               # the first causal row, and the rows behind it that see few keys
    q, k, v, table, do = _make(gpu, lens, lens, H, Hkv, D, 32, 132)
    if causal:
        dq = _all(K, geom, q, k, v, table, _cu(lens, gpu), None, do)[2]
        ref = R.attention(q[:64], k[:64], v[:64], table, [64], [64], H, Hkv, D, 32, 128, True, D ** -0.5, None, do[:64])["dq"]
        R.within(dq[:64], ref, "dq of the first rows", 1e-6)
