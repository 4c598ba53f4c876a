"""The norm - gate - residual - norm join on the GPU against 64-bit formulas, its gradients against differences, and refusals.

Bounds: x_new is one rounding to the stream's type of an fp32 result; y, dh (and dx in a bf16 stream) one rounding to bf16.  The fp32 arithmetic of a
row of C elements is good to (C + 16) 2^-24 of the sums it takes, so the elementwise bounds are u |ref| + (C + 16) 2^-24 x (the row's largest
term), column sums over R rows add R 2^-24 of the sum of the magnitudes."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import seq_ref as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
E32 = 2.0 ** -24

CASES = [
    # rows, C, kind, stream, gate, rows_per_group, post_b, pre_b, alpha, dx_new given
    (1, 8, "layer", F32, "none", None, False, True, 1.0, True),
    (1, 8192, "rms", BF16, "channel", None, False, False, 0.75, True),
    (98, 512, "layer", F32, "one", None, True, True, 1.0, True),
    (197, 768, "rms", BF16, "group", 50, False, False, 1.0, True),
    (333, 520, "layer", BF16, "group", 1, True, True, 1.5, False),
    (1000, 1032, "rms", F32, "group", 999, True, False, 1.0, True),
    (64, 2048, "layer", F32, "channel", None, True, True, 1.0, True),
    (50, 4096, "rms", F32, "one", None, False, False, 0.5, False),
    (37, 4104, "layer", BF16, "group", 9, False, True, 1.0, True),
    (2500, 192, "layer", F32, "group", 7, True, True, 1.0, True),
    (5000, 96, "rms", BF16, "group", 2048, False, False, 1.0, True),
    (3, 8184, "layer", F32, "channel", None, True, True, -1.0, True),
    (1, 8, "rms", BF16, "group", 5, True, True, 1.0, True),              # a group larger than the batch
    (77, 16, "layer", F32, "channel", None, True, False, 1.0, True),
    (4099, 128, "layer", F32, "group", 1, True, True, 1.0, True),        # a group to every row; more groups than blocks
    (9001, 136, "rms", BF16, "group", 4, False, True, 1.0, True),
    (6000, 256, "layer", BF16, "group", 3, True, False, 0.5, True),
    (2049, 512, "rms", F32, "group", 2, True, True, 1.0, False),
    (700, 264, "layer", F32, "one", None, False, False, 1.0, True),
    (1300, 1024, "rms", BF16, "none", None, True, True, 1.0, True),
    (520, 4096, "layer", BF16, "channel", None, True, True, 1.0, True),
    (600, 5120, "rms", F32, "group", 2, False, False, 1.0, True),
]


def _make(gpu, rows, C, kind, stream, gate, rpg, post_b, pre_b, seed):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    rn = lambda *s, dtype=F32, std=1.0, mean=0.0: (torch.randn(*s, generator=g, device=gpu) * std + mean).to(dtype)
    pitch = C + 16                                            # rows of a wider buffer
    x = rn(rows, pitch, dtype=stream, std=2.0)[:, 8:8 + C]
    h = rn(rows, pitch, dtype=BF16, std=1.5, mean=0.5)[:, 8:8 + C]
    shape = {"none": None, "one": (1,), "channel": (C,), "group": (-(-rows // (rpg or 1)), C)}[gate]
    return dict(x=x, h=h, gate=rn(*shape, std=0.5) if shape else None, w1=rn(C, std=0.2, mean=1.0), b1=rn(C, std=0.2) if post_b else None,
                w2=rn(C, std=0.2, mean=1.0), b2=rn(C, std=0.2) if pre_b else None, dy=rn(rows, C, dtype=BF16), dxn=rn(rows, C, dtype=stream))


def _close(got, ref, what, u, extra):
    d = (got.double() - ref).abs()
    bad = ~(d <= u * ref.abs() + extra)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((d - u * ref.abs()).max()):.3e} against {float(torch.as_tensor(extra).max()):.3e}"


@pytest.mark.parametrize("case", range(len(CASES)))
def test_values_and_gradients(stg, gpu, case):
    from stgcma import ops_seq, kernels as K
    rows, C, kind, stream, gate, rpg, pb, qb, alpha, with_dx = CASES[case]
    t = _make(gpu, rows, C, kind, stream, gate, rpg, pb, qb, 300 + case)
    how = dict(kind=kind, alpha=alpha, rows_per_group=rpg)
    leaf = {n: v.detach().requires_grad_(True) for n, v in t.items() if v is not None and n not in ("dy", "dxn")}
    a = [leaf.get(n) for n in ("x", "h", "gate", "w1", "b1", "w2", "b2")]
    xn, y = ops_seq.norm_join(*a, **how)
    ref = R.norm_join(*[t[n] for n in ("x", "h", "gate", "w1", "b1", "w2", "b2")], kind, alpha, 1e-5, rpg, t["dy"], t["dxn"] if with_dx else None, x_new=xn.detach())
    us = R.U if stream == BF16 else 2 * E32
    k32 = (C + 16) * E32
    rowmax = lambda v: v.double().abs().amax(1, keepdim=True)
    _close(xn.detach(), ref["x_new"], "x_new", us, k32 * rowmax(ref["x_new"]) * 4)
    _close(y.detach(), ref["y"], "y", R.U, k32 * rowmax(ref["y"]) * 4)
    grads = torch.autograd.grad([xn, y] if with_dx else [y], list(leaf.values()), [t["dxn"], t["dy"]] if with_dx else [t["dy"]])
    got = dict(zip(leaf, grads))
    _close(got["x"], ref["dx"], "dx", us, k32 * rowmax(ref["dx"]) * 4)
    # dh passes through two norms' backward: its row's terms are as large as the row's gradient times 1 / rms(h)
    r1 = 1.0 / t["h"].double().var(1, unbiased=False, keepdim=True).add(1e-5).sqrt() if kind == "layer" else 1.0 / t["h"].double().square().mean(1, keepdim=True).add(1e-5).sqrt()
    gs = 1.0 if t["gate"] is None else float(t["gate"].abs().max())
    through = rowmax(ref["dx"] / alpha) * gs * float(t["w1"].abs().max()) * r1
    _close(got["h"], ref["dh"], "dh", R.U, 8 * k32 * through)
    # column sums: fp32 sums of rows' terms
    hat = lambda v: ((v.double() - (v.double().mean(1, keepdim=True) if kind == "layer" else 0)) * (1 if v is None else 1))
    zmax = 8.0 * max(1.0, C ** 0.5 / 8)                        # |normalised value| <= sqrt(C); Gaussian rows stay below 8
    tmax = float((ref["dx"] / alpha).abs().max())
    big = {"gate": tmax * (zmax * float(t["w1"].abs().max()) + 1), "w1": tmax * gs * zmax, "b1": tmax * gs, "w2": float(t["dy"].double().abs().max()) * zmax,
           "b2": float(t["dy"].double().abs().max())}
    for n in ("gate", "w1", "b1", "w2", "b2"):
        if n not in got:
            continue
        r = ref["d" + {"gate": "gate", "w1": "post_w", "b1": "post_b", "w2": "pre_w", "b2": "pre_b"}[n]]
        terms = rows if n != "gate" or gate != "group" else min(rows, rpg)
        if n == "gate" and gate == "one":
            terms *= C
        _close(got[n], r, n, 0.0, (terms + C + 64) * E32 * terms ** 0.5 * big[n] + 1e-7)


def test_gradient_against_differences(stg, gpu):
    """The gradient along a direction against a central difference of the 64-bit forward (error ~ h^2): an fp32 stream, every input at once."""
    from stgcma import ops_seq
    rows, C, rpg = 40, 64, 16
    t = _make(gpu, rows, C, "layer", F32, "group", rpg, True, True, 17)
    names = ["x", "h", "gate", "w1", "b1", "w2", "b2"]
    leaf = [t[n].detach().requires_grad_(True) for n in names]
    xn, y = ops_seq.norm_join(*leaf, kind="layer", alpha=0.9, rows_per_group=rpg)
    grads = torch.autograd.grad([xn, y], leaf, [t["dxn"], t["dy"]])
    gen = torch.Generator().manual_seed(4)
    ways = [torch.randn(v.shape, generator=gen).to(gpu).double() for v in leaf]

    def loss(s):
        r = R.norm_join(*[t[n].double() + s * w for n, w in zip(names, ways)], "layer", 0.9, 1e-5, rpg)
        return float((r["x_new"] * t["dxn"].double()).sum() + (r["y"] * t["dy"].double()).sum())
    diff = (loss(1e-5) - loss(-1e-5)) / 2e-5
    got = float(sum((g.double() * w).sum() for g, w in zip(grads, ways)))
    size = float(sum((g.double() * w).abs().sum() for g, w in zip(grads, ways)))
    assert abs(got - diff) <= 2.0 ** -9 * size, (got, diff, size)        # dh is rounded to bf16; the rest is fp32


def test_same_call_same_bits_capture_and_streams(stg, gpu):
    from stgcma import ops_seq
    t = _make(gpu, 700, 768, "layer", BF16, "group", 197, True, True, 9)
    u = _make(gpu, 700, 768, "layer", BF16, "group", 197, True, True, 10)
    names = ["x", "h", "gate", "w1", "b1", "w2", "b2"]

    def step(s):
        leaf = [s[n].detach().requires_grad_(True) for n in names]
        xn, y = ops_seq.norm_join(*leaf, rows_per_group=197)
        return (xn.detach(), y.detach()) + torch.autograd.grad([xn, y], leaf, [s["dxn"], s["dy"]])
    want = [step(t), step(u)]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(t), want[0]))
    buf = {n: v.clone() for n, v in t.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(buf)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(buf)
    for i, s in ((1, u), (0, t), (1, u)):
        for n in buf:
            buf[n].copy_(s[n])
        graph.replay()
        step(t)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


def test_block_of_attention_and_join(stg, gpu):
    """The operators as a block uses them: projections around the attention, its output joined into the stream; every gradient arrives and agrees with
    64-bit autograd of the formulas to the bf16 roundings on the way (each of the five bf16 tensors between loss and leaf: 2^-8, summed in L2)."""
    from stgcma import kernels as K, ops_seq
    from stgcma.ops_head import linear
    lens, H, D = [60, 33, 7], 4, 32
    n, C = sum(lens), H * D
    g = torch.Generator().manual_seed(8)
    rn = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(gpu)
    P = dict(wqkv=rn(3 * C, C, std=C ** -0.5), wo=rn(C, C, std=C ** -0.5), table=rn(32, H), gate=rn(1), w1=rn(C, std=0.1) + 1, b1=rn(C, std=0.1), w2=rn(C, std=0.1) + 1,
             b2=rn(C, std=0.1))
    P = {k: torch.nn.Parameter(v) for k, v in P.items()}
    x, y0, dx, dy = rn(n, C), rn(n, C).to(BF16), rn(n, C), rn(n, C).to(BF16)
    geom = K.RelGeom(H, D, device=gpu)
    cu = torch.tensor([0, 60, 93, 100], dtype=torch.int32, device=gpu)
    qkv = linear(y0, P["wqkv"])
    o = ops_seq.rel_attention(qkv[:, :C], qkv[:, C:2 * C], qkv[:, 2 * C:], P["table"], geom, cu, max_q=60)
    xn, y = ops_seq.norm_join(x, linear(o, P["wo"]), P["gate"], P["w1"], P["b1"], P["w2"], P["b2"])
    torch.autograd.backward([xn, y], [dx, dy])
    Q = {k: v.detach().double().requires_grad_(True) for k, v in P.items()}
    z = y0.double() @ Q["wqkv"].t()
    outs, at = [], 0
    for m in lens:
        q, k, v = (z[at:at + m, i * C:(i + 1) * C].view(m, H, D).transpose(0, 1) for i in range(3))
        ids = torch.tensor([[R.bucket(j - i, 32, 128, False) for j in range(m)] for i in range(m)], device=gpu)
        s = q @ k.transpose(1, 2).contiguous() * D ** -0.5 + Q["table"].t()[:, ids]
        outs.append((torch.softmax(s, -1) @ v).transpose(0, 1).reshape(m, C))
        at += m
    hh = torch.cat(outs) @ Q["wo"].t()
    ln = lambda u, w, b: torch.nn.functional.layer_norm(u, (C,), w, b)
    xr = x.double() + Q["gate"] * ln(hh, Q["w1"], Q["b1"])
    yr = ln(xr, Q["w2"], Q["b2"])
    torch.autograd.backward([xr, yr], [dx.double(), dy.double()])
    tol = 5 * 2.0 ** -8
    assert float((y.double() - yr).norm() / yr.norm()) < tol and float((xn.double() - xr).norm() / xr.norm()) < tol
    for k in P:
        assert float((P[k].grad.double() - Q[k].grad).norm() / Q[k].grad.norm()) < tol, k


@pytest.mark.parametrize("gate", ["none", "one", "channel", "group"])
def test_no_rows(stg, gpu, gate):
    from stgcma import ops_seq
    C = 64
    t = _make(gpu, 0, C, "layer", F32, gate, 4 if gate == "group" else None, True, True, 5)
    leaf = {n: v.detach().requires_grad_(True) for n, v in t.items() if v is not None and n not in ("dy", "dxn")}
    xn, y = ops_seq.norm_join(*[leaf.get(n) for n in ("x", "h", "gate", "w1", "b1", "w2", "b2")], rows_per_group=4 if gate == "group" else None)
    assert xn.shape == y.shape == (0, C)
    for v, g in zip(leaf.values(), torch.autograd.grad([xn, y], list(leaf.values()), [t["dxn"], t["dy"]])):
        assert g.shape == v.shape and bool((g == 0).all())


def test_offsets_beyond_32_bits(stg, gpu):
    """Rows 2^23 elements apart (the last of 300 stands 2.5 * 10^9 elements behind the first) equal the dense call."""
    from stgcma import kernels as K
    rows, C = 300, 512
    t = _make(gpu, rows, C, "layer", BF16, "channel", None, True, True, 6)
    big = torch.empty(rows, 1 << 23, dtype=BF16, device=gpu)
    wide = {}
    for i, n in enumerate(("x", "h", "dy", "dxn")):
        wide[n] = big[:, 1024 * i:1024 * i + C]
        wide[n].copy_(t[n])
    w = [t[n] for n in ("gate", "w1", "b1", "w2", "b2")]
    out = []
    for s in (t, wide):
        xn, y, st = K.norm_join_fwd(s["x"], s["h"], *w)
        g = K.norm_join_bwd(xn, s["h"], *w, st, s["dy"], s["dxn"])
        out.append([xn, y, st] + list(g.values()))
    wide["x"].copy_(xn)                                        # the stored stream in rows as far apart
    out.append(out[0][:3] + list(K.norm_join_bwd(wide["x"], wide["h"], *w, st, wide["dy"], wide["dxn"]).values()))
    for other in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], other))


def test_autograd_corners(stg, gpu):
    """Saved tensors that hooks move and pack densely, single wanted gradients, only one of the two outputs used, strided incoming gradients, no second
    derivative."""
    from stgcma import ops_seq
    t = _make(gpu, 90, 96, "layer", F32, "group", 40, True, True, 12)
    names = ["x", "h", "gate", "w1", "b1", "w2", "b2"]
    run = lambda leaf: ops_seq.norm_join(*leaf, rows_per_group=40)
    leaf = [t[n].detach().requires_grad_(True) for n in names]
    want = torch.autograd.grad(run(leaf), leaf, [t["dxn"], t["dy"]])
    with torch.autograd.graph.saved_tensors_hooks(lambda a: a.cpu().contiguous(), lambda a: a.to(gpu)):
        out = run(leaf)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(out, leaf, [t["dxn"], t["dy"]])))
    turned = [t[n].t().contiguous().t() for n in ("dxn", "dy")]
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(run(leaf), leaf, turned)))
    for i in range(7):
        one = [t[n].detach().requires_grad_(i == j) for j, n in enumerate(names)]
        got, = torch.autograd.grad(run(one), [one[i]], [t["dxn"], t["dy"]])
        assert torch.equal(got, want[i]), names[i]
    ref = R.norm_join(*[t[n] for n in names], "layer", 1.0, 1e-5, 40, torch.zeros_like(t["dy"]), t["dxn"])
    xn, y = run(leaf)
    got = dict(zip(names, torch.autograd.grad(xn, leaf, t["dxn"], allow_unused=True)))       # the second norm's output unused
    k32 = (96 + 16) * E32
    _close(got["x"], ref["dx"], "dx", 2 * E32, k32 * ref["dx"].abs().amax(1, keepdim=True) * 4)
    assert bool((got["w2"] == 0).all()) and bool((got["b2"] == 0).all())
    out = run(leaf)
    (dx,) = torch.autograd.grad(out, leaf[:1], [t["dxn"], t["dy"]], create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(run(leaf), out))
    scalar = torch.tensor(0.7, device=gpu, requires_grad=True)  # a gate without dimensions
    one = torch.tensor([0.7], device=gpu, requires_grad=True)
    g0, g1 = (torch.autograd.grad(ops_seq.norm_join(*[t[n] for n in names[:2]], g, *[t[n] for n in names[3:]]), [g], [t["dxn"], t["dy"]])[0] for g in (scalar, one))
    assert g0.shape == () and g1.shape == (1,) and torch.equal(g0, g1[0])


def test_refusals_on_the_gpu(stg, gpu):
    from stgcma import kernels as K
    t = _make(gpu, 20, 64, "layer", F32, "channel", None, True, True, 3)
    a = [t[n] for n in ("x", "h", "gate", "w1", "b1", "w2", "b2")]
    xn, y, st = K.norm_join_fwd(*a)
    off = torch.zeros(65, device=gpu)[1:]

    def with_(**kw):
        b = dict(zip(("x", "h", "gate", "w1", "b1", "w2", "b2"), a))
        b.update(kw)
        return list(b.values())
    for bad in (with_(x=t["x"].half()), with_(h=t["h"].float()), with_(h=t["h"][:-1]), with_(h=t["h"][:, :56]), with_(x=t["x"].t().contiguous().t()), with_(x=t["x"][:, 1:]),
                with_(w1=None), with_(w2=None), with_(w1=off), with_(w1=t["w1"].to(BF16)), with_(b1=t["b1"][:56]), with_(w2=t["w2"].cpu()), with_(gate=t["gate"][:8]),
                with_(gate=t["gate"].to(BF16)), with_(gate=torch.ones(20, 64, device=gpu)), with_(gate=torch.ones(1, device="cpu")), with_(x=t["x"][0]),
                with_(x=t["x"][:, :60].contiguous(), h=t["h"][:, :60].contiguous())):
        with pytest.raises(RuntimeError):
            K.norm_join_fwd(*bad)
    for kw in (dict(kind="batch"), dict(rows_per_group=0, kind="none")):
        with pytest.raises(RuntimeError):
            K.norm_join_fwd(*a, **kw)
    with pytest.raises(RuntimeError):
        K.norm_join_fwd(*with_(gate=torch.ones(5, 64, device=gpu)), rows_per_group=3)
    for st_, dy, dxn in ((st, t["dy"].float(), None), (st[:-1], t["dy"], None), (None, t["dy"], None), (st, t["dy"], t["dxn"].to(BF16)), (st, t["dy"][:-1], None)):
        with pytest.raises(RuntimeError):
            K.norm_join_bwd(xn, *a[1:], st_, dy, dxn)
