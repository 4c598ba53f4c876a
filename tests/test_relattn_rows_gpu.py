"""Rows at the edges of the ragged attention: sequences with one visible key, rows behind the last sequence in a given output, single rows of wide
buffers, and query heads of a shared key / value head in fewer parts than heads."""
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


def _rn(gpu, seed):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    return lambda *s, dtype=BF16: torch.randn(*s, generator=g, device=gpu, dtype=F32).to(dtype)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_one_visible_key_of_many(stg, gpu, causal, D):
    """A mask that leaves one key of a long sequence, in its first tile of 64 or a later one, or none: the softmax is constant and dq, dk and dtable are zero."""
    from stgcma import kernels as K
    lens, shown, H, Hkv = [200, 90, 65, 130, 300], (130, 200 + 3, 290 + 64, 485 + 299), 4, 2
    n, rn = sum(lens), _rn(gpu, 810)
    q, k, v, do, table = rn(n, H * D), rn(n, Hkv * D), rn(n, Hkv * D), rn(n, H * D), rn(32, H, dtype=F32)
    mask = torch.zeros(n, dtype=torch.bool, device=gpu)
    mask[list(shown)] = True                                  # (the fourth sequence shows nothing)
    geom = K.RelGeom(H, D, kv_heads=Hkv, causal=causal, device=gpu)
    cu = _cu(lens, gpu)
    ref = R.attention(q, k, v, table, lens, lens, H, Hkv, D, 32, 128, causal, D ** -0.5, mask, do)
    o, lse = K.relattn_fwd(geom, q, k, v, table, cu, key_mask=mask)
    R.within(o, ref["o"], "o")
    for want_table in (True, False):
        dq, dk, dv, dt = K.relattn_bwd(geom, q, k, v, table, cu, None, o, lse, do, key_mask=mask, want_table=want_table)
        assert not dq.any() and not dk.any() and (dt is None or not dt.any())
        R.within(dv, ref["dv"], "dv", 1e-6)
    mask[131] = True                                          # two visible keys: gradients again
    ref = R.attention(q, k, v, table, lens, lens, H, Hkv, D, 32, 128, causal, D ** -0.5, mask, do)
    o, lse = K.relattn_fwd(geom, q, k, v, table, cu, key_mask=mask)
    got = K.relattn_bwd(geom, q, k, v, table, cu, None, o, lse, do, key_mask=mask)
    for name, t in zip(("dq", "dk", "dv", "dtable"), got):
        R.within(t, ref[name], name, 1e-6)
    assert bool(got[0][131:200].any()) and bool(got[1][130:132].any()) and not got[0][200:].any()


def test_log_sums_behind_the_last_sequence(stg, gpu):
    """lse is -inf behind the last sequence whether the output is fresh or given (whose own rows there stay as they were)."""
    from stgcma import kernels as K
    lens, tail, H, Hkv, D = [70, 33], 29, 4, 2, 64
    n, rn = sum(lens) + tail, _rn(gpu, 820)
    q, k, v, table = rn(n, H * D), rn(n, Hkv * D), rn(n, Hkv * D), rn(32, H, dtype=F32)
    geom = K.RelGeom(H, D, kv_heads=Hkv, device=gpu)
    cu = _cu(lens, gpu)
    want, want_lse = K.relattn_fwd(geom, q, k, v, table, cu, max_q=70)
    for hint in (70, None):
        for _ in range(4):
            junk = [torch.full((H, n), float("nan"), device=gpu) for _ in range(4)]
            del junk                                          # a fresh lse finds these
            mine = torch.full((n, H * D), 7.0, dtype=BF16, device=gpu)
            o, lse = K.relattn_fwd(geom, q, k, v, table, cu, max_q=hint, out=mine)
            assert torch.equal(lse, want_lse) and bool((lse[:, 103:] == -float("inf")).all())
            assert torch.equal(o[:103], want[:103]) and bool((o[103:] == 7.0).all())


def test_single_rows_of_wide_buffers(stg, gpu):
    """One row has no leading dimension to be misaligned: a row cut out of a buffer of any width goes through forward, backward and the single-token form."""
    from stgcma import kernels as K, ops_seq
    H, D = 4, 64
    rn = _rn(gpu, 830)
    big = rn(1, 3 * H * D + 5)
    q, k, v = (big[:, i * H * D:(i + 1) * H * D] for i in range(3))
    do, table = rn(1, H * D + 3)[:, :H * D], rn(32, H, dtype=F32)
    geom = K.RelGeom(H, D, device=gpu)
    cu = _cu([1], gpu)
    dense = [t.contiguous().clone() for t in (q, k, v)]
    outs = []
    for a in ([q, k, v], dense):
        leaf = [t.detach().requires_grad_(True) for t in a + [table]]
        o = ops_seq.rel_attention(*leaf, geom, cu)
        outs.append((o.detach(),) + torch.autograd.grad(o, leaf, do))
        o, lse = K.relattn_fwd(geom, *a, table, cu)
        outs[-1] += (o, lse) + K.relattn_bwd(geom, *a, table, cu, None, o, lse, do)
        outs[-1] += (K.relattn_decode(geom, a[0], a[1][None], a[2][None], table, torch.ones(1, dtype=torch.int32, device=gpu)),)
    assert all(torch.equal(x, y) for x, y in zip(*outs))


@pytest.mark.parametrize("H,Hkv,D,causal,S,rows", [(32, 8, 32, True, 52, 43), (48, 8, 32, False, 45, 20), (16, 4, 128, False, 50, 60), (32, 8, 64, True, 45, 64)])
def test_heads_of_a_group_in_a_few_parts(stg, gpu, H, Hkv, D, causal, S, rows):
    """dK / dV of a shared key / value head whose query heads go to more than one block and fewer than one block each."""
    from stgcma import kernels as K
    from stgcma import _lib
    import ctypes as C
    g = torch.Generator().manual_seed(5)
    lens = (rows + torch.randint(-9, 10, (S,), generator=g)).tolist()
    n, rn = sum(lens), _rn(gpu, 840 + H)
    q, k, v, do, table = rn(n, H * D), rn(n, Hkv * D), rn(n, Hkv * D), rn(n, H * D), rn(4, H, dtype=F32)
    geom = K.RelGeom(H, D, kv_heads=Hkv, num_buckets=4, max_distance=10, causal=causal, device=gpu)
    cu = _cu(lens, gpu)
    ref = R.attention(q, k, v, table, lens, lens, H, Hkv, D, 4, 10, causal, D ** -0.5, None, do)
    o, lse = K.relattn_fwd(geom, q, k, v, table, cu, max_q=max(lens))
    a = K._rel_fill(geom, q, k, v, o, lse, table, cu, None, max(lens), None, None)
    parts = _lib.lib().stg_relattn_bwd_ws_floats(C.byref(a), 0) // (2 * n * Hkv * D)       # the parts' share of the workspace
    assert 1 < parts < H // Hkv, parts
    for name, t in zip(("dq", "dk", "dv", "dtable"), K.relattn_bwd(geom, q, k, v, table, cu, None, o, lse, do, max_q=max(lens))):
        R.within(t, ref[name], name, 1e-6)
    ref = R.attention(q, k, v, table, lens, lens, H, Hkv, D, 4, 10, causal, D ** -0.5, None, do, table_grad=False)
    for name, t in zip(("dq", "dk", "dv"), K.relattn_bwd(geom, q, k, v, table, cu, None, o, lse, do, max_q=max(lens), want_table=False)):
        R.within(t, ref[name], name + " (frozen table)", 1e-6)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shown", [(10, 290), (0, 64), (63, 599), (255, 256), (511, 513), (598, 599)])
def test_two_visible_keys_anywhere(stg, gpu, causal, shown):
    """Two keys of 600, near each other or far apart: no constant softmax."""
    from stgcma import kernels as K
    n, H, Hkv, D, rn = 600, 2, 1, 64, _rn(gpu, 850)
    q, k, v, do, table = rn(n, H * D), rn(n, Hkv * D), rn(n, Hkv * D), rn(n, H * D), rn(32, H, dtype=F32)
    mask = torch.zeros(n, dtype=torch.bool, device=gpu)
    mask[list(shown)] = True
    geom = K.RelGeom(H, D, kv_heads=Hkv, causal=causal, device=gpu)
    cu = _cu([n], gpu)
    ref = R.attention(q, k, v, table, [n], [n], H, Hkv, D, 32, 128, causal, D ** -0.5, mask, do)
    o, lse = K.relattn_fwd(geom, q, k, v, table, cu, key_mask=mask)
    got = K.relattn_bwd(geom, q, k, v, table, cu, None, o, lse, do, key_mask=mask)
    for name, t in zip(("dq", "dk", "dv", "dtable"), got):
        R.within(t, ref[name], name, 1e-6)
    assert bool(got[0][shown[1]:].any())
