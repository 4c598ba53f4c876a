"""Host side of the sequence operators: the buckets, and every refusal -- of the Python calls and of the C entry points, which answer before any launch."""
import ctypes as C
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import seq_ref as R


@pytest.mark.parametrize("nb,far,causal", [(32, 128, False), (32, 128, True), (4, 2, False), (2, 2, True), (64, 800, True), (12, 100, False), (16, 9, False), (256, 2000, True)])
def test_buckets(stg, nb, far, causal):
    from stgcma import kernels as K
    g = K.RelGeom(2, 64, num_buckets=nb, max_distance=far, causal=causal)
    for d in range(-far - 50, far + 51):
        if causal and d > 0:
            continue
        assert g.bucket(d) == R.bucket(d, nb, far, causal), d
    assert g.far <= far and g.bucket(-10 ** 9) == g.bucket(-g.far) == (nb if causal else nb // 2) - 1
    plan = g.plan(torch.device("cpu")).tolist()
    assert len(plan) == 2 * g.far + 1 and all(0 <= b < nb for b in plan)
    assert plan[g.far] == 0


def test_geometry_refusals(stg):
    from stgcma import kernels as K
    for kw in (dict(num_buckets=3), dict(num_buckets=2), dict(num_buckets=1, causal=True), dict(num_buckets=300, causal=True), dict(max_distance=8), dict(max_distance=10.5)):
        with pytest.raises(ValueError):
            K.RelGeom(4, 64, **kw)
    for a, kw in (((4, 48), {}), ((4, 64), dict(kv_heads=3)), ((0, 64), {}), ((4, 64), dict(scale=0.0)), ((4, 64), dict(scale=-1.0)), ((4, 64), dict(max_distance=10 ** 6)),
                  ((4, 64), dict(scale=float("nan")))):
        with pytest.raises(RuntimeError):
            K.RelGeom(*a, **kw)


def test_python_refusals_without_a_gpu(stg):
    from stgcma import kernels as K, ops_seq
    g = K.RelGeom(2, 64)
    q = torch.zeros(4, 128, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        K.relattn_fwd(g, q, q, q, torch.zeros(32, 2), cu)
    with pytest.raises(RuntimeError, match="GPU"):
        K.relattn_decode(g, q, q[:, None], q[:, None], torch.zeros(32, 2), cu)
    with pytest.raises(RuntimeError, match="GPU"):
        ops_seq.norm_join(torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.bfloat16), None, torch.ones(64), None, torch.ones(64), None)


def _attn_args(**kw):
    from stgcma import _lib
    a = _lib.RelAttnArgs()
    for n in ("Q", "K", "V", "O", "lse", "cu_q", "cu_k", "table", "plan"):
        setattr(a, n, 4096)
    a.Tq = a.Tk = 10
    a.S, a.max_q, a.max_k, a.H, a.Hkv, a.D, a.scale, a.num_buckets, a.far = 1, 10, 10, 4, 2, 64, 0.125, 32, 91
    a.ldq = a.ldo = 256
    a.ldk = a.ldv = 128
    for n, v in kw.items():
        setattr(a, n, v)
    return a


BAD_ATTN = [dict(Q=None), dict(cu_q=None), dict(table=None), dict(plan=None), dict(D=48), dict(D=0), dict(H=3), dict(Hkv=0), dict(H=0), dict(S=-1), dict(S=70000), dict(Tq=-1),
            dict(Tq=2 ** 31), dict(max_q=-1), dict(ldq=255), dict(ldq=128), dict(ldk=64), dict(ldv=132), dict(ldk=2 ** 24 + 8), dict(ldq=2 ** 31), dict(Q=4104), dict(O=4104), dict(scale=0.0), dict(scale=float("nan")),
            dict(num_buckets=31), dict(num_buckets=2), dict(num_buckets=1000), dict(far=0), dict(far=5000)]


@pytest.mark.parametrize("bad", BAD_ATTN)
def test_c_refusals_attention(stg, bad):
    from stgcma import _lib
    lib = _lib.lib()
    assert lib.stg_relattn_fwd(C.byref(_attn_args(**bad)), None) < 0 and lib.stg_last_error()
    assert lib.stg_relattn_bwd(C.byref(_attn_args(**bad)), 4096, 256, 4096, 256, 4096, 128, 4096, 128, None, 4096, 10 ** 9, None) < 0


def test_c_refusals_backward_and_null(stg):
    from stgcma import _lib
    lib = _lib.lib()
    a = _attn_args()
    assert lib.stg_relattn_fwd(None, None) < 0 and lib.stg_relattn_bwd_ws_floats(None, 1) < 0
    good = [4096, 256, 4096, 256, 4096, 128, 4096, 128, 4096, 4096, 10 ** 9]
    for i, v in ((0, None), (2, None), (4, None), (6, None), (9, None), (1, 255), (3, 128), (5, 100), (7, 64), (0, 4098), (2, 4104), (10, 10)):
        w = list(good)
        w[i] = v
        assert lib.stg_relattn_bwd(C.byref(a), *w, None) < 0, (i, v)
    assert lib.stg_relattn_bwd(C.byref(_attn_args(lse=None)), *good, None) < 0


def test_c_refusals_decode(stg):
    from stgcma import _lib
    lib = _lib.lib()

    def args(**kw):
        a = _lib.RelAttnDecodeArgs()
        for n in ("Q", "K", "V", "O", "lens", "table", "plan"):
            setattr(a, n, 4096)
        a.S, a.cap, a.H, a.Hkv, a.D, a.scale, a.num_buckets, a.far, a.causal = 2, 100, 4, 2, 64, 0.125, 32, 113, 1
        a.ldq = a.ldo = 256
        a.ldk = a.ldv = 128
        a.bsk = a.bsv = 12800
        for n, v in kw.items():
            setattr(a, n, v)
        return a
    assert lib.stg_relattn_decode(None, None, 0, None) < 0
    for bad in (dict(Q=None), dict(K=None), dict(lens=None), dict(D=80), dict(H=5), dict(S=-1), dict(S=70000), dict(cap=-1), dict(ldk=64), dict(ldk=129), dict(bsk=12801), dict(bsk=-8),
                dict(K=4104), dict(Q=4104), dict(far=0), dict(num_buckets=1), dict(scale=-1.0), dict(table=None)):
        assert lib.stg_relattn_decode(C.byref(args(**bad)), 4096, 10 ** 9, None) < 0 and lib.stg_last_error(), bad
    need = lib.stg_relattn_decode_ws_floats(2, 2000, 4, 2, 64)
    assert need > 0 and lib.stg_relattn_decode(C.byref(args(cap=2000)), 4096, need - 1, None) == -4
    assert lib.stg_relattn_decode(C.byref(args(S=0)), None, 0, None) == 0


def test_c_refusals_norm_join(stg):
    from stgcma import _lib
    lib = _lib.lib()

    def args(**kw):
        a = _lib.NormJoinArgs()
        for n in ("x", "h", "gate", "w1", "b1", "w2", "b2", "xo", "y", "stats"):
            setattr(a, n, 4096)
        a.x_dtype, a.gate_kind, a.rows, a.C, a.alpha, a.eps = _lib.STG_F32, 2, 10, 64, 1.0, 1e-5
        a.ldx = a.ldh = a.ldxo = a.ldy = 64
        for n, v in kw.items():
            setattr(a, n, v)
        return a
    both = (dict(x_dtype=2), dict(C=60), dict(C=0), dict(C=8200), dict(rows=-1), dict(gate_kind=4), dict(gate_kind=0), dict(gate=None), dict(gate_kind=3), dict(w1=None), dict(h=None),
            dict(xo=None), dict(ldh=56), dict(ldxo=68), dict(h=4104), dict(w2=4100), dict(eps=-1.0), dict(stats=4104))
    for bad in both + (dict(x=None), dict(y=None), dict(ldx=63), dict(ldy=32), dict(x=4104)):
        assert lib.stg_norm_join_fwd(C.byref(args(**bad)), None) < 0 and lib.stg_last_error(), bad
    good = [4096, 64, 4096, 64, 4096, 64, 4096, 64, 4096, None, 4096, 10 ** 9]
    for bad in both + (dict(stats=None),):
        assert lib.stg_norm_join_bwd(C.byref(args(**bad)), *good, None) < 0, bad
    for i, v in ((0, None), (4, None), (6, None), (1, 56), (3, 60), (5, 8), (7, 100), (0, 4104), (2, 4104), (10, None), (11, 3)):
        w = list(good)
        w[i] = v
        assert lib.stg_norm_join_bwd(C.byref(args()), *w, None) < 0, (i, v)
    assert lib.stg_norm_join_fwd(None, None) < 0 and lib.stg_norm_join_bwd_ws_floats(None) < 0 and lib.stg_norm_join_param_floats(None) < 0
    assert lib.stg_norm_join_param_floats(C.byref(args())) == 5 * 64
