"""64-bit references of the sequence operators, with bounds derived beside them (no code of the package).

Attention.  The kernels round P (and in the backward dS) to bf16 before the second product and round the result to bf16; everything else is fp32.
With u = 2^-8 (half a bf16 step, relative) and e = the relative error of a probability,
    |o - ref|  <= u |ref| + (u + 2 e) sum_j p |v|
    |dv - ref| <= u |ref| + (u + 2 e) sum_i p |do|
    |dS - ref| <= 2 e p (|dP| + |delta|) + p E_i =: s_ij     E_i = error of delta_i: o's error where delta comes from the stored o (dq, and
                                                       dk without a table gradient, of sequences of more than 64 keys), fp32's where it
                                                       is summed again (dtable, dk, short sequences)
    |dq - ref| <= u |ref| + scale sum_j (u |dS| + (1 + u) s_ij) |k|,   dk alike,   dtable <= sum s_ij over the bucket + its own fp32 summation.
e: the score is a sum of D products in fp32 plus the bias, so its error is at most (D + 8) 2^-24 A with A = scale sum |q||k| + |bias| + |lse|, the
exponential and the row sum of n terms add (n + 8) 2^-24.
"""
import functools
import math

import torch

U = 2.0 ** -8
E32 = 2.0 ** -24


@functools.lru_cache(None)
def bucket(distance, buckets, far, causal):
    half = buckets if causal else buckets // 2
    first = half // 2
    n, d = half - first, abs(distance)
    if d < first:
        b = d
    else:
        b = max(t for t in range(n) if t == 0 or d ** n * first ** t >= far ** t * first ** n) + first
    return b + (half if distance > 0 and not causal else 0)


def attention(q, k, v, table, lens_q, lens_k, H, Hkv, D, buckets, far, causal, scale, mask=None, do=None, table_grad=True):
    """dict of name -> (value, bound), all float64, rows packed; rows behind the last sequence are zero (lse -inf)."""
    dev = q.device
    f = lambda t: t.double()
    Tq, Tk = q.shape[0], k.shape[0]
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=dev)
    out = {n: (z(*s), z(*s)) for n, s in (("o", (Tq, H * D)), ("dq", (Tq, H * D)), ("dk", (Tk, Hkv * D)), ("dv", (Tk, Hkv * D)), ("dtable", (buckets, H)))}
    out["lse"] = (torch.full((H, Tq), -math.inf, dtype=torch.float64, device=dev), z(H, Tq))
    a = b = 0
    for nq, nk in zip(lens_q, lens_k):
        rq, rk = slice(a, a + nq), slice(b, b + nk)
        a, b = a + nq, b + nk
        if nq == 0 or nk == 0:
            continue
        shift = nk - nq
        lo, hi = -(nk - 1) - abs(shift) - nq, nk + nq + abs(shift)
        ids = torch.tensor([bucket(d, buckets, far, causal) for d in range(lo, hi + 1)], device=dev)
        rel = torch.arange(nk, device=dev)[None, :] - (torch.arange(nq, device=dev)[:, None] + shift)
        bid = ids[rel - lo]
        hidden = torch.zeros(nq, nk, dtype=torch.bool, device=dev)
        if causal:
            hidden |= rel > 0
        if mask is not None:
            hidden |= ~mask[rk].bool()[None, :]
        for h in range(H):
            j = h // (H // Hkv)
            cq, ck = slice(h * D, (h + 1) * D), slice(j * D, (j + 1) * D)
            Q, Kk, V = f(q[rq, cq]), f(k[rk, ck]), f(v[rk, ck])
            dead = mask is not None and ~mask[rk].bool()
            if mask is not None:                                  # masked rows may hold anything
                Kk, V = Kk.masked_fill(dead[:, None], 0.0), V.masked_fill(dead[:, None], 0.0)
            bias = f(table)[:, h][bid]
            x = (scale * Q @ Kk.t() + bias).masked_fill(hidden, -math.inf)
            m = x.amax(1, keepdim=True)
            m = torch.where(m == -math.inf, torch.zeros_like(m), m)
            p = torch.exp(x - m)
            l = p.sum(1, keepdim=True)
            p = torch.where(l > 0, p / l, torch.zeros_like(p))
            lse = torch.where(l > 0, m + torch.log(l), torch.full_like(l, -math.inf))
            fin = lambda t: torch.where(torch.isfinite(t), t.abs(), torch.zeros_like(t))
            A = scale * Q.abs() @ Kk.abs().t() + fin(bias).clamp(max=1e4) + fin(lse)
            e = ((D + 8) * A.amax(1, keepdim=True) + nk + 8) * E32
            out["lse"][0][h, rq] = lse[:, 0]
            out["lse"][1][h, rq] = 2 * e[:, 0]
            O = p @ V
            pv = p @ V.abs()
            out["o"][0][rq, cq] = O
            out["o"][1][rq, cq] = U * O.abs() + (U + 2 * e) * pv
            if do is None:
                continue
            G = f(do[rq, cq])
            dP = G @ V.t()
            delta = (p * dP).sum(1, keepdim=True)
            dS = p * (dP - delta)
            dperr = (D + 8) * E32 * (G.abs() @ V.abs().t())

            def size(oerr):                                       # bounds of |dS - ref| and of that plus dS's own rounding
                E = (G.abs() * oerr).sum(1, keepdim=True) + (D + 8) * E32 * (G.abs() * O.abs()).sum(1, keepdim=True)
                s = 2 * e * p * (dP.abs() + delta.abs()) + p * (E + dperr)
                return s, U * dS.abs() + (1 + U) * s
            rounded = U * O.abs() + (U + 2 * e) * pv
            s, w = size(2 * e * pv if nk <= 64 else rounded)
            out["dq"][0][rq, cq] = scale * dS @ Kk
            out["dq"][1][rq, cq] = U * (scale * dS @ Kk).abs() + scale * w @ Kk.abs()
            s, w = size(2 * e * pv if table_grad or nk <= 64 else rounded)
            out["dk"][0][rk, ck] += scale * dS.t() @ Q
            out["dk"][1][rk, ck] += scale * w.t() @ Q.abs()
            out["dv"][0][rk, ck] += p.t() @ G
            out["dv"][1][rk, ck] += ((U + 2 * e) * p).t() @ G.abs()
            for t in range(buckets):
                sel = (bid == t) & ~hidden
                out["dtable"][0][t, h] += dS[sel].sum()
                out["dtable"][1][t, h] += s[sel].sum() + (nq + 64) * E32 * dS[sel].abs().sum()
    for n in ("dk", "dv"):
        out[n][1].add_(U * out[n][0].abs())
    return out


def within(got, ref, what, slack=0.0):
    """|got - value| <= bound + slack everywhere (and -inf where the value is -inf)."""
    val, bound = ref
    got = got.double()
    inf = torch.isinf(val)
    assert torch.equal(torch.isinf(got), inf), f"{what}: infinities differ"
    d = torch.where(inf, torch.zeros_like(val), got - torch.where(inf, got, val)).abs()
    bad = ~(d <= bound + slack)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound, worst {float((d - bound).max()):.3e} (value {float(val[bad][0]):.4e}, got {float(got[bad][0]):.4e})"


def norm_join(x, h, gate, w1, b1, w2, b2, kind, alpha, eps, rows_per_group=None, dy=None, dx_new=None, x_new=None):
    """Values in float64.  x_new: the stored stream the second norm reads (the kernel's own rounding of it when given)."""
    D = lambda t: None if t is None else t.double()
    x, h, gate, w1, b1, w2, b2 = map(D, (x, h, gate, w1, b1, w2, b2))

    def hat(u):
        if kind == "layer":
            u = u - u.mean(1, keepdim=True)
        r = 1.0 / torch.sqrt((u * u).mean(1, keepdim=True) + eps)
        return u * r, r

    def back(g, z, r):
        out = g - z * (g * z).mean(1, keepdim=True)
        if kind == "layer":
            out = out - g.mean(1, keepdim=True)
        return r * out
    z1, r1 = hat(h)
    n = z1 * w1 + (0 if b1 is None else b1)
    g = torch.ones(1, dtype=torch.float64, device=x.device) if gate is None else gate
    if gate is not None and gate.dim() == 2:
        g = gate.repeat_interleave(rows_per_group, 0)[:x.shape[0]]
    xn = alpha * x + g * n
    z2, r2 = hat(xn if x_new is None else x_new.double())
    out = {"x_new": xn, "y": z2 * w2 + (0 if b2 is None else b2)}
    if dy is None:
        return out
    dy = dy.double()
    t = back(dy * w2, z2, r2) + (0 if dx_new is None else dx_new.double())
    out["dx"] = alpha * t
    out["dh"] = back(t * g * w1, z1, r1)
    dn = t * n
    if gate is None:
        out["dgate"] = None
    elif gate.dim() == 2:
        out["dgate"] = torch.stack([c.sum(0) for c in dn.split(rows_per_group)])
    else:
        out["dgate"] = dn.sum().view(gate.shape) if gate.numel() == 1 else dn.sum(0)
    out["dpost_w"] = (t * g * z1).sum(0)
    out["dpost_b"] = None if b1 is None else (t * g).expand_as(n).sum(0)
    out["dpre_w"] = (dy * z2).sum(0)
    out["dpre_b"] = None if b2 is None else dy.sum(0)
    return out
