"""Bounds of the norm - gate - residual - norm join's column sums (weights, biases, gate), from their own terms in 64 bits; no code of the package.

With e = 2^-24.  A row's statistics are fp32 sums of C terms, each thread adding up to 16 and a tree joining the threads (6 steps in a wave, up to 8
waves in turn): at most 32 e of the sum of magnitudes.  So the normalised row z = (u - mean) r has
    |dz| <= 40 e (r mean|u| + |z|)                    (mean: 32 e mean|u|; r and the products: 8 e more, 16 e of |z| for the variance)
and the gradient at x', t = r2 (dy w2 - z2 c2 - c1) + dx' with c2 = mean(dy w2 z2), c1 = mean(dy w2),
    |dt| <= 48 e r2 (|dy w2| + m1 + |z2| m2) + r2 (|dz2| m2 + |z2| mean(|dy w2| |dz2|)) + 2 e |dx'|,      m1 = mean|dy w2|, m2 = mean|dy w2 z2|.
A sum over rows adds its terms' errors and its own: every term takes part in at most n additions, n = rows of a block in turn + a tree.  Blocks: at least 256
of them share the rows evenly, but a block takes whole gate groups where there are more groups than blocks: n <= 2 rows / 256 + rows of a group + 64, and no more
than rows + 64.  (Rows that threads of a block share make n smaller yet.)  The gate's single value also sums C products a row, 16 of them in a thread's own order."""
import torch

E32 = 2.0 ** -24


def column_sums(t, kind, alpha, eps, rows_per_group, x_new, dx_given):
    """name -> (value, bound, terms [rows, C] or None for the last: the single gate's terms).  t: x, h, gate, w1, b1, w2, b2, dy, dxn (or None)."""
    D = lambda v: None if v is None else v.double()
    h, gate, w1, b1, w2, b2, dy = (D(t[n]) for n in ("h", "gate", "w1", "b1", "w2", "b2", "dy"))
    xn = x_new.double()
    rows, C = h.shape

    def hat(u):
        c = u - u.mean(1, keepdim=True) if kind == "layer" else u
        r = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
        z = c * r
        return z, r, 40 * E32 * ((r * u.abs().mean(1, keepdim=True) if kind == "layer" else 0.0) + z.abs())
    z1, r1, dz1 = hat(h)
    z2, r2, dz2 = hat(xn)
    g = torch.ones(1, 1, dtype=torch.float64, device=h.device) if gate is None else gate
    group = rows
    if gate is not None and gate.dim() == 2:
        g = gate.repeat_interleave(rows_per_group, 0)[:rows]
        group = min(rows, rows_per_group)
    n = z1 * w1 + (0.0 if b1 is None else b1)
    dn = dz1 * w1.abs() + 2 * E32 * (n.abs() + (z1 * w1).abs())
    a = dy * w2
    c1, c2 = (a.mean(1, keepdim=True) if kind == "layer" else 0.0), (a * z2).mean(1, keepdim=True)
    m1, m2 = (a.abs().mean(1, keepdim=True) if kind == "layer" else 0.0), (a * z2).abs().mean(1, keepdim=True)
    dx = 0.0 if not dx_given else t["dxn"].double()
    tt = r2 * (a - z2 * c2 - c1) + dx
    dt = 48 * E32 * r2 * (a.abs() + m1 + z2.abs() * m2) + r2 * (dz2 * m2 + z2.abs() * (a.abs() * dz2).mean(1, keepdim=True)) + 2 * E32 * abs(dx)
    ag, ab = g.abs(), None
    terms = {"post_w": (tt * g * z1, dt * ag * z1.abs() + (tt * g).abs() * dz1), "post_b": ((tt * g).expand(rows, C), (dt * ag).expand(rows, C)),
             "pre_w": (dy * z2, dy.abs() * dz2), "pre_b": (dy, torch.zeros_like(dy)), "gate": (tt * n, dt * n.abs() + tt.abs() * dn)}
    if b1 is None:
        terms.pop("post_b")
    if b2 is None:
        terms.pop("pre_b")
    if gate is None:
        terms.pop("gate")
    whole = 2 * rows // 256 + (group if gate is not None and gate.dim() == 2 else 0) + 64
    adds = min(rows + 64, whole)
    out = {}
    for name, (v, err) in terms.items():
        if name == "gate" and gate.dim() == 2:
            parts = [(p, q) for p, q in zip(v.split(rows_per_group), err.split(rows_per_group))]
            val = torch.stack([p.sum(0) for p, _ in parts])
            bound = torch.stack([q.sum(0) + (min(group, adds) + 64) * E32 * p.abs().sum(0) for p, q in parts])
        elif name == "gate" and gate.numel() == 1:
            val, bound = v.sum().view(gate.shape), (err.sum() + 24 * E32 * v.abs().sum()).view(gate.shape)      # (compensated over a thread's rows)
        else:
            val, bound = v.sum(0), err.sum(0) + adds * E32 * v.abs().sum(0)
        out[name] = (val, bound, v)
    return out
