"""The sequence operators as they are measured: cases, inputs, the plain forms, the framework's calls and 64-bit results.

Three operators of transformer blocks over ragged token sequences:

  attn     attention with a learned relative position bias by buckets, forward alone or forward + backward (dQ, dK, dV and the bias
           table's gradient, the probabilities recomputed)
  decode   the same attention for one new token per sequence over a key / value cache
  join     norm after a block, gate, scaled residual sum, norm before the next block, forward alone or forward + backward

`own` selects the framework's calls; without it `run` computes the plain forms in 32 bits with elementary torch operations.
"""
import functools
import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


# ------------------------------------------------------------------------------------------------ cases

def _attn(name, seqs, shortest, longest, heads, kv_heads, dim, causal, train, masked, buckets, far):
    return dict(name=name, op="attn", seqs=seqs, shortest=shortest, longest=longest, heads=heads, kv_heads=kv_heads, dim=dim,
                causal=causal, train=train, masked=masked, buckets=buckets, far=far)


def _decode(name, seqs, shortest, longest, heads, kv_heads, dim, buckets, far):
    return dict(name=name, op="decode", seqs=seqs, shortest=shortest, longest=longest, heads=heads, kv_heads=kv_heads, dim=dim,
                causal=True, buckets=buckets, far=far)


def _join(name, rows, width, kind, stream, gate, group, post_bias, train, alpha):
    return dict(name=name, op="join", rows=rows, width=width, kind=kind, stream=stream, gate=gate, group=group,
                post_bias=post_bias, train=train, alpha=alpha)


def listed():
    return [
        # a batch of four questions of up to 14 words through a question encoder's layer: launches and latency
        _attn("attn_questions_train", 4, 3, 14, 8, 8, 64, False, True, False, 32, 128),
        # clips of up to ten frames of 49 audio tokens, some tokens masked and one clip with no token left
        _attn("attn_clips_train", 32, 131, 490, 12, 12, 64, False, True, True, 32, 128),
        # ten frames of 197 video tokens as one sequence, scored without gradients, 96-wide heads
        _attn("attn_frames_fwd", 8, 985, 1970, 8, 8, 96, False, False, False, 32, 128),
        # a decoder trained on documents of uneven length: causal, four query heads to a key / value head
        _attn("attn_documents_train", 3, 1311, 4097, 32, 8, 128, True, True, False, 32, 128),
        # one recording of 16384 tokens, far beyond the last bucket's border
        _attn("attn_recording_train", 1, 16384, 16384, 16, 16, 64, False, True, False, 64, 800),
        # one dialogue: the next token after some hundreds
        _decode("decode_single", 1, 701, 701, 12, 12, 64, 32, 128),
        # a server's batch at mixed ages
        _decode("decode_batch", 64, 1, 4096, 32, 8, 128, 32, 128),
        # few very long contexts
        _decode("decode_long", 8, 20011, 65536, 32, 8, 128, 32, 128),
        # the class tokens and prompts of a small batch
        _join("join_small_train", 98, 512, "layer", "f32", "one", 0, True, True, 1.0),
        # the tokens of 32 clips x 10 frames x 196 patches with one gate for the adapter's branch
        _join("join_clips_train", 62720, 512, "layer", "f32", "one", 0, True, True, 1.0),
        # frames of 197 tokens, each frame with gates of its own (conditioned on the other modality)
        _join("join_frames_train", 15760, 768, "rms", "bf16", "group", 197, False, True, 1.0),
        # a prompt of 16384 tokens through a wide model, one gate for each channel
        _join("join_prompt_fwd", 16384, 4096, "rms", "bf16", "channel", 0, False, False, 0.75),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "decode", "join", "join"])
    if op == "join":
        train = rng.random() < 0.6
        width = 8 * _log_int(rng, 4, 640)
        rows = max(1, min(_log_int(rng, 1, 80000), (1 << 25) // width))
        gate = rng.choice(["none", "one", "channel", "group"])
        group = _log_int(rng, 1, 400) if gate == "group" else 0
        kind = rng.choice(["layer", "rms"])
        return dict(op="join", rows=rows, width=width, kind=kind, stream=rng.choice(["f32", "bf16"]), gate=gate, group=group,
                    post_bias=kind == "layer" and rng.random() < 0.5, train=train, alpha=rng.choice([1.0, 0.75, 1.5]))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 7])
    dim = rng.choice([32, 64, 96, 128])
    buckets, far = rng.choice([(32, 128), (16, 40), (64, 800), (12, 100)])
    if op == "decode":
        longest = _log_int(rng, 1, 40000)
        seqs = max(1, min(_log_int(rng, 1, 200), (1 << 28) // (longest * kv_heads * dim)))
        return dict(op="decode", seqs=seqs, shortest=rng.randint(1, longest), longest=longest, heads=heads, kv_heads=kv_heads,
                    dim=dim, causal=True, buckets=buckets, far=far)
    longest = _log_int(rng, 1, 6000)
    seqs = max(1, min(_log_int(rng, 1, 48), int(6e8 / (longest * longest * heads))))
    return dict(op="attn", seqs=seqs, shortest=rng.randint(1, longest), longest=longest, heads=heads, kv_heads=kv_heads, dim=dim,
                causal=rng.random() < 0.5, train=rng.random() < 0.7, masked=rng.random() < 0.4, buckets=buckets, far=far)


def _lengths(case):
    """Lengths between the shortest and the longest, spread evenly and out of order; the longest is always there."""
    s, lo, hi = case["seqs"], case["shortest"], case["longest"]
    even = [hi - ((hi - lo) * i) // max(1, s - 1) for i in range(s)]
    step = next(d for d in (7, 5, 3, 2, 1) if math.gcd(d, s) == 1)
    return [even[(i * step) % s] for i in range(s)]


def work(case):
    if case["op"] == "join":
        r, c = case["rows"], case["width"]
        x = 4 if case["stream"] == "f32" else 2
        fwd = r * c * (2 + x + x + 2)                       # h, stream in, stream out, normalised out
        bwd = r * c * (2 + x + x + 2 + x + 2)               # dy, d stream, stream, h in; d stream, dh out
        return {"bytes": fwd + (bwd if case["train"] else 0), "flops": r * c * (14 + (30 if case["train"] else 0))}
    d, h, hk = case["dim"], case["heads"], case["kv_heads"]
    lens = _lengths(case)
    n = sum(lens)
    if case["op"] == "decode":
        return {"bytes": 2 * n * hk * d * 2 + 2 * len(lens) * h * d * 2, "flops": 4 * n * h * d}
    live = lens[:-1] if case["masked"] else lens
    pairs = sum(m * (m + 1) // 2 if case["causal"] else m * m for m in live)
    fwd = 2 * n * (2 * h + 2 * hk) * d + 4 * n * h
    bwd = 2 * n * (4 * h + 4 * hk) * d
    return {"bytes": fwd + (bwd if case["train"] else 0), "flops": (4 + (10 if case["train"] else 0)) * pairs * h * d}


# ------------------------------------------------------------------------------------------------ inputs

def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=BF16, std=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype).mul_(std).add_(mean)

    if case["op"] == "join":
        r, c = case["rows"], case["width"]
        stream = F32 if case["stream"] == "f32" else BF16
        t = {"x": normal(r, c, dtype=stream, std=2.0), "h": normal(r, c, std=1.5)}
        t["post_w"], t["pre_w"] = normal(c, dtype=F32, std=0.2, mean=1.0), normal(c, dtype=F32, std=0.2, mean=1.0)
        layer = case["kind"] == "layer"
        t["post_b"] = normal(c, dtype=F32, std=0.2) if case["post_bias"] else None
        t["pre_b"] = normal(c, dtype=F32, std=0.2) if layer else None
        shape = {"none": None, "one": (1,), "channel": (c,), "group": (-(-r // max(1, case["group"])), c)}[case["gate"]]
        t["gate"] = normal(*shape, dtype=F32, std=0.5) if shape else None
        if case["train"]:
            t["dy"], t["dx_out"] = normal(r, c), normal(r, c, dtype=stream)
        return t
    d, h, hk = case["dim"], case["heads"], case["kv_heads"]
    lens = _lengths(case)
    t = {"table": normal(case["buckets"], h, dtype=F32), "lens": lens}
    if case["op"] == "decode":
        s, cap = len(lens), case["longest"]
        t["q"] = normal(s, h * d)
        t["k"], t["v"] = normal(s, cap, hk * d), normal(s, cap, hk * d)
        t["len"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return t
    n = sum(lens)
    qkv = normal(n, (h + 2 * hk) * d)                       # the fused projection's output; q, k and v are column slices of it
    t["q"], t["k"], t["v"] = qkv[:, :h * d], qkv[:, h * d:(h + hk) * d], qkv[:, (h + hk) * d:]
    ends = [0]
    for m in lens:
        ends.append(ends[-1] + m)
    t["ends"] = ends
    t["cu"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    t["mask"] = None
    if case["masked"]:
        t["mask"] = torch.rand(n, generator=g, device="cuda") >= 0.1
        t["mask"][ends[-2]:] = False
    if case["train"]:
        t["do"] = normal(n, h * d)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, "t": t}
    if case["op"] != "join":
        state["borders"] = torch.tensor(_borders(case["buckets"], case["far"], case["causal"]), device="cuda")
    if own:
        from stgcma import kernels
        if case["op"] != "join":
            state["geom"] = kernels.RelGeom(case["heads"], case["dim"], kv_heads=case["kv_heads"], num_buckets=case["buckets"],
                                            max_distance=case["far"], causal=case["causal"], device="cuda")
        if case.get("train"):
            leaves = ["q", "k", "v", "table"] if case["op"] == "attn" else ["x", "h", "gate", "post_w", "post_b", "pre_w", "pre_b"]
            state["leaves"] = {n: t[n].detach().requires_grad_(True) for n in leaves if t[n] is not None}
    return state


# ------------------------------------------------------------------------------------------------ plain forms

def _borders(buckets, far, causal):
    """Smallest distance of each bucket of one side: single distances first, then borders evenly spaced in the logarithm up to `far`,
    found with whole numbers so that a distance on a border falls on one side for good."""
    half = buckets if causal else buckets // 2
    single = half // 2
    steps = half - single
    borders = list(range(single))
    for t in range(steps):
        d = single
        while d ** steps * single ** t < far ** t * single ** steps:
            d += 1
        borders.append(d)
    return borders


def _buckets(state, nq, nk, device):
    case = state["case"]
    rel = torch.arange(nk, device=device)[None, :] - (torch.arange(nq, device=device)[:, None] + (nk - nq))
    b = torch.bucketize(rel.abs(), state["borders"], right=True) - 1
    return (b if case["causal"] else b + (rel > 0) * (case["buckets"] // 2)), rel


def _plain_attn(state):
    case, t = state["case"], state["t"]
    d, h, hk = case["dim"], case["heads"], case["kv_heads"]
    rep, scale, train = h // hk, d ** -0.5, case["train"]
    n = t["q"].shape[0]
    out = {"o": torch.zeros(n, h * d, dtype=BF16, device="cuda")}
    if train:
        out["dq"] = torch.zeros_like(out["o"])
        out["dk"], out["dv"] = (torch.zeros(n, hk * d, dtype=BF16, device="cuda") for _ in range(2))
        dtable = torch.zeros(case["buckets"], h, dtype=F64, device="cuda")
    else:
        out["lse"] = torch.zeros(h, n, dtype=F32, device="cuda")
    for s, m in enumerate(t["lens"]):
        lo = t["ends"][s]
        rows = slice(lo, lo + m)
        bucket, rel = _buckets(state, m, m, "cuda")
        keep = torch.ones(1, m, dtype=torch.bool, device="cuda") if t["mask"] is None else t["mask"][None, rows]
        if case["causal"]:
            keep = keep & (rel <= 0)
        group = max(1, min(hk, (1 << 28) // (rep * m * m)))
        for j in range(0, hk, group):
            hs, ks = slice(j * rep, min(hk, j + group) * rep), slice(j, min(hk, j + group))
            q = t["q"][rows].float().view(m, h, d)[:, hs].transpose(0, 1)
            k0, v0 = (t[x][rows].float().view(m, hk, d)[:, ks].transpose(0, 1) for x in ("k", "v"))
            k, v = k0.repeat_interleave(rep, 0), v0.repeat_interleave(rep, 0)
            x = torch.matmul(q, k.transpose(1, 2)) * scale + t["table"][:, hs].t()[:, bucket]
            x = torch.where(keep, x, -math.inf)
            top = x.amax(-1, keepdim=True)
            top = torch.where(top == -math.inf, 0.0, top)
            p = torch.exp(x - top)
            total = p.sum(-1, keepdim=True)
            p = torch.where(total > 0, p / total, 0.0)
            out["o"][rows].view(m, h, d)[:, hs] = torch.matmul(p, v).transpose(0, 1).to(BF16)
            if not train:
                out["lse"][hs, rows] = (top + torch.log(total)).squeeze(-1)
                continue
            do = t["do"][rows].float().view(m, h, d)[:, hs].transpose(0, 1)
            dp = torch.matmul(do, v.transpose(1, 2))
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            heads = p.shape[0]
            out["dq"][rows].view(m, h, d)[:, hs] = (torch.matmul(ds, k) * scale).transpose(0, 1).to(BF16)
            dk = (torch.matmul(ds.transpose(1, 2), q) * scale).view(-1, rep, m, d).sum(1)
            dv = torch.matmul(p.transpose(1, 2), do).view(-1, rep, m, d).sum(1)
            out["dk"][rows].view(m, hk, d)[:, ks] = dk.transpose(0, 1).to(BF16)
            out["dv"][rows].view(m, hk, d)[:, ks] = dv.transpose(0, 1).to(BF16)
            # sums along the diagonals: rows upside down, one element more to each row, and the columns are the diagonals
            skew = torch.zeros(heads, m, 2 * m, device="cuda")
            skew[:, :, :m] = ds.flip(1)
            skew = skew.view(heads, -1)[:, :m * (2 * m - 1)].view(heads, m, 2 * m - 1).sum(1, dtype=F64)
            diag = torch.arange(2 * m - 1, device="cuda") - (m - 1)
            near = torch.bucketize(diag.abs(), state["borders"], right=True) - 1
            if not case["causal"]:
                near = near + (diag > 0) * (case["buckets"] // 2)
            hot = (near[:, None] == torch.arange(case["buckets"], device="cuda")).to(F64)
            dtable[:, hs] += torch.matmul(skew, hot).t()
    if train:
        out["dtable"] = dtable.float()
    return out


def _plain_decode(state):
    case, t = state["case"], state["t"]
    d, h, hk = case["dim"], case["heads"], case["kv_heads"]
    s, cap = t["k"].shape[:2]
    q = t["q"].float().view(s, hk, h // hk, d)
    k, v = (t[x].float().view(s, cap, hk, d).permute(0, 2, 1, 3) for x in ("k", "v"))
    x = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5                      # [sequence, kv head, query head, position]
    pos = torch.arange(cap, device="cuda")
    back = t["len"][:, None].long() - 1 - pos
    bucket = torch.bucketize(back.clamp(min=0), state["borders"], right=True) - 1
    bias = t["table"][bucket].permute(0, 2, 1).reshape(s, hk, h // hk, cap)
    x = torch.where((back >= 0)[:, None, None], x + bias, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p, v).reshape(s, h * d).to(BF16)


def _norm(x, w, b, kind, eps=1e-5):
    mean = x.mean(-1, keepdim=True) if kind == "layer" else 0.0
    c = x - mean
    hat = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + eps)
    y = hat * w
    return (y if b is None else y + b), hat


def _norm_back(dy, x, hat, w, kind, eps=1e-5):
    mean = x.mean(-1, keepdim=True) if kind == "layer" else 0.0
    c = x - mean
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + eps)
    g = dy * w
    dx = g - hat * (g * hat).mean(-1, keepdim=True)
    return r * (dx - g.mean(-1, keepdim=True) if kind == "layer" else dx)


def _rows_of(gate, case):
    if gate is None:
        return 1.0
    if case["gate"] == "group":
        return gate.repeat_interleave(case["group"], 0)[:case["rows"]]
    return gate


def _plain_join(state):
    case, t = state["case"], state["t"]
    x, h = t["x"].float(), t["h"].float()
    kind, alpha = case["kind"], case["alpha"]
    n, hat1 = _norm(h, t["post_w"], t["post_b"], kind)
    gate = _rows_of(t["gate"], case)
    new = (alpha * x + gate * n).to(t["x"].dtype)           # the stream is stored in its own type, and the next norm reads what is stored
    z = new.float()
    y, hat2 = _norm(z, t["pre_w"], t["pre_b"], kind)
    out = {"x": new, "y": y.to(BF16)}
    if not case["train"]:
        return out
    dy = t["dy"].float()
    total = t["dx_out"].float() + _norm_back(dy, z, hat2, t["pre_w"], kind)
    dn = total * gate
    out["dx"] = (alpha * total).to(t["x"].dtype)
    out["dh"] = _norm_back(dn, h, hat1, t["post_w"], kind).to(BF16)
    if t["gate"] is not None:
        dg = total * n
        if case["gate"] == "one":
            out["dgate"] = dg.sum(dtype=F64).float().view(1)
        elif case["gate"] == "channel":
            out["dgate"] = dg.sum(0, dtype=F64).float()
        else:
            groups, size = t["gate"].shape[0], case["group"]
            full = torch.zeros(groups * size, dg.shape[1], device="cuda")
            full[:dg.shape[0]] = dg
            out["dgate"] = full.view(groups, size, -1).sum(1, dtype=F64).float()
    out["dpost_w"] = (dn * hat1).sum(0, dtype=F64).float()
    if t["post_b"] is not None:
        out["dpost_b"] = dn.sum(0, dtype=F64).float()
    out["dpre_w"] = (dy * hat2).sum(0, dtype=F64).float()
    if t["pre_b"] is not None:
        out["dpre_b"] = dy.sum(0, dtype=F64).float()
    return out


# ------------------------------------------------------------------------------------------------ the framework's calls

def _own_attn(state):
    from stgcma import kernels, ops_seq
    case, t, geom = state["case"], state["t"], state["geom"]
    if not case["train"]:
        o, lse = kernels.relattn_fwd(geom, t["q"], t["k"], t["v"], t["table"], t["cu"], max_q=case["longest"], key_mask=t["mask"])
        return {"o": o, "lse": lse}
    a = state["leaves"]
    o = ops_seq.rel_attention(a["q"], a["k"], a["v"], a["table"], geom, t["cu"], max_q=case["longest"], key_mask=t["mask"])
    dq, dk, dv, dtable = torch.autograd.grad(o, [a["q"], a["k"], a["v"], a["table"]], t["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}


def _own_decode(state):
    from stgcma import kernels
    t = state["t"]
    return kernels.relattn_decode(state["geom"], t["q"], t["k"], t["v"], t["table"], t["len"])


def _own_join(state):
    from stgcma import kernels, ops_seq
    case, t = state["case"], state["t"]
    names = ["x", "h", "gate", "post_w", "post_b", "pre_w", "pre_b"]
    how = dict(kind=case["kind"], alpha=case["alpha"], rows_per_group=case["group"] or None)
    if not case["train"]:
        new, y, _ = kernels.norm_join_fwd(*[t[n] for n in names], want_stats=False, **how)
        return {"x": new, "y": y}
    a = state["leaves"]
    new, y = ops_seq.norm_join(*[a.get(n) for n in names], **how)
    grads = torch.autograd.grad([new, y], list(a.values()), [t["dx_out"], t["dy"]])
    out = {"x": new.detach(), "y": y.detach()}
    out.update({"d" + n: g for n, g in zip(a, grads)})
    return {k: out[k] for k in ("x", "y", "dx", "dh", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b") if k in out}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attn": _own_attn, "decode": _own_decode, "join": _own_join}[op](state)
    return {"attn": _plain_attn, "decode": _plain_decode, "join": _plain_join}[op](state)


# ------------------------------------------------------------------------------------------------ 64-bit results from the definitions

@functools.lru_cache(maxsize=None)
def _bucket_of(distance, buckets, far, causal):
    """Bucket of a signed distance (key position - query position), from the definition, with whole numbers."""
    half = buckets if causal else buckets // 2
    first = half // 2
    d = abs(distance)
    b = min(d, first)
    while b >= first and b < half - 1 and d ** (half - first) * first ** (b + 1 - first) >= far ** (b + 1 - first) * first ** (half - first):
        b += 1
    return b + (half if not causal and distance > 0 else 0)


def _bias_by_distance(case, table, n):
    """[heads, 2 n - 1] bias of the distances -(n - 1) .. n - 1, and their buckets."""
    lim = min(n - 1, case["far"])
    ids = [_bucket_of(x, case["buckets"], case["far"], case["causal"]) for x in range(-lim, lim + 1)]
    ids = [ids[0]] * (n - 1 - lim) + ids + [ids[-1]] * (n - 1 - lim)
    ids = torch.tensor(ids, device="cuda")
    return table.double()[ids].t(), ids


def _exact_attn(case, t):
    d, h, hk = case["dim"], case["heads"], case["kv_heads"]
    n = t["q"].shape[0]
    train = case["train"]
    o = torch.zeros(n, h, d, dtype=F64, device="cuda")
    lse = torch.full((h, n), -math.inf, dtype=F64, device="cuda")
    dq, dk, dv = torch.zeros_like(o), torch.zeros(n, hk, d, dtype=F64, device="cuda"), torch.zeros(n, hk, d, dtype=F64, device="cuda")
    dtable = torch.zeros(case["buckets"], h, dtype=F64, device="cuda")
    for s, m in enumerate(t["lens"]):
        a, b = t["ends"][s], t["ends"][s] + m
        bias, ids = _bias_by_distance(case, t["table"], m)
        at = torch.arange(m, device="cuda")
        which = at[None, :] - at[:, None] + (m - 1)
        hidden = torch.zeros(m, m, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= at[None, :] > at[:, None]
        if t["mask"] is not None:
            hidden |= ~t["mask"][a:b][None, :]
        dead = hidden.all(1)
        for i in range(h):
            j = i // (h // hk)
            q = t["q"][a:b, i * d:(i + 1) * d].double()
            k, v = (t[x][a:b, j * d:(j + 1) * d].double() for x in ("k", "v"))
            x = (q @ k.t()) / math.sqrt(d) + bias[i][which]
            x.masked_fill_(hidden, -math.inf)
            z = torch.logsumexp(x, 1)
            x.sub_(z[:, None]).exp_()
            x[dead] = 0.0
            lse[i, a:b] = z
            o[a:b, i] = x @ v
            if not train:
                continue
            g = t["do"][a:b, i * d:(i + 1) * d].double()
            dv[a:b, j] += x.t() @ g
            dx = g @ v.t()
            dx.sub_((g * o[a:b, i]).sum(1, keepdim=True)).mul_(x)
            dq[a:b, i] = dx @ k / math.sqrt(d)
            dk[a:b, j] += dx.t() @ q / math.sqrt(d)
            member = ids[:, None] == torch.arange(case["buckets"], device="cuda")
            dtable[:, i] += _diagonals(dx) @ member.double()
    out = {"o": o.flatten(1)}
    if not train:
        out["lse"] = lse
        return out
    out.update(dq=dq.flatten(1), dk=dk.flatten(1), dv=dv.flatten(1), dtable=dtable)
    return out


def _diagonals(a):
    """Sums of a square matrix's diagonals, lowest first, through a window whose rows step one element less than a row's length."""
    m = a.shape[0]
    wide = torch.zeros(m, 3 * m - 2, dtype=a.dtype, device=a.device)
    wide[:, m - 1:2 * m - 1] = a
    return wide.as_strided((m, 2 * m - 1), (3 * m - 1, 1)).sum(0)


def _exact_decode(case, t):
    d, h, hk = case["dim"], case["heads"], case["kv_heads"]
    o = torch.zeros(len(t["lens"]), h, d, dtype=F64, device="cuda")
    for s, m in enumerate(t["lens"]):
        bias, _ = _bias_by_distance(case, t["table"], m)
        q = t["q"][s].double().view(hk, h // hk, d)
        k, v = (t[x][s, :m].double().view(m, hk, d).transpose(0, 1) for x in ("k", "v"))
        x = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(d) + bias[:, :m].reshape(hk, h // hk, m)
        o[s] = torch.bmm(torch.softmax(x, -1), v.contiguous()).view(h, d)
    return o.flatten(1)


def _exact_join(case, t):
    eps = 1e-5
    layer = case["kind"] == "layer"
    x, h = t["x"].double(), t["h"].double()
    pw, qw = t["post_w"].double(), t["pre_w"].double()

    def hat_of(u):
        u = u - u.mean(1, keepdim=True) if layer else u
        r = 1.0 / torch.sqrt(u.square().mean(1, keepdim=True) + eps)
        return u * r, r

    def through(dhat, hat, r):                               # gradient of the normalisation
        out = dhat - hat * (dhat * hat).mean(1, keepdim=True)
        return r * (out - dhat.mean(1, keepdim=True)) if layer else r * out

    hat1, r1 = hat_of(h)
    n = hat1 * pw + (t["post_b"].double() if t["post_b"] is not None else 0.0)
    gate = t["gate"].double() if t["gate"] is not None else torch.ones(1, dtype=F64, device="cuda")
    who = None
    if case["gate"] == "group":
        who = torch.arange(case["rows"], device="cuda") // case["group"]
        gate = gate[who]
    new = case["alpha"] * x + gate * n
    stored = new.to(t["x"].dtype).double()                   # the definition: the next norm reads the stream as it is stored
    hat2, r2 = hat_of(stored)
    y = hat2 * qw + (t["pre_b"].double() if t["pre_b"] is not None else 0.0)
    out = {"x": new, "y": y}
    if not case["train"]:
        return out
    dy = t["dy"].double()
    total = t["dx_out"].double() + through(dy * qw, hat2, r2)
    out["dx"] = case["alpha"] * total
    out["dh"] = through(total * gate * pw, hat1, r1)
    if t["gate"] is not None:
        if who is not None:
            full = torch.zeros(t["gate"].shape[0] * case["group"], case["width"], dtype=F64, device="cuda")
            full[:case["rows"]] = total * n
            out["dgate"] = full.view(-1, case["group"], case["width"]).sum(1)
        else:
            out["dgate"] = (total * n).sum().view(1) if case["gate"] == "one" else (total * n).sum(0)
    out["dpost_w"] = (total * gate * hat1).sum(0)
    if t["post_b"] is not None:
        out["dpost_b"] = (total * gate).expand_as(n).sum(0)
    out["dpre_w"] = (dy * hat2).sum(0)
    if t["pre_b"] is not None:
        out["dpre_b"] = dy.sum(0)
    return out


def exact(case, seed):
    t = _inputs(case, seed)
    return {"attn": _exact_attn, "decode": _exact_decode, "join": _exact_join}[case["op"]](case, t)
