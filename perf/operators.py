"""The float attention operators as a program calls them: the norms of queries
and keys for each head with the position rotation, attention with shaped
scores (tanh cap, bias by distance, documents, prefix and window masks, shared
key heads), and the learned bias by distance buckets with its gradient; each
forward alone, as serving runs it, and with its backward, as training does.

`run` makes the framework's calls where `own` is true and computes the same in
elementary 32-bit operations otherwise; `exact` has the definitions in 64
bits, sequence by sequence, with differentiated gradients.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BUCKETS, REACH = 32, 128  # learned bias: buckets, distance past which the last one holds
THETA = 10000.0
EPS = 1e-6


def _attend(**kw):
    base = dict(op="attend", type="bf16", heads=12, kv_heads=12, dim=64, seqs=1, lo=15, hi=15, one=False, cap=0.0,
                slopes=False, table=False, docs=False, causal=False, prefix=False, window=-1, train=False)
    return dict(base, **kw)


def _rope(**kw):
    base = dict(op="rope", type="bf16", heads=12, kv_heads=12, dim=64, seqs=1, lo=15, hi=15, norm="rms", rot=64,
                pairs="halves", train=False)
    return dict(base, **kw)


def listed():
    return [
        # one short query on the small shape: the smallest call, latency only
        _rope(name="rope_query", heads=4, kv_heads=4),
        # the headline batch's lengths on the base shape, Q and K slices of
        # the packed QKV rows
        _rope(name="rope_base", seqs=256, lo=64, hi=512),
        # a training step's half on shared key heads: LayerNorm a head, half
        # of it rotated, neighbours paired
        _rope(name="rope_train", type="f16", heads=16, kv_heads=4, dim=128, seqs=8, lo=2048, hi=2048, norm="layer",
              pairs="neighbours", train=True),
        # the same short query's attention, in the framework's float32
        _attend(name="attend_query", type="f32", heads=4, kv_heads=4, slopes=True),
        # the headline batch through a local layer with capped scores
        _attend(name="attend_base", seqs=256, lo=64, hi=512, cap=30.0, window=64),
        # four documents of the longest length, a bidirectional prefix each
        _attend(name="attend_long", seqs=4, lo=8192, hi=8192, causal=True, prefix=True),
        # a single new token a sequence over all its keys, as serving asks
        _attend(name="attend_token", type="f16", heads=16, kv_heads=4, dim=128, seqs=32, lo=512, hi=8192, one=True,
                slopes=True),
        # a padded batch at 512 tokens a row, several documents in each row
        _attend(name="attend_padded", type="f16", heads=6, kv_heads=6, seqs=64, lo=512, hi=512, cap=50.0, docs=True),
        # a training step over packed documents, causal, shared key heads
        _attend(name="attend_train", heads=16, kv_heads=4, dim=128, seqs=8, lo=2048, hi=2048, docs=True, causal=True,
                cap=50.0, train=True),
        # the headline batch with a learned bias in place of the rotation
        _attend(name="bias_base", seqs=256, lo=64, hi=512, table=True),
        # a float32 training step with the bias' gradient, ragged lengths
        _attend(name="bias_train", type="f32", heads=6, kv_heads=6, dim=48, seqs=24, lo=33, hi=300, table=True,
                train=True),
        # norms, rotation, biased attention and all their gradients in one
        # training step, as a layer runs them
        _attend(name="layer_train", op="layer", seqs=48, lo=64, hi=512, table=True, train=True, norm="rms", rot=64,
                pairs="halves"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attend", "attend", "attend", "layer"])
    dim = rng.choice([64, 64, 128, 128, 32, 48, 80, 96])
    kv = rng.choice([1, 2, 3, 4, 6])
    heads = kv * rng.choice([1, 1, 2, 4])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.4
    hi = _log(rng, 1, 8192 if not train and kind != "f32" else 2048)
    lo = max(1, min(hi, _log(rng, max(1, hi // 16), hi)))
    one = op == "attend" and not train and rng.random() < 0.2
    # rows by the largest listed case: its score matrix, or its rows
    most = 98304 if op == "rope" or one else max(hi, min(65536, int(4.0e8 / heads / hi)))
    seqs = max(1, min(256, 2 * _log(rng, hi, max(hi, most)) // (lo + hi)))
    norm = dict(norm=rng.choice(["rms", "rms", "layer", "none"]), rot=rng.choice([dim // 16 * 16, 32, 16]),
                pairs=rng.choice(["halves", "halves", "neighbours"]))
    size = dict(type=kind, heads=heads, kv_heads=kv, dim=dim, seqs=seqs, lo=lo, hi=hi, train=train)
    if op == "rope":
        return _rope(**size, **norm)
    causal = rng.random() < 0.4
    c = _attend(op=op, **size, one=one, cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.25,
                table=rng.random() < 0.4, docs=not one and rng.random() < 0.3, causal=causal,
                prefix=causal and rng.random() < 0.5, window=-1 if rng.random() < 0.7 else _log(rng, 4, 512))
    return dict(c, **norm) if op == "layer" else c


# ---- what follows from a case alone: lengths, documents, prefixes ---------


def _layout(case):
    """Key lengths, query lengths, prefix lengths, and the document of each
    key row (None: no documents; -1: padding)."""
    rng = np.random.default_rng([case["seqs"], case["lo"], case["hi"], case["heads"]])
    k = rng.integers(case["lo"], case["hi"] + 1, size=case["seqs"])
    q = np.ones_like(k) if case.get("one") else k
    prefix = rng.integers(0, k // 2 + 1)
    docs = None
    if case.get("docs"):
        rows = []
        for n in k:
            cuts = np.sort(rng.integers(0, n, size=3))
            ids = np.searchsorted(cuts, np.arange(n), side="right")
            ids[n - int(rng.integers(0, n // 8 + 1)):] = -1  # the row's padding
            rows.append(ids)
        docs = np.concatenate(rows)
    return k, q, prefix, docs


def _buckets():
    """The bucket of each distance -REACH..REACH (key minus query): half of
    the buckets for each direction; the near half of those one distance each,
    the others on a logarithmic scale, its borders in whole numbers."""
    half, near = BUCKETS // 2, BUCKETS // 4
    steps = half - near
    out = []
    for d in range(-REACH, REACH + 1):
        a = abs(d)
        if a >= near:
            # the largest t with a >= near * (REACH / near) ** (t / steps)
            t = sum(a**steps * near**t >= near**steps * REACH**t for t in range(1, steps))
            a = near + t
        out.append(a + (half if d > 0 else 0))
    return np.array(out, np.int32)


def _pairs(case):
    """Visible (query, key) pairs of all sequences."""
    k, q, prefix, docs = _layout(case)
    total, at = 0, 0
    for n, m, pre in zip(k, q, prefix):
        p = np.arange(m) + n - m
        hi, lo = np.full(m, n - 1), np.zeros(m, np.int64)
        if case["causal"]:
            hi = np.minimum(hi, np.maximum(p, pre - 1) if case["prefix"] else p)
        if case["window"] >= 0:
            hi, lo = np.minimum(hi, p + case["window"]), np.maximum(lo, p - case["window"])
        if docs is None:
            total += int(np.maximum(0, hi - lo + 1).sum())
        else:
            d = docs[at:at + n]
            seen = np.concatenate([np.zeros((1, int(d.max(initial=0)) + 2), np.int64),
                                   np.cumsum(d[:, None] == np.arange(int(d.max(initial=0)) + 2), 0)])
            mine = d[n - m:]
            c = np.where(hi >= lo, seen[hi + 1, np.maximum(mine, 0)] - seen[lo, np.maximum(mine, 0)], 0)
            total += int(c[mine >= 0].sum())
        at += n
    return total


def work(case):
    k, q, _, _ = _layout(case)
    size = {"f32": 4}.get(case["type"], 2)
    d, hq, hk = case["dim"], case["heads"], case["kv_heads"]
    nq, nk = int(q.sum()), int(k.sum())
    rq, rk = nq * hq * d * size, nk * hk * d * size  # bytes of Q's rows, of K's
    out = {"bytes": 0, "flops": 0}
    if case["op"] in ("rope", "layer"):
        out["bytes"] += (5 if case["train"] else 2) * (rq + rk) + 8 * nk
        out["flops"] += (20 if case["train"] else 8) * (nq * hq + nk * hk) * d
    if case["op"] in ("attend", "layer"):
        out["bytes"] += 2 * rq + 2 * rk + 4 * nq * hq + 4 * (nq + nk) * bool(case["docs"])
        out["flops"] += 4 * d * hq * _pairs(case)
        if case["train"]:
            # dO, o, Q, K, V read again; dQ, dK, dV written
            out["bytes"] += 4 * rq + 4 * rk + 4 * nq * hq
            out["flops"] += 10 * d * hq * _pairs(case)
    return out


# ---- what a program holds before the call ----------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    k, q, prefix, docs = _layout(case)
    nq, nk = int(q.sum()), int(k.sum())

    def rows(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(t)

    def ints(a):
        return torch.from_numpy(np.asarray(a, np.int32)).cuda()

    s = {"case": case, "q_len": int(q.max()), "k_len": int(k.max())}
    s["offs"] = ints(np.concatenate([[0], np.cumsum(q)]))
    s["k_offs"] = ints(np.concatenate([[0], np.cumsum(k)])) if case.get("one") else None
    if case.get("one"):
        s["q"], s["k"], s["v"] = rows(nq, hq, d), rows(nk, hk, d), rows(nk, hk, d)
    else:  # heads of the packed rows that one projection wrote
        s["qkv"] = rows(nk, hq + 2 * hk, d)
        s["q"], s["k"], s["v"] = s["qkv"].split([hq, hk, hk], 1)
    if case["op"] in ("rope", "layer"):
        rot, longest = case["rot"], int(k.max())
        a = np.arange(longest)[:, None] * THETA ** (-np.arange(0, rot, 2) / rot)
        s["cos"], s["sin"] = (torch.from_numpy(f(a).astype(np.float32)).cuda() for f in (np.cos, np.sin))
        s["pos"] = ints(np.concatenate([np.arange(n) for n in k]))
        with_norm = case["norm"] != "none"
        # a trained layer's gammas have the type of its rows
        gt = t if case["op"] == "layer" else torch.float32
        s["q_gamma"], s["k_gamma"] = ((1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(gt) if with_norm else None
                                      for _ in range(2))
    if case["op"] in ("attend", "layer"):
        s["slopes"] = None
        if case["slopes"]:
            s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device="cuda")
        s["table"] = rows(BUCKETS, hq) if case["table"] else None
        s["buckets"] = ints(_buckets()) if case["table"] else None
        s["prefix"] = ints(prefix) if case["prefix"] else None
        s["docs"] = ints(docs) if docs is not None else None
    if case["train"]:
        if case["op"] == "rope":
            s["dq"], s["dk"] = rows(nq, hq, d), rows(nk, hk, d)
        else:
            s["do"] = rows(nq, hq, d)
    return s


# ---- the framework's calls --------------------------------------------------


def _own(s):
    from indecis_amd import attention

    c = s["case"]
    out = {}
    q, k = s["q"], s["k"]
    if c["op"] in ("rope", "layer"):
        norm = dict(pos=s["pos"], q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], norm=c["norm"], eps=EPS, pairs=c["pairs"])
        q, k = attention.qk_norm_rope(q, k, s["cos"], s["sin"], **norm)
        out["q"], out["k"] = q, k
        if c["op"] == "rope":
            if c["train"]:
                out["dq"], out["dk"], out["dq_gamma"], out["dk_gamma"] = attention.qk_norm_rope_backward(
                    s["dq"], s["dk"], s["q"], s["k"], s["cos"], s["sin"], **norm)
            return out
    shape = dict(cap=c["cap"], slopes=s["slopes"], table=s["table"], buckets=s["buckets"], docs=s["docs"],
                 causal=c["causal"], prefix=s["prefix"], window=c["window"])
    if not c["train"]:
        return dict(out, o=attention.attend(q, k, s["v"], s["offs"], s["k_offs"], **shape))
    out["o"], lse = attention.attend(q, k, s["v"], s["offs"], s["k_offs"], want_lse=True, **shape)
    dq, dk, out["dv"], out["dtable"] = attention.attend_backward(
        s["do"], q, k, s["v"], out["o"], lse, s["offs"], s["k_offs"], **shape)
    if c["op"] == "attend":
        out["lse"] = lse
    else:
        dq, dk, out["dq_gamma"], out["dk_gamma"] = attention.qk_norm_rope_backward(
            dq, dk, s["q"], s["k"], s["cos"], s["sin"], **norm)
    out["dq"], out["dk"] = dq, dk
    return out


# ---- the plain form ---------------------------------------------------------


def _normed(x, c):
    """x in 32 bits, centred and scaled, with its scale."""
    x = x.float()
    if c["norm"] == "none":
        return x, None
    if c["norm"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r, r


def _turn(y, cos, sin, c):
    """y with its first `rot` columns rotated by the rows' angles."""
    rot = c["rot"]
    if c["pairs"] == "halves":
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., rot:]], -1)
    a, b = y[..., 0:rot:2], y[..., 1:rot:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), y[..., rot:]], -1)


def _plain_rope(x, gamma, s):
    c = s["case"]
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    y, _ = _normed(x, c)
    return _turn(y if gamma is None else y * gamma.float(), cos, sin, c).to(x.dtype)


def _plain_rope_backward(dy, x, gamma, s):
    c = s["case"]
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    dy = _turn(dy.float(), cos, -sin, c)
    if c["norm"] == "none":
        return dy.to(x.dtype), None
    xh, r = _normed(x, c)
    dgamma = (dy * xh).sum((0, 1)).to(gamma.dtype)
    dy = dy * gamma.float()
    dx = dy - xh * (dy * xh).mean(-1, keepdim=True)
    if c["norm"] == "layer":
        dx = dx - dy.mean(-1, keepdim=True)
    return (dx * r).to(x.dtype), dgamma


def _padded(offs, n):
    """Row of each (sequence, position < n), and which of them are there."""
    at = offs[:-1, None].long() + torch.arange(n, device=offs.device)
    there = at < offs[1:, None]
    return torch.where(there, at, 0), there


def _plain_attend(q, k, v, s):
    """Forward over the batch padded to its longest sequence; what the
    backward needs is kept."""
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    k_offs = s["offs"] if s["k_offs"] is None else s["k_offs"]
    qi, q_there = _padded(s["offs"], s["q_len"])
    ki, k_there = _padded(k_offs, s["k_len"])

    def heads(x, at, there, times=1):  # [B][H][L][D] in 32 bits
        x = (x[at].float() * there[..., None, None]).transpose(1, 2)
        return (x if times == 1 else x.repeat_interleave(times, 1)).contiguous()

    qp, kp, vp = heads(q, qi, q_there), heads(k, ki, k_there, group), heads(v, ki, k_there, group)
    lens = (k_offs[1:] - k_offs[:-1]).long() - (s["offs"][1:] - s["offs"][:-1]).long()
    p = torch.arange(s["q_len"], device=q.device) + lens[:, None]  # [B][Lq]
    j = torch.arange(s["k_len"], device=q.device)
    dist = j - p[..., None]  # [B][Lq][Lk]
    see = q_there[..., None] & k_there[:, None]
    if c["causal"]:
        ahead = dist <= 0
        see &= ahead | (j < s["prefix"][:, None, None]) if c["prefix"] else ahead
    if c["window"] >= 0:
        see &= dist.abs() <= c["window"]
    if s["docs"] is not None:
        see &= (s["docs"][qi][..., None] == s["docs"][ki][:, None]) & (s["docs"][ki][:, None] >= 0)
    z = torch.matmul(qp, kp.transpose(2, 3)).mul_(c["dim"] ** -0.5)
    slope = None
    if c["cap"] > 0:
        th = torch.tanh(z / c["cap"])
        z, slope = th * c["cap"], 1 - th * th
    if s["slopes"] is not None:
        z = z - s["slopes"][:, None, None] * dist.abs()[:, None]
    where = None
    if s["table"] is not None:
        where = s["buckets"].long()[dist.clamp(-REACH, REACH) + REACH]
        z = z + s["table"].float().t()[:, where].transpose(0, 1)
    z = z.masked_fill_(~see[:, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    e = z.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = e.sum(-1, keepdim=True)
    e = e.div_(total.masked_fill(total == 0, 1.0))
    o = torch.matmul(e, vp)
    lse = (top + total.log()).squeeze(-1)  # [B][H][Lq]
    flat = o.transpose(1, 2)[q_there], lse.transpose(1, 2)[q_there].t().contiguous()
    return flat, dict(q=qp, k=kp, v=vp, p=e, slope=slope, where=where, qi=qi, q_there=q_there, k_there=k_there, o=o)


def _plain_attend_backward(do, s, m):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    do = (do[m["qi"]].float() * m["q_there"][..., None, None]).transpose(1, 2).contiguous()

    def shared(x):  # the sum over the heads that share a key head
        return x.unflatten(1, (c["kv_heads"], group)).sum(2).transpose(1, 2)[m["k_there"]]

    dv = shared(torch.matmul(m["p"].transpose(2, 3), do))
    dz = torch.matmul(do, m["v"].transpose(2, 3))
    dz = dz.sub_((do * m["o"]).sum(-1, keepdim=True)).mul_(m["p"])
    dtable = None
    if s["table"] is not None:
        # sums of many small terms: in 64 bits. As many queries as keys, so a
        # place has the same distance in every sequence
        here = m["where"][0].flatten()[:, None] == torch.arange(BUCKETS, device=do.device)
        dtable = (dz.sum(0, dtype=torch.float64).flatten(1) @ here.double()).t()
    if m["slope"] is not None:
        dz = dz.mul_(m["slope"])
    dz = dz.mul_(c["dim"] ** -0.5)
    dq = torch.matmul(dz, m["k"]).transpose(1, 2)[m["q_there"]]
    dk = shared(torch.matmul(dz.transpose(2, 3), m["q"]))
    return dq, dk, dv, dtable


def run(s):
    if own:
        return _own(s)
    c = s["case"]
    t = s["q"].dtype
    out = {}
    q, k = s["q"], s["k"]
    if c["op"] in ("rope", "layer"):
        q, k = _plain_rope(q, s["q_gamma"], s), _plain_rope(k, s["k_gamma"], s)
        out["q"], out["k"] = q, k
        if c["op"] == "rope":
            if c["train"]:
                out["dq"], out["dq_gamma"] = _plain_rope_backward(s["dq"], s["q"], s["q_gamma"], s)
                out["dk"], out["dk_gamma"] = _plain_rope_backward(s["dk"], s["k"], s["k_gamma"], s)
            return out
    (o, lse), kept = _plain_attend(q, k, s["v"], s)
    out["o"] = o.to(t)
    if not c["train"]:
        return out
    if c["op"] == "attend":
        out["lse"] = lse
    dq, dk, dv, dtable = _plain_attend_backward(s["do"], s, kept)
    dq, dk, out["dv"] = dq.to(t), dk.to(t), dv.to(t)
    out["dtable"] = None if dtable is None else dtable.to(t)
    if c["op"] == "layer":
        dq, out["dq_gamma"] = _plain_rope_backward(dq, s["q"], s["q_gamma"], s)
        dk, out["dk_gamma"] = _plain_rope_backward(dk, s["k"], s["k_gamma"], s)
    out["dq"], out["dk"] = dq, dk
    return out


# ---- the definitions in 64 bits ---------------------------------------------


def _exact_rope(x, gamma, s):
    c = s["case"]
    rot = c["rot"]
    if c["norm"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    if c["norm"] != "none":
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * gamma
    angle = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
    part = x[..., :rot]
    halves = c["pairs"] == "halves"
    two = part.unflatten(-1, (2, rot // 2)).transpose(-1, -2) if halves else part.unflatten(-1, (rot // 2, 2))
    two = torch.view_as_real(torch.view_as_complex(two.contiguous()) * angle)
    two = two.transpose(-1, -2) if halves else two
    return torch.cat([two.flatten(-2), x[..., rot:]], -1)


def _exact_sequence(q, k, v, b, s, prefix, docs, table):
    """One sequence's outputs and logarithms of sums, heads first."""
    c = s["case"]
    n, m = k.shape[1], q.shape[1]
    i = torch.arange(m, device=q.device)[:, None] + (n - m)
    j = torch.arange(n, device=q.device)[None]
    z = q @ k.transpose(1, 2) / math.sqrt(c["dim"])
    if c["cap"] > 0:
        z = c["cap"] * torch.tanh(z / c["cap"])
    if s["slopes"] is not None:
        z = z - s["slopes"].double()[:, None, None] * (i - j).abs()
    if table is not None:
        z = z + table[s["buckets"].long()[(j - i).clamp(-REACH, REACH) + REACH]].permute(2, 0, 1)
    hide = torch.zeros_like(i - j, dtype=torch.bool)
    if c["causal"]:
        hide |= j > (torch.clamp(i, min=int(prefix[b]) - 1) if c["prefix"] else i)
    if c["window"] >= 0:
        hide |= (i - j).abs() > c["window"]
    if docs is not None:
        d = docs
        hide |= (d[n - m:, None] != d[None]) | (d[None] < 0)
    z = z.masked_fill(hide, -math.inf)
    empty = hide.all(1)
    w = torch.softmax(z.masked_fill(empty[:, None], 0.0), -1).masked_fill(empty[:, None], 0.0)
    return w @ v, torch.logsumexp(z.masked_fill(empty[:, None], 0.0), -1).masked_fill(empty, -math.inf)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    qx, kx, vx = (s[n].double().requires_grad_(c["train"]) for n in ("q", "k", "v"))
    leaves = {"dq": qx, "dk": kx}
    out = {}
    q, k = qx, kx
    with torch.set_grad_enabled(c["train"]):
        if c["op"] in ("rope", "layer"):
            gammas = []
            for name in ("q_gamma", "k_gamma"):
                gammas.append(None if s[name] is None else s[name].double().requires_grad_(c["train"]))
                leaves["d" + name] = gammas[-1]
            q, k = _exact_rope(q, gammas[0], s), _exact_rope(k, gammas[1], s)
            out["q"], out["k"] = q.detach(), k.detach()
            if c["op"] == "rope":
                if c["train"]:
                    there = {n: x for n, x in leaves.items() if x is not None}
                    grads = torch.autograd.grad([q, k], list(there.values()), [s["dq"].double(), s["dk"].double()])
                    out.update({n: None for n in leaves})
                    out.update(zip(there, grads))
                return out
        table = None
        if s["table"] is not None:
            table = s["table"].double().requires_grad_(c["train"])
        klen, qlen, prefix, docs = _layout(case)
        group = c["heads"] // c["kv_heads"]
        docs = None if docs is None else torch.from_numpy(docs).cuda()
        # each sequence differentiated by itself, down to the packed rows
        grad = {n: torch.zeros_like(x) for n, x in (("q", q), ("k", k), ("v", vx))}
        gtable = None if table is None else torch.zeros_like(table)
        os, ls, qa, ka = [], [], 0, 0
        for b, (n, m) in enumerate(zip(klen.tolist(), qlen.tolist())):
            qs, ks, vs = (x[a:a + w].detach().requires_grad_(c["train"])
                          for x, a, w in ((q, qa, m), (k, ka, n), (vx, ka, n)))
            ds = None if docs is None else docs[ka:ka + n]
            # a key head with its group at a time, for the scores' memory
            for h in range(c["kv_heads"]):
                hq = slice(h * group, (h + 1) * group)
                sh = dict(s, slopes=None if s["slopes"] is None else s["slopes"][hq])
                o, l = _exact_sequence(qs[:, hq].transpose(0, 1), ks[:, h:h + 1].transpose(0, 1),
                                       vs[:, h:h + 1].transpose(0, 1), b, sh, prefix, ds,
                                       None if table is None else table[:, hq])
                os.append(o.detach())
                ls.append(l.detach())
                if c["train"]:
                    want = [qs, ks, vs] + ([] if table is None else [table])
                    got = torch.autograd.grad(o.transpose(0, 1), want, s["do"][qa:qa + m, hq].double())
                    for name, g, at, w in zip("qkv", got, (qa, ka, ka), (m, n, n)):
                        grad[name][at:at + w] += g
                    if table is not None:
                        gtable += got[3]
            qa, ka = qa + m, ka + n
        per = c["kv_heads"]
        out["o"] = torch.cat([torch.cat(os[i:i + per]).transpose(0, 1) for i in range(0, len(os), per)])
        if not c["train"]:
            return out
        if c["op"] == "attend":
            out["lse"] = torch.cat([torch.cat(ls[i:i + per]) for i in range(0, len(ls), per)], 1)
        out["dv"], out["dtable"] = grad["v"], gtable
        if c["op"] == "layer":
            there = {n: x for n, x in leaves.items() if x is not None}
            got = torch.autograd.grad([q, k], list(there.values()), [grad["q"], grad["k"]])
            out.update({n: None for n in leaves})
            out.update(zip(there, got))
        else:
            out["dq"], out["dk"] = grad["q"], grad["k"]
    return out
