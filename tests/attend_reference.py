"""The float attention operators in 64 bits, sequence by sequence (numpy),
with bounds on how far a kernel's rounded results may be from them.

Bounds. u is half a step of the rows' type (0 for float32 where only 32-bit
sums round), w = 2^-24 half a step of float32.
 - a score: a sum of dim products in 32 bits, scaled, biased: (dim + 8) w of
   the sum of its terms' absolute values; the 16-bit kernels' tanh is within
   2^-20 of tanh (its exponent's argument and the exponential round to 2 w
   each, times |x| u (1 - u) < 0.28, four times; the reciprocal 2 w, doubled),
   float32's within 4 w.
 - a probability: exp's argument is a difference of two scores, so its
   relative error is at most twice the largest error of a score in the row,
   plus (keys + 16) w for the exponential, the sum and the division.
 - o: probabilities rounded to the type (u each), the 32-bit sum, one last
   rounding.
 - dZ = P (dP - delta): delta is taken of the rounded o, so it is off by
   |dO| times o's bound; dP is a sum of dim products.
 - dQ, dK, dV: dZ (P) rounded to the type, the 32-bit sum, one last rounding.
 - below 2^-14 float16's values are 2^-24 apart, so that each rounding to it
   may be off by half of that, 2^-25, whatever the value (a key whose only
   query sees nothing else has dZ = 0 but for delta's own rounding, and a dK
   of some 1e-8): 2^-25 for a result, and for each P and dZ that it sums,
   times the other factor. bfloat16 and float32 have normal values down to
   2^-126: their share is inside the 1e-30.
Every second-order term is covered by a factor of 1.05."""
import math

import numpy as np

W = 2.0 ** -24


def bias_and_mask(nq, nk, *, heads, slopes, table, buckets, docs_q, docs_k, causal, prefix, window):
    """([heads][nq][nk] bias, [nq][nk] visible, [nq][nk] bucket or None)."""
    p = np.arange(nq)[:, None] + nk - nq
    j = np.arange(nk)[None]
    see = np.ones((nq, nk), bool)
    if causal:
        see &= (j <= p) | (j < (0 if prefix is None else prefix))
    if window >= 0:
        see &= np.abs(j - p) <= window
    if docs_q is not None:
        see &= (docs_q[:, None] == docs_k[None]) & (docs_k[None] >= 0)
    bias = np.zeros((heads, nq, nk))
    if slopes is not None:
        bias -= slopes[:, None, None] * np.abs(j - p)
    at = None
    if table is not None:
        reach = len(buckets) // 2
        at = buckets[np.clip(j - p, -reach, reach) + reach]
        inside = (at >= 0) & (at < len(table))
        bias += np.where(inside[..., None], table[np.where(inside, at, 0)], 0).transpose(2, 0, 1)
        at = np.where(inside, at, -1)
    return bias, see, at


def attend(q, k, v, q_offs, k_offs, *, u, scale=None, cap=0.0, slopes=None, table=None, buckets=None, docs=None,
           k_docs=None, causal=False, prefix=None, window=-1, d_out=None):
    """A dict of name -> (value, bound) of o and lse, and with d_out of dq, dk,
    dv and dtable. Rows outside the sequences are NaN."""
    nq, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    tiny = 2.0 ** -25 if u == 2.0 ** -11 else 1e-30  # a rounding below the type's normal values
    tanh_err = 4 * W if u == 0 else 2.0 ** -20
    out = {n: [np.full(s, np.nan), np.zeros(s)] for n, s in
           (("o", q.shape), ("lse", (heads, nq)), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape))}
    dtable = [np.zeros(table.shape), np.zeros(table.shape)] if table is not None else None
    for b in range(len(q_offs) - 1):
        q0, q1, k0, k1 = q_offs[b], q_offs[b + 1], k_offs[b], k_offs[b + 1]
        n, m = q1 - q0, k1 - k0
        kd = None if docs is None else (docs if k_docs is None else k_docs)[k0:k1]
        bias, see, at = bias_and_mask(n, m, heads=heads, slopes=slopes, table=table, buckets=buckets,
                                      docs_q=None if docs is None else docs[q0:q1], docs_k=kd, causal=causal,
                                      prefix=None if prefix is None else prefix[b], window=window)
        for h in range(heads):
            g = h // group
            qh, kh, vh = q[q0:q1, h], k[k0:k1, g], v[k0:k1, g]
            if kd is not None:  # padding holds anything
                kh, vh = np.where(kd[:, None] < 0, 0, kh), np.where(kd[:, None] < 0, 0, vh)
            seen = see.any(1)
            qh = np.where(seen[:, None], qh, 0)
            s = scale * (qh @ kh.T)
            es = (dim + 8) * W * scale * (np.abs(qh) @ np.abs(kh).T)
            slope = 1.0
            if cap > 0:
                th = np.tanh(s / cap)
                slope = 1 - th * th
                z, ez = cap * th, es + cap * (tanh_err + 4 * W)
            else:
                z, ez = s, es
            z = z + bias[h]
            ez = ez + 4 * W * (np.abs(z) + np.abs(bias[h]))
            z = np.where(see, z, -np.inf)
            top = np.where(seen, z.max(1, initial=-np.inf), 0)[:, None]
            e = np.exp(z - top)
            total = e.sum(1, keepdims=True)
            p = e / np.where(total == 0, 1, total)
            worst = np.where(see, ez, 0).max(1, initial=0)[:, None]
            ep = 2 * worst + (m + 16) * W  # relative, of p
            o, ov = p @ vh, p @ np.abs(vh)
            eo = 1.05 * (u * np.abs(o) + (u + ep + W * m) * ov + W * np.abs(o) + tiny * (see @ np.abs(vh))) + tiny
            out["o"][0][q0:q1, h], out["o"][1][q0:q1, h] = o, eo
            with np.errstate(divide="ignore"):
                lse = np.where(seen, top[:, 0] + np.log(total[:, 0]), -np.inf)
            out["lse"][0][h, q0:q1] = lse
            out["lse"][1][h, q0:q1] = np.where(seen, 1.05 * (worst[:, 0] + (m + 8) * W * (1 + np.abs(np.where(seen, lse, 0)))), 0)
            if d_out is None:
                continue
            do = np.where(seen[:, None], d_out[q0:q1, h], 0)
            dp = do @ vh.T
            edp = (dim + 4) * W * (np.abs(do) @ np.abs(vh).T)
            delta = (do * o).sum(1, keepdims=True)
            edelta = (np.abs(do) * eo).sum(1, keepdims=True) + (dim + 4) * W * (np.abs(do) * np.abs(o)).sum(1, keepdims=True)
            # P comes from lse here: one more rounding of it
            ep = ep + np.where(seen, 4 * W * (1 + np.abs(np.where(seen, lse, 0))), 0)[:, None] + worst
            dz = p * (dp - delta)
            edz = 1.05 * (p * (edp + edelta) + (ep + 4 * W) * np.abs(dz))
            if table is not None:
                for idx in np.unique(at[at >= 0]):
                    hit = at == idx
                    dtable[0][idx, h] += dz[hit].sum()
                    dtable[1][idx, h] += edz[hit].sum() + (hit.sum() + 64) * W * np.abs(dz[hit]).sum()
            ds = dz * slope
            # 1 - tanh^2 from the reciprocal, absolutely as near as tanh
            eds = edz * np.abs(slope) + (0 if cap == 0 else 4 * (tanh_err + 4 * W) + 2 * es / cap) * np.abs(dz)
            size = (u + (m + n + 8) * W) * np.abs(ds) + eds + tiny * see
            for name, val, err, sl, hh in (
                    ("dq", scale * (ds @ kh), scale * (size @ np.abs(kh)), slice(q0, q1), h),
                    ("dk", scale * (ds.T @ qh), scale * (size.T @ np.abs(qh)), slice(k0, k1), g),
                    ("dv", p.T @ do, ((u + ep + (n + 8) * W) * p + tiny * see).T @ np.abs(do), slice(k0, k1), g)):
                if name == "dq" or h % group == 0:
                    out[name][0][sl, hh] = 0
                out[name][0][sl, hh] += val
                out[name][1][sl, hh] += 1.05 * err
    res = {"o": out["o"], "lse": out["lse"]}
    if d_out is not None:
        for name in ("dq", "dk", "dv"):
            out[name][1] += (u + W) * np.nan_to_num(np.abs(out[name][0])) + tiny
            res[name] = out[name]
        if dtable is not None:
            dtable[1] = 1.05 * dtable[1] + (u + W) * np.abs(dtable[0]) + tiny
            res["dtable"] = dtable
    return res


def turn(y, cos, sin, pairs):
    """The first columns of y [n][heads][dim] rotated by cos, sin [n][rot / 2]."""
    half = cos.shape[1]
    y = y.copy()
    if half == 0:
        return y
    i = np.arange(half)
    ia, ib = (i, i + half) if pairs == "halves" else (2 * i, 2 * i + 1)
    a, b, c, s = y[..., ia], y[..., ib], cos[:, None], sin[:, None]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def norm_rope(x, gamma, cos, sin, *, norm, eps, pairs):
    """(y, normalised rows, their scale) of x [n][heads][dim]."""
    xc = x - x.mean(-1, keepdims=True) if norm == "layer" else x
    r = 1.0 if norm == "none" else 1 / np.sqrt((xc * xc).mean(-1, keepdims=True) + eps)
    xh = xc * r
    return turn(xh * gamma, cos, sin, pairs), xh, r


def norm_rope_backward(dy, x, gamma, cos, sin, *, norm, eps, pairs):
    """(dx, dgamma)."""
    _, xh, r = norm_rope(x, gamma, cos, sin, norm=norm, eps=eps, pairs=pairs)
    d = turn(dy, cos, -sin, pairs)
    dgamma = (d * xh).sum((0, 1))
    d = d * gamma
    if norm == "none":
        return d, dgamma
    dx = d - xh * (d * xh).mean(-1, keepdims=True)
    if norm == "layer":
        dx = dx - d.mean(-1, keepdims=True)
    return dx * r, dgamma


def alibi(heads):
    return np.array([math.pow(2.0, -8.0 * (h + 1) / heads) for h in range(heads)])
