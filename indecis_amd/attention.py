"""Float attention on device rows (include/indecis_hip.h): the norms of
queries and keys for each head with the position rotation, attention with
shaped scores, the learned bias by distance, each with its gradients.

For encoders and prefix models whose layers are not the reference's (its int8
attention is linalg.attend8). Tensors are torch's, on one GPU; a call queues
its work on torch's current stream of that GPU and returns. Nothing is
recorded for torch's own differentiation: the backward is a call.

Rows are packed: q [rows][heads][dim] holds its sequences one after another,
sequence b in rows offs[b] to offs[b+1] (int32 on the GPU), as ids and offs of
Model.encode_seqs. The rows may be slices of wider ones (the Q, K and V
columns of one projection): strides and pointers are multiples of 16 bytes,
the values of a head stand side by side.
"""
import ctypes as C

import numpy as np
import torch

from . import _lib

_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}


def _need(ok, op, what):
    if not ok:
        raise ValueError(f"linalg: {op}: {what}")


def _rows(op, name, t, like=None):
    """Checks rows of heads; `like`: a tensor with the same type and GPU."""
    _need(t.dim() == 3, op, f"{name} is not [rows][heads][dim]")
    _need(t.dtype in _TYPES, op, f"{name} of type {t.dtype}")
    _need(t.is_cuda, op, f"{name} is not on a GPU")
    _need(t.shape[2] == 0 or t.stride(2) == 1, op, f"{name}: the values of a head do not stand side by side")
    if like is not None:
        _need(t.dtype == like.dtype and t.device == like.device, op, f"{name} has another type or GPU")


def _heads(t):
    # the stride along one row or one head says nothing
    n, h, d = t.shape
    head = t.stride(1) if h > 1 else d
    return _lib.IxhHeads(t.data_ptr(), t.stride(0) if n > 1 else h * d, head)


def _plain(op, name, t, like, dtype, shape):
    """The address of a contiguous array on like's GPU, or None."""
    if t is None:
        return None
    _need(t.dtype == dtype and tuple(t.shape) == shape, op, f"{name} is not {dtype} of shape {shape}")
    _need(t.device == like.device and t.is_contiguous(), op, f"{name} is not contiguous on the rows' GPU")
    return t.data_ptr()


def _out(op, name, t, like, shape):
    if t is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    _rows(op, name, t, like)
    _need(tuple(t.shape) == shape, op, f"{name} is not of shape {shape}")
    return t


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _space(t, n):
    return torch.empty(n, dtype=torch.uint8, device=t.device) if n else None


def _attend_args(op, q, k, v, offs, k_offs, scale, cap, slopes, table, buckets, docs, k_docs, causal, prefix, window):
    _rows(op, "q", q)
    _rows(op, "k", k, q)
    _rows(op, "v", v, q)
    nq, heads, dim = q.shape
    nk, kv_heads, _ = k.shape
    _need(k.shape == v.shape and k.shape[2] == dim, op, "q, k and v do not fit together")
    _need(offs.dim() == 1 and len(offs) >= 1, op, "offs is not [sequences + 1]")
    B = len(offs) - 1
    a = _lib.IxhAttendArgs()
    a.type, a.B, a.nq, a.nk, a.heads, a.kv_heads, a.dim = _TYPES[q.dtype], B, nq, nk, heads, kv_heads, dim
    a.q, a.k, a.v = _heads(q), _heads(k), _heads(v)
    a.q_offs = _plain(op, "offs", offs, q, torch.int32, (B + 1,))
    a.k_offs = _plain(op, "k_offs", k_offs, q, torch.int32, (B + 1,))
    a.scale = dim ** -0.5 if scale is None else scale
    a.cap = cap
    a.slopes = _plain(op, "slopes", slopes, q, torch.float32, (heads,))
    if table is not None:
        _need(table.dim() == 2 and buckets is not None and buckets.dim() == 1 and len(buckets) % 2 == 1, op,
              "a table [buckets][heads] needs the buckets of an odd number of distances")
        a.n_buckets, a.reach = len(table), len(buckets) // 2
        a.table = _plain(op, "table", table, q, q.dtype, (len(table), heads))
        a.buckets = _plain(op, "buckets", buckets, q, torch.int32, (len(buckets),))
    a.q_docs = _plain(op, "docs", docs, q, torch.int32, (nq,))
    a.k_docs = _plain(op, "k_docs", k_docs, q, torch.int32, (nk,))
    a.causal = 1 if causal else 0
    a.prefix = _plain(op, "prefix", prefix, q, torch.int32, (B,))
    a.window = -1 if window is None else window
    return a


def _with_space(a, q, backward):
    n = C.c_int64()
    _lib.check(_lib.lib().ixh_attend_workspace(C.byref(a), backward, C.byref(n)))
    space = _space(q, n.value)
    if space is not None:
        a.workspace, a.workspace_bytes = space.data_ptr(), n.value
    return space


def attend(q, k, v, offs, k_offs=None, *, scale=None, cap=0.0, slopes=None, table=None, buckets=None, docs=None,
           k_docs=None, causal=False, prefix=None, window=-1, out=None, want_lse=False):
    """softmax(scores) v over each query's visible keys: [rows][heads][dim],
    with want_lse also the logarithms of the sums, [heads][rows] float32,
    which attend_backward takes.

    Head h reads key head h // (heads // kv_heads). A sequence's last query
    stands at its last key, so one query with k_offs of a longer sequence is
    its newest token. Scores: scale * q.k (scale: dim ** -0.5 by default);
    cap > 0: cap * tanh(score / cap); slopes [heads]: less slope * distance;
    table [buckets][heads] (of q's type) with buckets from rel_buckets: plus
    the entry of the distance's bucket. Visible: the query's own document
    (docs, k_docs: int32 a row, below 0 for padding); causal: no later key,
    but the first prefix[b] for every query; window >= 0: keys at most that
    far off. A query that sees nothing gets 0 (and -inf). Rows outside the
    sequences are left as they are."""
    op = "Attend"
    a = _attend_args(op, q, k, v, offs, k_offs, scale, cap, slopes, table, buckets, docs, k_docs, causal, prefix, window)
    out = _out(op, "out", out, q, tuple(q.shape))
    lse = torch.empty((a.heads, a.nq), dtype=torch.float32, device=q.device) if want_lse else None
    a.o = _heads(out)
    a.lse = lse.data_ptr() if want_lse else None
    space = _with_space(a, q, 0)  # held until the call has queued its work
    _lib.check(_lib.lib().ixh_attend(q.device.index, C.byref(a), _stream(q)))
    return (out, lse) if want_lse else out


def attend_backward(d_out, q, k, v, out, lse, offs, k_offs=None, *, scale=None, cap=0.0, slopes=None, table=None,
                    buckets=None, docs=None, k_docs=None, causal=False, prefix=None, window=-1, dq=None, dk=None,
                    dv=None):
    """The gradients (dq, dk, dv, dtable) of attend at the same arguments,
    from its output and lse; dtable [buckets][heads] of the table's type, None
    without a table."""
    op = "AttendBackward"
    a = _attend_args(op, q, k, v, offs, k_offs, scale, cap, slopes, table, buckets, docs, k_docs, causal, prefix, window)
    for name, t in (("d_out", d_out), ("out", out)):
        _rows(op, name, t, q)
        _need(t.shape == q.shape, op, f"{name} is not of q's shape")
    dq = _out(op, "dq", dq, q, tuple(q.shape))
    dk = _out(op, "dk", dk, q, tuple(k.shape))
    dv = _out(op, "dv", dv, q, tuple(v.shape))
    dtable = torch.empty_like(table) if table is not None else None
    _need(lse is not None, op, "lse is missing")
    a.o, a.lse = _heads(out), _plain(op, "lse", lse, q, torch.float32, (a.heads, a.nq))
    g = _lib.IxhAttendGrads(_heads(d_out), _heads(dq), _heads(dk), _heads(dv),
                            None if dtable is None else dtable.data_ptr())
    space = _with_space(a, q, 1)
    _lib.check(_lib.lib().ixh_attend_backward(q.device.index, C.byref(a), C.byref(g), _stream(q)))
    return dq, dk, dv, dtable


def rel_buckets(buckets, max_distance, bidirectional=True):
    """The bucket of each distance -max_distance..max_distance (key less
    query) of a learned bias, int32: one a distance up to half of a
    direction's buckets, then on a logarithmic scale. Host only."""
    out = np.zeros(2 * max(int(max_distance), 0) + 1, np.int32)
    _lib.check(_lib.lib().ixh_rel_buckets(int(buckets), int(max_distance), 1 if bidirectional else 0,
                                          out.ctypes.data_as(C.c_void_p)))
    return out


def _norm_rope_args(op, q, k, cos, sin, pos, q_gamma, k_gamma, norm, eps, pairs):
    _rows(op, "q", q)
    _rows(op, "k", k, q)
    n, dim = q.shape[0], q.shape[2]
    _need(k.shape[0] == n and k.shape[2] == dim, op, "q and k do not fit together")
    _need(norm in _lib.HEAD_NORMS and pairs in _lib.PAIRS, op, f"norm {norm!r}, pairs {pairs!r}")
    a = _lib.IxhNormRopeArgs()
    a.type, a.n, a.q_heads, a.k_heads, a.dim = _TYPES[q.dtype], n, q.shape[1], k.shape[1], dim
    a.q, a.k = _heads(q), _heads(k)
    a.norm, a.eps, a.pairs = _lib.HEAD_NORMS[norm], eps, _lib.PAIRS[pairs]
    gamma = q_gamma if q_gamma is not None else k_gamma
    dtype = torch.float32 if gamma is None else gamma.dtype
    _need(dtype in _TYPES, op, f"gammas of type {dtype}")
    a.gamma_type = _TYPES[dtype]
    a.q_gamma = _plain(op, "q_gamma", q_gamma, q, dtype, (dim,))
    a.k_gamma = _plain(op, "k_gamma", k_gamma, q, dtype, (dim,))
    if cos is not None:
        _need(cos.dim() == 2 and sin is not None, op, "cos and sin are not [rows][columns / 2]")
        a.rows, a.rot = cos.shape[0], 2 * cos.shape[1]
        a.cos = _plain(op, "cos", cos, q, torch.float32, tuple(cos.shape))
        a.sin = _plain(op, "sin", sin, q, torch.float32, tuple(cos.shape))
    a.pos = _plain(op, "pos", pos, q, torch.int32, (n,))
    return a


def qk_norm_rope(q, k, cos=None, sin=None, *, pos=None, q_gamma=None, k_gamma=None, norm="rms", eps=1e-6,
                 pairs="halves", q_out=None, k_out=None):
    """The norm of each head of q [rows][heads][dim] and k [rows][kv_heads]
    [dim] and the rotation of its first columns, in one pass: (q_out, k_out),
    which may be q and k themselves. norm: "rms", "layer" (its mean taken off
    first) or "none"; gammas [dim] (float32 or the rows' type). cos and sin
    [rows][columns / 2] float32, read at pos (int32 a row; by default the row
    itself; a place past the tables gives NaN); pairs: "halves" (column i with
    i + columns / 2) or "neighbours" (2i with 2i + 1)."""
    op = "QKNormRope"
    a = _norm_rope_args(op, q, k, cos, sin, pos, q_gamma, k_gamma, norm, eps, pairs)
    q_out = _out(op, "q_out", q_out, q, tuple(q.shape))
    k_out = _out(op, "k_out", k_out, q, tuple(k.shape))
    a.q_out, a.k_out = _heads(q_out), _heads(k_out)
    _lib.check(_lib.lib().ixh_qk_norm_rope(q.device.index, C.byref(a), _stream(q)))
    return q_out, k_out


def qk_norm_rope_backward(dq_out, dk_out, q, k, cos=None, sin=None, *, pos=None, q_gamma=None, k_gamma=None,
                          norm="rms", eps=1e-6, pairs="halves", dq=None, dk=None):
    """The gradients (dq, dk, dq_gamma, dk_gamma) of qk_norm_rope at the same
    arguments (q and k as they went in); a gamma's is None without it. dq and
    dk may be dq_out and dk_out themselves."""
    op = "QKNormRopeBackward"
    a = _norm_rope_args(op, q, k, cos, sin, pos, q_gamma, k_gamma, norm, eps, pairs)
    for name, t, like in (("dq_out", dq_out, q), ("dk_out", dk_out, k)):
        _rows(op, name, t, q)
        _need(t.shape == like.shape, op, f"{name} has another shape than its rows")
    dq = _out(op, "dq", dq, q, tuple(q.shape))
    dk = _out(op, "dk", dk, q, tuple(k.shape))
    dq_gamma = None if q_gamma is None else torch.empty_like(q_gamma)
    dk_gamma = None if k_gamma is None else torch.empty_like(k_gamma)
    g = _lib.IxhNormRopeGrads(_heads(dq_out), _heads(dk_out), _heads(dq), _heads(dk),
                              None if dq_gamma is None else dq_gamma.data_ptr(),
                              None if dk_gamma is None else dk_gamma.data_ptr())
    space = None
    if dq_gamma is not None or dk_gamma is not None:
        n = C.c_int64()
        _lib.check(_lib.lib().ixh_qk_norm_rope_workspace(C.byref(a), C.byref(n)))
        space = _space(q, n.value)
        a.workspace, a.workspace_bytes = space.data_ptr(), n.value
    _lib.check(_lib.lib().ixh_qk_norm_rope_backward(q.device.index, C.byref(a), C.byref(g), _stream(q)))
    return dq, dk, dq_gamma, dk_gamma
