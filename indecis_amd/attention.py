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
import struct

import numpy as np
import torch

from . import _lib

_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}

# The library's argument structs, packed in one go: a call of the smallest
# size is as long as its host side.
_ATTEND = struct.Struct("@7i" + 4 * "Pqq" + "2P2f3P2i2PiPi2Pq")
_GRADS = struct.Struct("@" + 4 * "Pqq" + "P")
_NORM_ROPE = struct.Struct("@5i" + 4 * "Pqq" + "idi4P3iP" + "Pq")
_NORM_ROPE_GRADS = struct.Struct("@" + 4 * "Pqq" + "2P")
for _s, _c in ((_ATTEND, _lib.IxhAttendArgs), (_GRADS, _lib.IxhAttendGrads), (_NORM_ROPE, _lib.IxhNormRopeArgs),
               (_NORM_ROPE_GRADS, _lib.IxhNormRopeGrads)):
    assert _s.size == C.sizeof(_c)


def _need(ok, op, what):
    if not ok:
        raise ValueError(f"linalg: {op}: {what}")


def _heads(op, name, t, like=None, shape=None):
    """(address, row stride, head stride) of rows of heads; `like`: a tensor
    with the same type and GPU."""
    size, strides = t.shape, t.stride()
    if (len(size) != 3 or not t.is_cuda or (strides[2] != 1 and size[2] > 0) or (like is None and t.dtype not in _TYPES)
            or (like is not None and (t.dtype is not like.dtype or t.get_device() != like.get_device()))
            or (shape is not None and size != shape)):
        _need(len(size) == 3, op, f"{name} is not [rows][heads][dim]")
        _need(t.dtype in _TYPES, op, f"{name} of type {t.dtype}")
        _need(t.is_cuda, op, f"{name} is not on a GPU")
        _need(strides[2] == 1 or size[2] == 0, op, f"{name}: the values of a head do not stand side by side")
        _need(like is None or (t.dtype is like.dtype and t.get_device() == like.get_device()), op,
              f"{name} has another type or GPU")
        _need(False, op, f"{name} is not of shape {tuple(shape)}")
    n, h, d = size
    # the stride along one row or one head says nothing
    return t.data_ptr(), strides[0] if n > 1 else h * d, strides[1] if h > 1 else d


def _plain(op, name, t, like, dtype, shape):
    """The address of a contiguous array on like's GPU; 0 for None."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.shape != shape or t.get_device() != like.get_device() or not t.is_contiguous():
        _need(t.dtype is dtype and t.shape == shape, op, f"{name} is not {dtype} of shape {tuple(shape)}")
        _need(False, op, f"{name} is not contiguous on the rows' GPU")
    return t.data_ptr()


def _out(op, name, t, like):
    """An output of like's shape, and its place."""
    if t is None:
        t = like.new_empty(like.shape)
        return t, (t.data_ptr(), t.stride(0), t.stride(1))
    return t, _heads(op, name, t, like, like.shape)


_WORKSPACE = struct.Struct("@Pq")  # the argument structs' last two


def _call(f, like, *args):
    device = like.get_device()
    _lib.check(f(device, *args, _stream(device)))


def _stream(device):
    """The address of torch's current stream of the GPU."""
    return torch.cuda.current_stream(device).cuda_stream


# the same without the object around it, where this torch has it
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _stream)


def _with_space(packed, like, size, *more):
    """The packed arguments with the workspace that `size` asks for, and the
    workspace: held until the call has queued its work."""
    n = C.c_int64()
    _lib.check(size(packed, *more, C.byref(n)))
    if n.value == 0:
        return packed, None
    space = like.new_empty(n.value, dtype=torch.uint8)
    return packed[:-_WORKSPACE.size] + _WORKSPACE.pack(space.data_ptr(), n.value), space


def _attend_args(op, q, k, v, offs, k_offs, scale, cap, slopes, table, buckets, docs, k_docs, causal, prefix, window):
    """The values of ixh_attend_args before and after o, up to lse."""
    qh, kh, vh = _heads(op, "q", q), _heads(op, "k", k, q), _heads(op, "v", v, q)
    nq, heads, dim = q.shape
    nk, kv_heads, k_dim = k.shape
    _need(k.shape == v.shape and k_dim == dim and dim > 0, op, "q, k and v do not fit together")
    B = offs.numel() - 1
    _need(B >= 0, op, "offs is not [sequences + 1]")
    n_buckets = reach = 0
    if table is not None:
        _need(table.dim() == 2 and buckets is not None and buckets.dim() == 1 and len(buckets) % 2 == 1, op,
              "a table [buckets][heads] needs the buckets of an odd number of distances")
        n_buckets, reach = len(table), len(buckets) // 2
    i32 = torch.int32
    return (_TYPES[q.dtype], B, nq, nk, heads, kv_heads, dim, *qh, *kh, *vh), (
        _plain(op, "offs", offs, q, i32, (B + 1,)),
        _plain(op, "k_offs", k_offs, q, i32, (B + 1,)),
        dim ** -0.5 if scale is None else scale, cap,
        _plain(op, "slopes", slopes, q, torch.float32, (heads,)),
        _plain(op, "table", table, q, q.dtype, (n_buckets, heads)),
        _plain(op, "buckets", buckets, q, i32, (2 * reach + 1,)) if table is not None else 0,
        n_buckets, reach,
        _plain(op, "docs", docs, q, i32, (nq,)),
        _plain(op, "k_docs", k_docs, q, i32, (nk,)),
        1 if causal else 0,
        _plain(op, "prefix", prefix, q, i32, (B,)),
        -1 if window is None else window)


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
    before, after = _attend_args(op, q, k, v, offs, k_offs, scale, cap, slopes, table, buckets, docs, k_docs, causal,
                                 prefix, window)
    out, place = _out(op, "out", out, q)
    lse = q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32) if want_lse else None
    L = _lib.lib()
    args, space = _with_space(_ATTEND.pack(*before, *place, *after, lse.data_ptr() if want_lse else 0, 0, 0), q,
                              L.ixh_attend_workspace, 0)
    _call(L.ixh_attend, q, args)
    return (out, lse) if want_lse else out


def attend_backward(d_out, q, k, v, out, lse, offs, k_offs=None, *, scale=None, cap=0.0, slopes=None, table=None,
                    buckets=None, docs=None, k_docs=None, causal=False, prefix=None, window=-1, dq=None, dk=None,
                    dv=None):
    """The gradients (dq, dk, dv, dtable) of attend at the same arguments,
    from its output and lse; dtable [buckets][heads] of the table's type, None
    without a table."""
    op = "AttendBackward"
    before, after = _attend_args(op, q, k, v, offs, k_offs, scale, cap, slopes, table, buckets, docs, k_docs, causal,
                                 prefix, window)
    _need(lse is not None, op, "lse is missing")
    lse_at = _plain(op, "lse", lse, q, torch.float32, (q.shape[1], q.shape[0]))
    given = _heads(op, "d_out", d_out, q, q.shape)
    place = _heads(op, "out", out, q, q.shape)
    (dq, dq_at), (dk, dk_at), (dv, dv_at) = _out(op, "dq", dq, q), _out(op, "dk", dk, k), _out(op, "dv", dv, v)
    dtable = torch.empty_like(table) if table is not None else None
    L = _lib.lib()
    args, space = _with_space(_ATTEND.pack(*before, *place, *after, lse_at, 0, 0), q, L.ixh_attend_workspace, 1)
    _call(L.ixh_attend_backward, q, args,
          _GRADS.pack(*given, *dq_at, *dk_at, *dv_at, dtable.data_ptr() if dtable is not None else 0))
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
    """The values of ixh_norm_rope_args before and after q_out and k_out, up
    to the workspace."""
    qh, kh = _heads(op, "q", q), _heads(op, "k", k, q)
    n, q_heads, dim = q.shape
    n_k, k_heads, k_dim = k.shape
    _need(n_k == n and k_dim == dim, op, "q and k do not fit together")
    if norm not in _lib.HEAD_NORMS or pairs not in _lib.PAIRS:
        _need(False, op, f"norm {norm!r}, pairs {pairs!r}")
    gamma = q_gamma if q_gamma is not None else k_gamma
    dtype = torch.float32 if gamma is None else gamma.dtype
    _need(dtype in _TYPES, op, "gammas of another type than float32 and the rows'")
    rows = half = 0
    if cos is not None:
        _need(cos.dim() == 2 and sin is not None, op, "cos and sin are not [rows][columns / 2]")
        rows, half = cos.shape
    return (_TYPES[q.dtype], n, q_heads, k_heads, dim, *qh, *kh), (
        _lib.HEAD_NORMS[norm], eps, _TYPES[dtype],
        _plain(op, "q_gamma", q_gamma, q, dtype, (dim,)), _plain(op, "k_gamma", k_gamma, q, dtype, (dim,)),
        _plain(op, "cos", cos, q, torch.float32, (rows, half)),
        _plain(op, "sin", sin, q, torch.float32, (rows, half)) if cos is not None else 0,
        rows, 2 * half, _lib.PAIRS[pairs], _plain(op, "pos", pos, q, torch.int32, (n,)))


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
    before, after = _norm_rope_args(op, q, k, cos, sin, pos, q_gamma, k_gamma, norm, eps, pairs)
    (q_out, q_at), (k_out, k_at) = _out(op, "q_out", q_out, q), _out(op, "k_out", k_out, k)
    _call(_lib.lib().ixh_qk_norm_rope, q, _NORM_ROPE.pack(*before, *q_at, *k_at, *after, 0, 0))
    return q_out, k_out


def qk_norm_rope_backward(dq_out, dk_out, q, k, cos=None, sin=None, *, pos=None, q_gamma=None, k_gamma=None,
                          norm="rms", eps=1e-6, pairs="halves", dq=None, dk=None):
    """The gradients (dq, dk, dq_gamma, dk_gamma) of qk_norm_rope at the same
    arguments (q and k as they went in); a gamma's is None without it. dq and
    dk may be dq_out and dk_out themselves."""
    op = "QKNormRopeBackward"
    before, after = _norm_rope_args(op, q, k, cos, sin, pos, q_gamma, k_gamma, norm, eps, pairs)
    given = (*_heads(op, "dq_out", dq_out, q, q.shape), *_heads(op, "dk_out", dk_out, q, k.shape))
    (dq, dq_at), (dk, dk_at) = _out(op, "dq", dq, q), _out(op, "dk", dk, k)
    dq_gamma = None if q_gamma is None else torch.empty_like(q_gamma)
    dk_gamma = None if k_gamma is None else torch.empty_like(k_gamma)
    none = (0, 0, 0)
    L = _lib.lib()
    args, space = _NORM_ROPE.pack(*before, *none, *none, *after, 0, 0), None
    if dq_gamma is not None or dk_gamma is not None:
        args, space = _with_space(args, q, L.ixh_qk_norm_rope_workspace)
    _call(L.ixh_qk_norm_rope_backward, q, args,
          _NORM_ROPE_GRADS.pack(*given, *dq_at, *dk_at, dq_gamma.data_ptr() if dq_gamma is not None else 0,
                                dk_gamma.data_ptr() if dk_gamma is not None else 0))
    return dq, dk, dq_gamma, dk_gamma
