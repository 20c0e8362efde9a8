"""CPU checks of the float attention operators' boundary: what the entry
points refuse (before any GPU call), the buckets of the learned bias, and
the tests' own 64-bit reference against differences of itself."""
import ctypes as C

import numpy as np
import pytest

import attend_reference as ref
from indecis_amd import _lib

torch = pytest.importorskip("torch")
from indecis_amd import attention  # noqa: E402

P = 1 << 20  # an aligned address that no refused call reads


def heads(p=P, row=256, head=64):
    return _lib.IxhHeads(p, row, head)


def attend_args(**kw):
    a = _lib.IxhAttendArgs()
    a.type, a.B, a.nq, a.nk, a.heads, a.kv_heads, a.dim = _lib.TYPE_BF16, 1, 10, 10, 4, 4, 64
    a.q = a.k = a.v = a.o = heads()
    a.q_offs = P
    a.scale, a.window = 0.125, -1
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,say", [
    (dict(type=7), "type 7"),
    (dict(B=-1), "-1 sequences"),
    (dict(nq=(1 << 30) + 1), "2\\^30"),
    (dict(nq=1 << 30, nk=1 << 30, heads=8), "too many rows and heads"),
    (dict(dim=136), "head dimension 136"),
    (dict(dim=12), "head dimension 12"),
    (dict(dim=0), "head dimension 0"),
    (dict(heads=6), "6 heads over 4"),
    (dict(kv_heads=0), "over 0 key heads"),
    (dict(scale=0.0), "scale 0"),
    (dict(scale=float("nan")), "scale nan"),
    (dict(scale=float("inf")), "scale inf"),
    (dict(cap=-1.0), "cap -1"),
    (dict(prefix=P), "prefix needs causal"),
    (dict(q_offs=None), "q_offs is missing"),
    (dict(nk=11), "need k_offs"),
    (dict(k_docs=P), "k_docs without q_docs"),
    (dict(nk=11, k_offs=P, q_docs=P), "need k_docs"),
    (dict(table=P, n_buckets=4, reach=2), "needs buckets"),
    (dict(table=P, buckets=P, n_buckets=4, reach=0), "reach 0"),
    (dict(table=P, buckets=P, n_buckets=4, reach=1025), "reach 1025"),
    (dict(table=P, buckets=P, n_buckets=0, reach=2), "table of 0 buckets"),
    (dict(q=heads(p=None)), "q is missing"),
    (dict(k=heads(p=P + 8)), "k needs a pointer and strides"),
    (dict(v=heads(row=260)), "v needs a pointer and strides"),
    (dict(o=heads(head=12)), "o needs a pointer and strides"),
])
def test_attend_refuses(kw, say):
    a = attend_args(**kw)
    L = _lib.lib()
    with pytest.raises(_lib.IxhError, match=say) as e:
        _lib.check(L.ixh_attend(0, C.byref(a), None))
    assert e.value.code == _lib.IXH_EINVAL
    g = _lib.IxhAttendGrads(heads(), heads(), heads(), heads(), None)
    a.lse = P
    with pytest.raises(_lib.IxhError, match=say):
        _lib.check(L.ixh_attend_backward(0, C.byref(a), C.byref(g), None))


@pytest.mark.parametrize("a_kw,g_kw,say", [
    (dict(lse=None), {}, "lse is missing"),
    ({}, dict(d_out=heads(p=None)), "d_out is missing"),
    ({}, dict(dq=heads(p=P + 4)), "dq needs"),
    ({}, dict(dk=heads(row=9)), "dk needs"),
    ({}, dict(dv=heads(p=None)), "dv is missing"),
    ({}, dict(dtable=P), "dtable without a table"),
    (dict(workspace_bytes=16), {}, "bytes of workspace"),
    (dict(workspace=None), {}, "bytes of workspace"),
    (dict(workspace=P + 4), {}, "bytes of workspace"),
])
def test_attend_backward_refuses(a_kw, g_kw, say):
    a = attend_args(lse=P, workspace=P, workspace_bytes=1 << 30)
    for n, v in a_kw.items():
        setattr(a, n, v)
    g = _lib.IxhAttendGrads(heads(), heads(), heads(), heads(), None)
    for n, v in g_kw.items():
        setattr(g, n, v)
    with pytest.raises(_lib.IxhError, match=say):
        _lib.check(_lib.lib().ixh_attend_backward(0, C.byref(a), C.byref(g), None))
    with pytest.raises(_lib.IxhError, match="no gradients"):
        a = attend_args(lse=P, workspace=P, workspace_bytes=1 << 30)
        _lib.check(_lib.lib().ixh_attend_backward(0, C.byref(a), None, None))


def test_nothing_to_do():
    L = _lib.lib()
    for kw in (dict(B=0), dict(nq=0, k_offs=P)):
        _lib.check(L.ixh_attend(0, C.byref(attend_args(**kw)), None))
    n = C.c_int64(-1)
    _lib.check(L.ixh_attend_workspace(C.byref(attend_args()), 0, C.byref(n)))
    assert n.value == 0
    _lib.check(L.ixh_attend_workspace(C.byref(attend_args()), 1, C.byref(n)))
    assert n.value >= 4 * 4 * 10
    with pytest.raises(_lib.IxhError, match="no arguments"):
        _lib.check(L.ixh_attend(0, None, None))


def norm_rope_args(**kw):
    a = _lib.IxhNormRopeArgs()
    a.type, a.n, a.q_heads, a.k_heads, a.dim = _lib.TYPE_F16, 10, 4, 2, 64
    a.q = a.k = a.q_out = a.k_out = heads()
    a.norm, a.eps, a.gamma_type = 1, 1e-6, _lib.TYPE_F32
    a.cos = a.sin = P
    a.rows, a.rot = 10, 64
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,say", [
    (dict(type=3), "type 3"),
    (dict(n=-1), "-1 rows"),
    (dict(q_heads=-1), "-1 and 2 heads"),
    (dict(dim=264), "head dimension 264"),
    (dict(dim=20), "head dimension 20"),
    (dict(n=1 << 30), "too many rows for one launch"),
    (dict(norm=3), "norm 3"),
    (dict(eps=-1.0), "eps -1"),
    (dict(eps=float("nan")), "eps nan"),
    (dict(gamma_type=_lib.TYPE_BF16), "gammas of type"),
    (dict(q_gamma=P + 4), "gammas need a pointer"),
    (dict(pairs=2), "pairs 2"),
    (dict(rot=24), "24 rotated columns"),
    (dict(rot=80), "80 rotated columns"),
    (dict(pairs=1, rot=7), "7 rotated columns"),
    (dict(cos=None), "needs cos and sin"),
    (dict(rows=0), "needs cos and sin"),
    (dict(q=heads(p=P + 2)), "q needs a pointer and strides"),
    (dict(k=heads(head=4)), "k needs a pointer and strides"),
    (dict(q_out=heads(p=None)), "q_out is missing"),
])
def test_norm_rope_refuses(kw, say):
    with pytest.raises(_lib.IxhError, match=say) as e:
        _lib.check(_lib.lib().ixh_qk_norm_rope(0, C.byref(norm_rope_args(**kw)), None))
    assert e.value.code == _lib.IXH_EINVAL


@pytest.mark.parametrize("kw,say", [
    (dict(dq_out=heads(p=None)), "dq_out is missing"),
    (dict(dk=heads(row=3)), "dk needs"),
    (dict(dq_gamma=P), "bytes of workspace"),
])
def test_norm_rope_backward_refuses(kw, say):
    g = _lib.IxhNormRopeGrads(heads(), heads(), heads(), heads(), None, None)
    for n, v in kw.items():
        setattr(g, n, v)
    with pytest.raises(_lib.IxhError, match=say):
        _lib.check(_lib.lib().ixh_qk_norm_rope_backward(0, C.byref(norm_rope_args()), C.byref(g), None))
    with pytest.raises(_lib.IxhError, match="no gradients"):
        _lib.check(_lib.lib().ixh_qk_norm_rope_backward(0, C.byref(norm_rope_args()), None, None))


def test_python_refuses_before_the_library():
    q = torch.zeros(4, 2, 64)
    offs = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="q is not on a GPU"):
        attention.attend(q, q, q, offs)
    with pytest.raises(ValueError, match="q is not \\[rows\\]\\[heads\\]\\[dim\\]"):
        attention.attend(q[0], q, q, offs)
    with pytest.raises(ValueError, match="q of type"):
        attention.qk_norm_rope(q.double(), q)


@pytest.mark.parametrize("buckets,most,both", [(32, 128, True), (32, 128, False), (4, 2, True), (2, 5, False),
                                               (64, 1024, True), (7, 100, False), (1024, 1000, True)])
def test_rel_buckets(buckets, most, both):
    got = attention.rel_buckets(buckets, most, both)
    assert got.shape == (2 * most + 1,)
    half = buckets // 2 if both else buckets
    near = half // 2
    steps = half - near
    for d in range(-most, most + 1):
        a = abs(d) if both else max(-d, 0)
        if a >= near:  # borders compared as whole numbers
            a = near + sum(a ** steps >= near ** (steps - t) * most ** t for t in range(1, steps))
        assert got[d + most] == a + (half if both and d > 0 else 0), d


def test_rel_buckets_borders_where_a_float_logarithm_misses():
    # 16 = 8 * (128 / 8) ** (2 / 8): exactly on the border of bucket 10
    m = attention.rel_buckets(32, 128)
    assert m[128 - 15] == 9 and m[128 - 16] == 10 and m[128 - 32] == 12 and m[128 - 64] == 14


@pytest.mark.parametrize("args", [(3, 100, True), (2, 100, True), (33, 128, True), (1, 10, False), (1026, 1024, True),
                                  (32, 8, True), (32, 1025, True), (0, 5, False), (-2, 5, False), (32, -1, True)])
def test_rel_buckets_refuses(args):
    with pytest.raises(_lib.IxhError, match="RelBuckets"):
        attention.rel_buckets(*args)


def test_reference_gradients_are_its_differences():
    """The oracle's formulas against central differences in 64 bits."""
    rng = np.random.default_rng(3)
    offs = np.array([0, 5, 5, 12])
    x = {n: rng.standard_normal(s) for n, s in (("q", (12, 4, 8)), ("k", (12, 2, 8)), ("v", (12, 2, 8)),
                                                ("table", (6, 4)))}
    do = rng.standard_normal((12, 4, 8))
    docs = np.array([0, 0, 1, 1, -1, 0, 0, 2, 2, 2, 0, 0])
    kw = dict(u=0, cap=2.0, slopes=ref.alibi(4), buckets=np.array([0, 1, 2, 3, 4, 5, -1]), docs=docs, causal=True,
              prefix=np.array([2, 0, 3]))

    def loss():
        o = ref.attend(x["q"], x["k"], x["v"], offs, offs, table=x["table"], **kw)["o"][0]
        return (o * do).sum()

    r = ref.attend(x["q"], x["k"], x["v"], offs, offs, table=x["table"], d_out=do, **kw)
    h = 1e-5
    for name in x:
        d = rng.standard_normal(x[name].shape)
        x[name] += h * d
        up = loss()
        x[name] -= 2 * h * d
        down = loss()
        x[name] += h * d
        # a third derivative of order 1 times h^2, and 1e-16 * loss / h
        assert abs((up - down) / (2 * h) - (r["d" + name][0] * d).sum()) < 1e-8


@pytest.mark.parametrize("norm", ["none", "rms", "layer"])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
def test_reference_norm_gradients_are_its_differences(norm, pairs):
    rng = np.random.default_rng(4)
    x, dy, g = rng.standard_normal((5, 3, 24)), rng.standard_normal((5, 3, 24)), 1 + 0.1 * rng.standard_normal(24)
    ang = rng.standard_normal((5, 8))
    kw = dict(norm=norm, eps=1e-6, pairs=pairs)
    dx, dg = ref.norm_rope_backward(dy, x, g, np.cos(ang), np.sin(ang), **kw)

    def loss(x, g):
        return (ref.norm_rope(x, g, np.cos(ang), np.sin(ang), **kw)[0] * dy).sum()

    h, d, e = 1e-5, rng.standard_normal(x.shape), rng.standard_normal(24)
    assert abs((loss(x + h * d, g) - loss(x - h * d, g)) / (2 * h) - (dx * d).sum()) < 1e-7
    assert abs((loss(x, g + h * e) - loss(x, g - h * e)) / (2 * h) - (dg * e).sum()) < 1e-7
