"""The float attention operators on the GPU against their definitions in 64
bits (tests/attend_reference.py, whose bounds each result has to keep value
by value), at the lengths, masks and layouts where they can go wrong, and run
together as a layer's training step runs them."""
import numpy as np
import pytest

import attend_reference as ref
from indecis_amd import _lib

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from indecis_amd import attention  # noqa: E402

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(t):
    return 0 if t == torch.float32 else torch.finfo(t).eps / 2


def f64(t):
    return t.detach().double().cpu().numpy()


def ints(a):
    return torch.from_numpy(np.asarray(a, np.int32)).cuda()


def rows(rng, t, *shape):
    """Normal rows of the type, as the type holds them."""
    return torch.from_numpy(rng.standard_normal(shape)).to(t).cuda()


def within(name, got, want, err):
    got = f64(got)
    here = ~np.isnan(want)
    fin = here & np.isfinite(want)
    assert np.array_equal(got[here & ~fin], want[here & ~fin]), name
    off = np.abs(got[fin] - want[fin]) - err[fin]
    assert not np.isnan(off).any(), f"{name}: NaN"
    if off.size and off.max() > 0:
        worst = np.unravel_index(np.where(fin, np.abs(np.nan_to_num(got - want)) - err, -1).argmax(), got.shape)
        raise AssertionError(f"{name}: {np.mean(off > 0):.2%} past the bound, worst at {worst}: "
                             f"{got[worst]} for {want[worst]} +- {err[worst]}")


def check(rng, t, q_lens, k_lens=None, *, heads=4, kv_heads=2, dim=64, table=None, buckets=None, docs=None, k_docs=None,
          slopes=None, prefix=None, backward=True, tensors=None, **kw):
    t = TYPES[t]
    q_offs = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    k_offs = q_offs if k_lens is None else np.concatenate([[0], np.cumsum(k_lens)]).astype(np.int32)
    nq, nk = q_offs[-1], k_offs[-1]
    if tensors is None:
        q, k, v, do = (rows(rng, t, n, h, dim) for n, h in ((nq, heads), (nk, kv_heads), (nk, kv_heads), (nq, heads)))
    else:
        q, k, v, do = tensors
    tab = None if table is None else torch.from_numpy(table).to(t).cuda()
    call = dict(kw, slopes=None if slopes is None else torch.from_numpy(slopes).float().cuda(), table=tab,
                buckets=None if buckets is None else ints(buckets), docs=None if docs is None else ints(docs),
                k_docs=None if k_docs is None else ints(k_docs), prefix=None if prefix is None else ints(prefix))
    where = (ints(q_offs), None if k_lens is None else ints(k_offs))
    o, lse = attention.attend(q, k, v, *where, want_lse=True, **call)
    got = {"o": o, "lse": lse}
    if backward:
        got["dq"], got["dk"], got["dv"], got["dtable"] = attention.attend_backward(do, q, k, v, o, lse, *where, **call)
    want = ref.attend(f64(q), f64(k), f64(v), q_offs, k_offs, u=half_step(t),
                      slopes=None if slopes is None else slopes.astype(np.float32).astype(np.float64),
                      table=None if tab is None else f64(tab), buckets=buckets, docs=docs, k_docs=k_docs,
                      prefix=prefix, d_out=f64(do) if backward else None, **kw)
    for name, (val, err) in want.items():
        within(name, got[name], val, err)
    if not backward:
        assert torch.equal(attention.attend(q, k, v, *where, **call), o)
    return got


LENS = [1, 0, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 2]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 8, 40, 72])
def test_lengths_and_dims(t, dim):
    check(np.random.default_rng(dim), t, LENS, heads=2, kv_heads=1, dim=dim)


FEATURES = {
    "cap": dict(cap=5.0),
    "slopes": dict(slopes=ref.alibi(4)),
    "table": dict(table=np.random.default_rng(1).standard_normal((8, 4)), buckets=np.arange(-5, 6) % 8),
    "table_gaps": dict(table=np.random.default_rng(2).standard_normal((6, 4)),
                       buckets=np.array([0, -1, 2, 9, 5, 5, 1])),
    "table_far": dict(table=np.random.default_rng(3).standard_normal((32, 4)), buckets=attention.rel_buckets(32, 128)),
    "causal": dict(causal=True),
    "window": dict(window=7),
    "window_0": dict(window=0),
    "window_wide": dict(window=70),
    "causal_window": dict(causal=True, window=40),
    "all": dict(cap=3.0, slopes=ref.alibi(4), table=np.random.default_rng(4).standard_normal((8, 4)),
                buckets=np.arange(-20, 21) % 8, causal=True, window=90),
}


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("name", FEATURES)
def test_scores_and_masks(t, name):
    check(np.random.default_rng(7), t, [130, 1, 33, 257], **FEATURES[name])


@pytest.mark.parametrize("name", ["cap", "table", "all"])
@pytest.mark.parametrize("dim", [48, 128])
def test_scores_at_other_dims(name, dim):
    check(np.random.default_rng(8), "f16", [70, 140], dim=dim, **FEATURES[name])


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_prefix(t):
    check(np.random.default_rng(9), t, [200, 40, 70, 5], causal=True, prefix=np.array([130, 0, 70, 99]))


def test_prefix_in_a_window():
    check(np.random.default_rng(9), "bf16", [200, 150], causal=True, prefix=np.array([130, 3]), window=20)


@pytest.mark.parametrize("name", ["plain", "causal", "all"])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_documents(t, name):
    """Packed, interleaved and padded documents; a sequence that is padding."""
    rng = np.random.default_rng(10)
    lens = [300, 40, 33, 130]
    docs = np.concatenate([np.sort(rng.integers(0, 5, 300)), rng.integers(0, 3, 40), np.full(33, -1),
                           np.sort(rng.integers(0, 2, 130))])
    docs[250:300] = -1
    docs[340 - 7:340] = -7
    check(rng, t, lens, docs=docs, **FEATURES.get(name, {}))


def test_documents_of_one_id_leave_no_mask():
    check(np.random.default_rng(11), "bf16", [256, 128], docs=np.repeat([4, 2], [256, 128]))


def test_padding_holds_anything():
    """NaN and infinities in the rows of padding, in Q, K, V and dO."""
    rng = np.random.default_rng(12)
    lens, docs = [100, 64, 30], np.repeat([0, -1, 1, 2, -1], [70, 30, 64, 20, 10])
    ts = [rows(rng, torch.bfloat16, 194, h, 64) for h in (4, 2, 2, 4)]
    for x in ts:
        x[70:85] = float("nan")
        x[85:100] = float("inf")
        x[184:] = -float("inf")
    clean = [torch.where(torch.from_numpy(docs < 0).cuda()[:, None, None], 0, x) for x in ts]
    got = check(rng, "bf16", lens, docs=docs, tensors=clean)
    again = check_equal_inputs(ts, lens, docs)
    for name in again:
        assert torch.equal(got[name], again[name]), name


def check_equal_inputs(ts, lens, docs):
    q, k, v, do = ts
    offs = ints(np.concatenate([[0], np.cumsum(lens)]))
    o, lse = attention.attend(q, k, v, offs, docs=ints(docs), want_lse=True)
    dq, dk, dv, _ = attention.attend_backward(do, q, k, v, o, lse, offs, docs=ints(docs))
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("kw", [{}, dict(causal=True), dict(window=9), dict(causal=True, cap=4.0, window=33)])
def test_other_lengths_of_queries_and_keys(t, kw):
    """More queries than keys leave rows that see nothing; keys without
    queries and queries without keys."""
    check(np.random.default_rng(13), t, [70, 5, 0, 40, 129, 1], [20, 140, 33, 0, 129, 65], **kw)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (8, 2), (6, 1), (12, 4)])
def test_heads(heads, kv_heads):
    check(np.random.default_rng(14), "bf16", [90, 33], heads=heads, kv_heads=kv_heads, causal=True,
          slopes=ref.alibi(heads))


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("name", ["plain", "cap", "table", "all"])
@pytest.mark.parametrize("heads,copies", [(40, 1), (80, 2)])
def test_keys_past_two_workgroups_a_cu(t, name, heads, copies):
    """Gradients over more keys and key heads than the blocks of 64 keys are
    taken for, a key head each head and shared."""
    lens = [200, 129, 1, 90, 0, 64, 300, 33, 70] * copies
    kv_heads = 40
    assert sum(lens) * kv_heads > 128 * 256 * (heads // kv_heads)
    rng = np.random.default_rng(22)
    kw = {}
    if name in ("cap", "all"):
        kw["cap"] = 4.0
    if name in ("table", "all"):
        kw.update(table=rng.standard_normal((8, heads)), buckets=np.arange(-20, 21) % 8)
    if name == "all":
        docs = np.sort(rng.integers(0, 9, sum(lens)))
        docs[-12:] = -1
        kw.update(slopes=ref.alibi(heads), causal=True, window=90, docs=docs)
    check(rng, t, lens, heads=heads, kv_heads=kv_heads, dim=32, **kw)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 40])
@pytest.mark.parametrize("name", ["plain", "all", "prefix", "documents", "other_keys"])
def test_gradients_of_few_long_sequences(t, dim, name):
    """Few blocks of keys and queries, in parts that are added up; beside a
    long sequence one of a single step and one row."""
    rng = np.random.default_rng(23)
    lens, k_lens, kw = [2010, 30, 1], None, {}
    if t != "f32":
        lens = [2010, 30]
    n = sum(lens)
    if name == "all":
        kw.update(cap=4.0, slopes=ref.alibi(2), table=rng.standard_normal((8, 2)), buckets=np.arange(-20, 21) % 8,
                  causal=True, window=700)
    if name == "prefix":
        kw.update(causal=True, prefix=np.array([900, 3, 0][:len(lens)]))
    if name == "documents":
        docs = np.sort(rng.integers(0, 3, n))
        docs[1990:2010] = -1
        kw["docs"] = docs
    if name == "other_keys":
        k_lens = [800, 1300, 0][:len(lens)]
        kw["causal"] = True
    seed = np.random.default_rng(24)
    first = check(seed, t, lens, k_lens, heads=2, kv_heads=1, dim=dim, **kw)
    again = check(np.random.default_rng(24), t, lens, k_lens, heads=2, kv_heads=1, dim=dim, **kw)
    for out in first:
        assert first[out] is None or torch.equal(first[out], again[out]), out


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (8, 2, 128), (8, 1, 72), (40, 1, 64)])
def test_one_token(t, heads, kv_heads, dim):
    """A single new query over all its keys: with and without shared key
    heads in one block, the keys split and joined."""
    rng = np.random.default_rng(15)
    check(rng, t, [1] * 6, [1, 700, 64, 2001, 0, 333], heads=heads, kv_heads=kv_heads, dim=dim, backward=False,
          slopes=ref.alibi(heads), causal=True)
    check(rng, t, [1, 1], [4100, 3000], heads=heads, kv_heads=kv_heads, dim=dim, backward=False, cap=6.0,
          table=rng.standard_normal((8, heads)), buckets=np.arange(-9, 10) % 8)


def test_few_queries_over_documents_split():
    rng = np.random.default_rng(16)
    docs_k = np.concatenate([np.sort(rng.integers(0, 3, 4000)), np.full(96, -1)])
    check(rng, "bf16", [3], [4096], heads=4, kv_heads=1, docs=np.array([1, 2, -1]), k_docs=docs_k, backward=False)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_long_split_with_window(t):
    check(np.random.default_rng(17), t, [40], [5000], heads=2, kv_heads=1, window=2000, backward=False)


def test_strided_rows():
    """Heads of packed rows, heads before rows, and rows with gaps."""
    rng = np.random.default_rng(18)
    lens = [100, 29]
    qkv = rows(rng, torch.bfloat16, 129, 4 + 2 + 2, 64)
    q, k, v = qkv.split([4, 2, 2], 1)
    do = rows(rng, torch.bfloat16, 4, 129, 64).transpose(0, 1)
    check(rng, "bf16", lens, tensors=(q, k, v, do), causal=True)
    wide = rows(rng, torch.float32, 258, 4, 48)
    check(rng, "f32", lens, dim=40, tensors=(wide[::2, :, :40], wide[1::2, :2, 8:], wide[::2, 2:, :40], wide[1::2, :, 8:]))


def test_outputs_in_slices_and_rows_outside_left():
    rng = np.random.default_rng(19)
    n, lens = 150, [60, 0, 50]
    offs = np.array([20, 80, 80, 130], np.int32)
    q, do = (rows(rng, torch.float16, n, 4, 64) for _ in range(2))
    k, v = (rows(rng, torch.float16, n, 2, 64) for _ in range(2))
    into = torch.full((n, 8, 64), 7.0, dtype=torch.float16, device="cuda")
    o, dq = into[:, :4], torch.full_like(q, 7.0)
    grads = torch.full((n, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    dk, dv = grads.split(2, 1)
    _, lse = attention.attend(q, k, v, ints(offs), out=o, want_lse=True)
    attention.attend_backward(do, q, k, v, o, lse, ints(offs), dq=dq, dk=dk, dv=dv)
    for x in (into, dq, grads):
        assert (x[:20] == 7).all() and (x[130:] == 7).all()
        assert not (x[20:130] == 7).all(-1).all()
    assert (into[:, 4:] == 7).all()
    want = ref.attend(f64(q), f64(k), f64(v), offs, offs, u=half_step(torch.float16), d_out=f64(do))
    for name, x in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv)):
        within(name, x, *want[name])


def test_rows_past_32_bits():
    """Keys whose rows stand more than 2^31 values apart."""
    rng = np.random.default_rng(20)
    step, n = 1 << 23, 300  # values a row: the last at 2.5e9
    room = torch.empty(step * (n - 1) + 256, dtype=torch.bfloat16, device="cuda")
    views = []
    for i, h in enumerate((2, 1, 1)):
        x = room.as_strided((n, h, 64), (step, 64, 1), 64 * (0, 2, 3)[i])
        x.copy_(rows(rng, torch.bfloat16, n, h, 64))
        views.append(x)
    check(rng, "bf16", [40, 260], heads=2, kv_heads=1, tensors=(*views, rows(rng, torch.bfloat16, n, 2, 64)), causal=True)
    q, k, _ = views
    pos = ints(np.arange(n) % 50)
    ang = rng.standard_normal((50, 32)).astype(np.float32)
    cos, sin = torch.from_numpy(np.cos(ang)).cuda(), torch.from_numpy(np.sin(ang)).cuda()
    a = attention.qk_norm_rope(q, k, cos, sin, pos=pos)
    b = attention.qk_norm_rope(q.contiguous(), k.contiguous(), cos, sin, pos=pos)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_large_scores_and_far_rows():
    """Rows whose scores lie far apart: the running maximum jumps, and a
    probability under the type's range is 0."""
    rng = np.random.default_rng(21)
    ts = [rows(rng, torch.bfloat16, 300, h, 64) for h in (4, 2, 2, 4)]
    ts[0] *= 12
    ts[1][::7] *= 9
    check(rng, "bf16", [300], tensors=ts)


def _training(ts, offs, kw):
    q, k, v, do = ts
    o, lse = attention.attend(q, k, v, offs, want_lse=True, **kw)
    return (o, lse, *attention.attend_backward(do, q, k, v, o, lse, offs, **kw))


def test_runs_are_equal_bit_for_bit():
    rng = np.random.default_rng(22)
    offs = ints([0, 500, 700, 1400])
    ts = [rows(rng, torch.bfloat16, 1400, h, 64) for h in (8, 2, 2, 8)]
    kw = dict(table=rows(rng, torch.bfloat16, 32, 8), buckets=ints(attention.rel_buckets(32, 128)), cap=9.0)
    first = _training(ts, offs, kw)
    for _ in range(3):
        for a, b in zip(first, _training(ts, offs, kw)):
            assert torch.equal(a, b)


def test_captured_steps_replay():
    """Two captured training steps and eager calls between their replays, on
    inputs that change; workspaces come from each graph's own memory."""
    rng = np.random.default_rng(23)
    offs = ints([0, 130, 131, 400])
    ts = [rows(rng, torch.bfloat16, 400, h, 64) for h in (4, 2, 2, 4)]
    kws = [dict(causal=True, docs=ints(np.repeat([0, 1], 200))),
           dict(table=rows(rng, torch.bfloat16, 8, 4), buckets=ints(np.arange(-30, 31) % 8))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for kw in kws:
            _training(ts, offs, kw)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for kw in kws:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _training(ts, offs, kw)
        graphs.append((g, out))
    for step in range(4):
        for x in ts:
            x.copy_(rows(rng, torch.bfloat16, *x.shape))
        for g, _ in graphs:
            g.replay()
        eager = [_training(ts, offs, kw) for kw in kws]
        torch.cuda.synchronize()
        for (_, out), want in zip(graphs, eager):
            for a, b in zip(out, want):
                assert (a is None and b is None) or torch.equal(a, b), f"replay {step}"


def test_steps_in_parts_captured_and_at_once():
    """Few long sequences, whose gradients come in parts: two graphs replayed
    on streams of their own at once, with eager calls between."""
    rng = np.random.default_rng(25)
    offs = ints([0, 1700, 2400])
    sets = [[rows(rng, torch.bfloat16, 2400, h, 64) for h in (4, 2, 2, 4)] for _ in range(2)]
    kw = dict(causal=True, table=rows(rng, torch.bfloat16, 8, 4), buckets=ints(np.arange(-30, 31) % 8))
    streams = [torch.cuda.Stream() for _ in sets]
    graphs = []
    for st, ts in zip(streams, sets):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            _training(ts, offs, kw)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _training(ts, offs, kw)
        graphs.append((g, out))
    for step in range(3):
        for ts in sets:
            for x in ts:
                x.copy_(rows(rng, torch.bfloat16, *x.shape))
        torch.cuda.synchronize()
        for st, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for ts, (_, out) in zip(sets, graphs):
            for a, b in zip(out, _training(ts, offs, kw)):
                assert torch.equal(a, b), f"replay {step}"


def test_streams_at_once():
    """Two calls at once on streams of their own, neither the default."""
    rng = np.random.default_rng(24)
    offs = ints([0, 1, 800, 1500])
    sets = [[rows(rng, torch.float16, 1500, h, 64) for h in (4, 2, 2, 4)] for _ in range(2)]
    want = [_training(ts, offs, {}) for ts in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for st, ts in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(_training(ts, offs, {}))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for a, b in zip(g, w):
                assert (a is None and b is None) or torch.equal(a, b)


def test_offsets_out_of_range_read_nothing_out_of_range():
    """Offsets past the rows are taken as their ends (the values are then
    those of the clamped offsets)."""
    rng = np.random.default_rng(25)
    ts = [rows(rng, torch.bfloat16, 90, h, 64) for h in (4, 2, 2, 4)]
    got = _training(ts, ints([-5, 40, 1 << 30]), {})
    want = _training(ts, ints([0, 40, 90]), {})
    for a, b in zip(got[:5], want[:5]):
        assert torch.equal(a, b)


def test_offsets_that_do_not_ascend_stay_inside():
    """Whatever the offsets hold, nothing before the first row, past the last,
    or in a row that no sequence names is written."""
    rng = np.random.default_rng(27)
    n = 700
    q, k, v, do = (rows(rng, torch.bfloat16, n, h, 64) for h in (4, 2, 2, 4))
    table = rows(rng, torch.bfloat16, 8, 4)
    kw = dict(table=table, buckets=ints(np.arange(-9, 10) % 8))
    for offs in ([100, 600, 300, 500, 400], [600, 100, 650, 650, 0], [300, -7, 1 << 30, 200, 600]):
        room = torch.full((3 * n, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        grads = [torch.full((3 * n, h, 64), 7.0, dtype=torch.bfloat16, device="cuda") for h in (4, 2, 2)]
        o = room[n:2 * n]
        _, lse = attention.attend(q, k, v, ints(offs), out=o, want_lse=True, **kw)
        lse = torch.where(torch.isnan(lse), 0.0, lse)
        attention.attend_backward(do, q, k, v, o, lse, ints(offs), dq=grads[0][n:2 * n], dk=grads[1][n:2 * n],
                                  dv=grads[2][n:2 * n], **kw)
        torch.cuda.synchronize()
        for x in (room, *grads):
            assert (x[:n] == 7).all() and (x[2 * n:] == 7).all()
            assert (x[n:n + min(max(offs[0], 0), *(max(a, 0) for a in offs))] == 7).all()


def test_gradient_against_differences():
    """A float32 loss's central difference along the gradient's own
    direction. h moves the scores by about 1e-2, so the third derivative's
    part is under (1e-2)^2 / 6 of the first times a small factor (taken 20),
    3.4e-4 of it; the sums' rounding is smaller by far."""
    rng = np.random.default_rng(26)
    offs = ints([0, 50, 120])
    q, k, v, do = (rows(rng, torch.float32, 120, h, 64) for h in (4, 2, 2, 4))
    table = rows(rng, torch.float32, 8, 4)
    kw = dict(buckets=ints(np.arange(-12, 13) % 8), cap=4.0, causal=True)

    def loss(q, k, v, table):
        return float((attention.attend(q, k, v, offs, table=table, **kw).double() * do.double()).sum())

    o, lse = attention.attend(q, k, v, offs, table=table, want_lse=True, **kw)
    grads = attention.attend_backward(do, q, k, v, o, lse, offs, table=table, **kw)
    xs = [q, k, v, table]
    for i, g in enumerate(grads):
        h = 1e-2 / float(g.abs().max())
        ends = []
        for s in (h, -h):
            moved = list(xs)
            moved[i] = xs[i] + s * g
            ends.append(loss(*moved))
        size = float((g.double() ** 2).sum())
        assert abs((ends[0] - ends[1]) / (2 * h) - size) < 3.4e-4 * size


# ---- norms and rotation -----------------------------------------------------


def rope_case(rng, t, n, heads, kv_heads, dim, rot, gamma, pos_rows=40):
    t = TYPES[t]
    q, k, dq, dk = (rows(rng, t, n, h, dim) for h in (heads, kv_heads, heads, kv_heads))
    ang = rng.uniform(-4, 4, (pos_rows, rot // 2))
    cos, sin = (torch.from_numpy(f(ang).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    pos = rng.integers(0, pos_rows, n)
    gt = torch.float32 if gamma == "f32" else t
    gammas = [None] * 2 if gamma is None else [torch.from_numpy(1 + 0.2 * rng.standard_normal(dim)).to(gt).cuda() for _ in "qk"]
    return q, k, dq, dk, cos, sin, pos, gammas


def check_rope(rng, t, n, heads=3, kv_heads=2, dim=64, rot=64, norm="rms", pairs="halves", gamma="f32", eps=1e-6):
    """Bounds, w = 2^-24, u half a step of the type. Forward: the sums of dim
    terms, the root, the division and four more operations, (dim + 16) w of
    the absolute terms of a rotation |x r gamma| (|c| + |s|) (with a mean
    taken off, of |x| + |mean| in place of |x|), and one rounding. Backward:
    the same of every product's absolute terms; a gamma's gradient sums
    rows * heads of them in 32 bits."""
    q, k, dq, dk, cos, sin, pos, gammas = rope_case(rng, t, n, heads, kv_heads, dim, rot, gamma)
    kw = dict(norm=norm, eps=eps, pairs=pairs)
    call = dict(kw, pos=ints(pos), q_gamma=gammas[0], k_gamma=gammas[1])
    tabs = (cos, sin) if rot else (None, None)
    got = attention.qk_norm_rope(q, k, *tabs, **call)
    back = attention.qk_norm_rope_backward(dq, dk, q, k, *tabs, **call)
    u, w = half_step(TYPES[t]), ref.W
    c, s = (f64(x)[pos] for x in (cos, sin))
    turned = np.concatenate([c, s], 1)
    for i, (x, dy) in enumerate(((q, dq), (k, dk))):
        x, dy = f64(x), f64(dy)
        g = np.ones(dim) if gammas[i] is None else f64(gammas[i])
        y, xh, r = ref.norm_rope(x, g, c, s, **kw)
        size = np.abs(x) + (np.abs(x).mean(-1, keepdims=True) if norm == "layer" else 0)
        terms = ref.turn(size * r * np.abs(g), np.abs(c), -np.abs(s), pairs)  # a|c| + b|s|
        terms = np.maximum(terms, ref.turn(size * r * np.abs(g), np.abs(c), np.abs(s), pairs))
        within("y", got[i], y, u * np.abs(y) + 1.05 * (dim + 16) * w * terms + 1e-30)
        dx, dg = ref.norm_rope_backward(dy, x, g, c, s, **kw)
        d = np.maximum(ref.turn(np.abs(dy), np.abs(c), -np.abs(s), pairs), ref.turn(np.abs(dy), np.abs(c), np.abs(s), pairs))
        dn, xs = d * np.abs(g), size * r
        mean = (dn * xs).mean(-1, keepdims=True)
        terms = (dn + xs * mean + dn.mean(-1, keepdims=True)) * r if norm != "none" else dn
        within("dx", back[i], dx, u * np.abs(dx) + 1.05 * (3 * dim + 32) * w * terms + 1e-30)
        if gammas[i] is not None:
            gu = half_step(gammas[i].dtype)
            within("dgamma", back[2 + i], dg,
                   (gu + w) * np.abs(dg) + 1.05 * (n * x.shape[1] + dim + 32) * w * (d * xs).sum((0, 1)) + 1e-30)
        else:
            assert back[2 + i] is None


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("norm", ["rms", "layer", "none"])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
def test_norm_rope(t, norm, pairs):
    check_rope(np.random.default_rng(30), t, 77, norm=norm, pairs=pairs)


@pytest.mark.parametrize("dim,rot", [(8, 0), (8, 8), (24, 16), (32, 32), (40, 32), (64, 16), (72, 48), (96, 96),
                                     (128, 128), (136, 64), (256, 256)])
def test_norm_rope_dims(dim, rot):
    pairs = "halves" if rot % 16 == 0 else "neighbours"
    check_rope(np.random.default_rng(dim), "bf16", 21, dim=dim, rot=rot, pairs=pairs)
    check_rope(np.random.default_rng(dim), "f32", 5, dim=dim, rot=max(rot - 2, 0), pairs="neighbours", norm="layer")


@pytest.mark.parametrize("n,heads,kv_heads", [(1, 1, 1), (1, 12, 4), (33, 7, 1), (3000, 5, 2)])
@pytest.mark.parametrize("gamma", ["f32", "own", None])
def test_norm_rope_rows_and_gammas(n, heads, kv_heads, gamma):
    check_rope(np.random.default_rng(n), "f16", n, heads, kv_heads, gamma=gamma)


def test_norm_rope_in_place_and_in_slices():
    rng = np.random.default_rng(31)
    q, k, dq, dk, cos, sin, pos, gammas = rope_case(rng, "bf16", 50, 4, 2, 64, 64, "f32")
    call = dict(pos=ints(pos), q_gamma=gammas[0], k_gamma=gammas[1])
    want = attention.qk_norm_rope(q, k, cos, sin, **call)
    back = attention.qk_norm_rope_backward(dq, dk, q, k, cos, sin, **call)
    packed = torch.cat([q, k, q], 1)
    qs, ks, rest = packed.split([4, 2, 4], 1)
    attention.qk_norm_rope(qs, ks, cos, sin, q_out=qs, k_out=ks, **call)
    assert torch.equal(qs, want[0]) and torch.equal(ks, want[1]) and torch.equal(rest, q)
    attention.qk_norm_rope_backward(dq, dk, q, k, cos, sin, dq=dq, dk=dk, **call)
    assert torch.equal(dq, back[0]) and torch.equal(dk, back[1])


def test_norm_rope_places():
    """No pos: the row itself; a place past the tables gives NaN there only."""
    rng = np.random.default_rng(32)
    q, k, _, _, cos, sin, _, _ = rope_case(rng, "f32", 40, 2, 1, 64, 32, None)
    a = attention.qk_norm_rope(q, k, cos, sin)
    b = attention.qk_norm_rope(q, k, cos, sin, pos=ints(np.arange(40)))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    pos = np.arange(40)
    pos[[3, 9]] = 40, -1
    c = attention.qk_norm_rope(q, k, cos, sin, pos=ints(pos))
    for x, y in zip(c, a):
        assert torch.isnan(x[[3, 9], :, :32]).all() and torch.equal(x[[3, 9], :, 32:], y[[3, 9], :, 32:])
        keep = [i for i in range(40) if i not in (3, 9)]
        assert torch.equal(x[keep], y[keep])


def test_nothing_to_do_on_the_gpu():
    q = torch.empty(0, 4, 64, device="cuda")
    offs = ints([0])
    assert attention.attend(q, q, q, offs).shape == (0, 4, 64)
    table = torch.ones(8, 4, device="cuda")
    o, lse = attention.attend(q, q, q, offs, want_lse=True, table=table, buckets=ints(np.zeros(9)))
    r = attention.attend_backward(q, q, q, q, o, lse, offs, table=table, buckets=ints(np.zeros(9)))
    assert not r[3].any()
    g = torch.ones(64, device="cuda")
    attention.qk_norm_rope(q, q, q_gamma=g)
    assert not attention.qk_norm_rope_backward(q, q, q, q, q_gamma=g, k_gamma=g)[2].any()
    # keys without a single query
    k = torch.randn(30, 4, 64, device="cuda")
    _, dk, dv, _ = attention.attend_backward(q, q, k, k, q, torch.empty(4, 0, device="cuda"), ints([0, 0]), ints([0, 30]))
    assert not dk.any() and not dv.any()


def test_arguments_refused():
    q = torch.zeros(4, 2, 64, device="cuda")
    offs = ints([0, 4])
    for bad in (dict(docs=ints([0] * 3)), dict(slopes=torch.zeros(3, device="cuda")), dict(prefix=ints([1, 2])),
                dict(table=torch.zeros(4, 2, device="cuda")), dict(out=torch.zeros(4, 2, 32, device="cuda")),
                dict(out=torch.zeros(4, 2, 64))):
        with pytest.raises(ValueError, match="linalg: Attend"):
            attention.attend(q, q, q, offs, causal=True, **bad)
    with pytest.raises(ValueError, match="another type"):
        attention.attend(q, q.half(), q, offs)
    with pytest.raises(ValueError, match="side by side"):
        attention.attend(q.transpose(1, 2), q, q, offs)
    with pytest.raises(_lib.IxhError, match="strides"):
        attention.attend(torch.zeros(4, 2, 65, device="cuda")[..., :64], q, q, offs)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_a_layer_of_them(t):
    """Norms and rotation, biased attention over padded documents, and back,
    each operator on the one before's outputs, as a training step runs them:
    each output keeps its own operator's bound at its own inputs."""
    rng = np.random.default_rng(40)
    t_ = TYPES[t]
    lens, dim = [150, 70], 64
    n = sum(lens)
    qkv = rows(rng, t_, n, 4 + 2 + 2, dim)
    q, k, v = qkv.split([4, 2, 2], 1)
    do = rows(rng, t_, n, 4, dim)
    pos = np.concatenate([np.arange(m) for m in lens])
    ang = np.arange(150)[:, None] * 10000.0 ** (-np.arange(32) / 32)
    cos, sin = (torch.from_numpy(f(ang).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    gam = [torch.from_numpy(1 + 0.1 * rng.standard_normal(dim)).float().cuda() for _ in "qk"]
    norm = dict(pos=ints(pos), q_gamma=gam[0], k_gamma=gam[1])
    qn, kn = attention.qk_norm_rope(q, k, cos, sin, **norm)
    docs = np.repeat([0, 1, -1, 2], [100, 40, 10, 70])
    got = check(rng, t, lens, tensors=(qn, kn, v, do), docs=docs, cap=20.0,
                table=rng.standard_normal((32, 4)), buckets=attention.rel_buckets(32, 128))
    dq, dk, _, _ = attention.qk_norm_rope_backward(got["dq"], got["dk"], q, k, cos, sin, **norm)
    # against the whole chain in 64 bits, from the rounded q and k on: the
    # gradients' bounds go through the norm's linear backward
    kw = dict(norm="rms", eps=1e-6, pairs="halves")
    for x, g, d, y in ((q, gam[0], got["dq"], dq), (k, gam[1], got["dk"], dk)):
        want, _ = ref.norm_rope_backward(f64(d), f64(x), f64(g), np.cos(ang).astype(np.float32)[pos].astype(np.float64),
                                         np.sin(ang).astype(np.float32)[pos].astype(np.float64), **kw)
        size = np.abs(f64(d)).sum(-1, keepdims=True) * (1 + np.abs(f64(x)))
        within("layer", y, want, half_step(t_) * np.abs(want) + 400 * ref.W * size)
