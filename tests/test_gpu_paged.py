"""rq_attn_paged against a plain computation in 64 bits; the tolerances are those
derived in test_gpu_attn.py (the same arithmetic, the keys in pages)."""
import numpy as np
import pytest

from rusty_amd import DType, PagedCache, QuantizedTensor, UnifiedTensor
from rusty_amd._lib import call
from rusty_amd.hiprt import Graph, Stream
from test_gpu_attn import KIND, attend, check

pytestmark = pytest.mark.gpu

NAN = float("nan")


def make(seed, lengths, heads, kv, dim, page, order, dtype, extra=2, fill=NAN, width=None):
    """q, pools whose rows that hold no cached position are `fill`, the table (pages of
    random places, -1 past the end), and per sequence its keys and values [kv, length, dim]."""
    g = np.random.default_rng(seed)
    t = KIND[dtype][0]
    need = [-(-n // page) for n in lengths]
    places = g.permutation(sum(need) + extra)
    table = np.full((len(lengths), max(width or 0, max(need), 1)), -1, np.int32)
    shape = (sum(need) + extra, kv, page, dim)
    pools = [np.full(shape, fill, t) for _ in range(2)]
    rows, first = [], 0
    for s, n in enumerate(lengths):
        table[s, :need[s]] = places[first:first + need[s]]
        first += need[s]
        kv_rows = [g.standard_normal((kv, n, dim)).astype(t) for _ in range(2)]
        for pool, r in zip(pools, kv_rows):
            for i in range(need[s]):
                part = r[:, i * page:(i + 1) * page]
                pool[table[s, i], :, :part.shape[1]] = part
        rows.append(kv_rows)
    if order == "positions":
        pools = [np.ascontiguousarray(p.transpose(0, 2, 1, 3)) for p in pools]
    return g.standard_normal((len(lengths), heads, dim)).astype(t), pools, table, rows


def truth(q, rows, scale, f16, keep=None):
    n_seqs, heads, dim = q.shape
    o, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s, (k, v) in enumerate(rows):
        n, grp = k.shape[1], heads // k.shape[0]
        for g in range(k.shape[0]):
            see = np.ones((grp, n), bool) if keep is None else np.tile(keep[s], (grp, 1))
            h = slice(g * grp, (g + 1) * grp)
            o[s, h], tol[s, h] = attend(q[s, h], k[g], v[g], see, scale, f16)
    return o, tol


def dev(ctx, a, dtype=None):
    return UnifiedTensor.new(ctx, a, dtype=dtype)


def run(ctx, engine, q, pools, table, lengths, order, dtype, **kw):
    kind = KIND[dtype][1]
    cache = PagedCache(dev(ctx, pools[0], kind), dev(ctx, pools[1], kind), dev(ctx, table, DType.I32), order)
    Q, out = dev(ctx, q, kind), dev(ctx, np.full(q.shape, 7.0), kind)
    work = engine.attn_paged_workspace(ctx, Q, cache)
    call("rq_memset", ctx.handle, work.ptr, 0xFF, work.nbytes, None)  # NaN: nothing of it may be read before it is written
    engine.attn_paged(ctx, Q, cache, dev(ctx, np.asarray(lengths, np.int32), DType.I32), out, workspace=work, **kw)
    return out.to_vec()


LENGTHS = {"one": [1], "zeros": [0, 1, 0, 0, 3, 0], "edges": [15, 16, 17, 31, 32, 33, 63, 64, 65], "tiles": [127, 128, 129, 130],
           "ragged": [700, 2, 350, 41, 0, 1], "long": [3000]}
HEADS = [(4, 4, 64), (8, 1, 64), (6, 2, 128), (5, 1, 128), (40, 2, 64), (33, 1, 128)]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("page,order", [(16, "heads"), (64, "positions"), (1, "heads"), (8, "positions")])
def test_paged(ctx, engine, dtype, heads, kv, dim, lengths, page, order):
    n = LENGTHS[lengths]
    q, pools, table, rows = make(len(lengths) + heads + page, n, heads, kv, dim, page, order, dtype)
    want, tol = truth(q, rows, 1 / np.sqrt(dim), dtype == "f16")
    check(run(ctx, engine, q, pools, table, n, order, dtype), want, tol, f"{lengths} {heads}/{kv}x{dim} {dtype} page {page}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n_seqs,most", [(64, 40), (65, 300), (130, 5), (1000, 3), (4200, 2)])
def test_many_sequences(ctx, engine, dtype, n_seqs, most):
    """More sequences than a wave has lanes; zero-length ones among them."""
    n = np.random.default_rng(n_seqs).integers(0, most + 1, n_seqs).tolist()
    q, pools, table, rows = make(n_seqs, n, 2, 1, 64, 4, "heads", dtype)
    want, tol = truth(q, rows, 1 / 8, dtype == "f16")
    check(run(ctx, engine, q, pools, table, n, "heads", dtype), want, tol, f"{n_seqs} sequences {dtype}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim,lengths,page", [(8, 2, 64, [20000, 5, 130, 9000], 256), (4, 1, 128, [30000], 16),
                                                       (32, 8, 128, [5000, 4000], 32), (16, 16, 64, [3000, 1, 2999], 128)])
def test_cut_sequences(ctx, engine, dtype, heads, kv, dim, lengths, page):
    """Long sequences, cut over many blocks, beside short ones."""
    q, pools, table, rows = make(7, lengths, heads, kv, dim, page, "heads", dtype)
    want, tol = truth(q, rows, 1 / np.sqrt(dim), dtype == "f16")
    check(run(ctx, engine, q, pools, table, lengths, "heads", dtype), want, tol, f"cut {lengths} {dtype}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_every_key_once(ctx, engine, dtype):
    """Keys of one score and values of whole numbers: the mean comes out exactly wherever it is cut."""
    for n, page in ((1, 1), (47, 16), (1024, 16), (4096, 64), (8192, 8)):
        q, pools, table, _ = make(n, [n], 4, 2, 64, page, "heads", dtype, fill=0.0)
        v = np.zeros(pools[1].shape, pools[1].dtype)
        # position p has the value 1 in dimension p % 64: each mean is its count / n
        for p in range(n):
            v[table[0, p // page], :, p % page, p % 64] = 1.0
        got = run(ctx, engine, np.zeros_like(q), [pools[0], v], table, [n], "heads", dtype)
        count = np.bincount(np.arange(n) % 64, minlength=64)
        want = (count / n).astype(np.float32).astype(v.dtype)
        assert np.array_equal(got, np.broadcast_to(want, got.shape)), (n, page)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_missing_pages(ctx, engine, dtype):
    """Entries that name no page (below zero, past the pool) hide their positions; a
    sequence with none left gets zeros."""
    n, page = [100, 64, 300, 33], 16
    q, pools, table, rows = make(3, n, 6, 2, 64, page, "heads", dtype, width=30)
    bad = [[1, 3], [0, 1, 2, 3], [0, 5, 6, 18], [2]]
    keep = []
    for s, cut in enumerate(bad):
        k = np.ones(n[s], bool)
        for j, c in enumerate(cut):
            table[s, c] = [-1, len(pools[0]), 2 ** 31 - 1, -2 ** 31][j % 4]
            k[c * page:(c + 1) * page] = False
        keep.append(k)
    want, tol = truth(q, rows, 1 / 8, dtype == "f16", keep)
    got = run(ctx, engine, q, pools, table, n, "heads", dtype)
    check(got, want, tol, "missing pages")
    assert np.all(got[1] == 0)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_lengths_are_clamped(ctx, engine, dtype):
    """Below zero: none; past the capacity: all of it."""
    q, pools, table, rows = make(4, [48, 48, 48], 4, 2, 64, 16, "heads", dtype)
    want, tol = truth(q, [[r[:, :n] for r in rows[s]] for s, n in enumerate((0, 48, 48))], 1 / 8, dtype == "f16")
    check(run(ctx, engine, q, pools, table, [-5, 1 << 30, 49], "heads", dtype), want, tol, "clamped")


def test_empty_pool(ctx, engine):
    """A cache of no pages: zeros."""
    kind = DType.FP16
    k = UnifiedTensor(ctx, 0, (0, 2, 16, 64), kind, owner=False)
    cache = PagedCache(k, k, dev(ctx, np.zeros((3, 4), np.int32), DType.I32))
    q, out = dev(ctx, np.ones((3, 4, 64), np.float16)), dev(ctx, np.full((3, 4, 64), 7.0, np.float16))
    engine.attn_paged(ctx, q, cache, dev(ctx, np.array([0, 5, 64], np.int32), DType.I32), out)
    assert np.all(out.to_vec() == 0)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_values_that_are_not_finite(ctx, engine, dtype):
    """Infinities and NaN at seen positions reach the heads and dimensions that plain
    arithmetic gives, and no other."""
    n = [70, 200]
    q, pools, table, rows = make(5, n, 4, 2, 64, 16, "heads", dtype)
    def put(s, p, g, dim, value, what):
        rows[s][what][g, p, dim] = value
        pools[what][table[s, p // 16], g, p % 16, dim] = value
    put(0, 3, 0, 5, np.inf, 1)
    put(0, 69, 0, 6, NAN, 1)
    put(1, 150, 1, 7, -np.inf, 1)
    put(1, 10, 0, 0, NAN, 0)  # a NaN score: the whole head
    got = run(ctx, engine, q, pools, table, n, "heads", dtype)
    assert np.all(got[0, :2, 5] == np.inf) and np.all(np.isnan(got[0, :2, 6])) and np.all(got[1, 2:, 7] == -np.inf)
    assert np.all(np.isnan(got[1, :2]))
    finite = np.isfinite(got)
    assert finite.sum() == got.size - 2 - 2 - 2 - 2 * 64
    clean = [[np.where(np.isfinite(r), r, 0) for r in p] for p in rows]
    want, tol = truth(q, clean, 1 / 8, dtype == "f16")
    check(got[finite], want[finite], tol[finite], "the others")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_scores_of_minus_infinity(ctx, engine, dtype):
    """One key's score is -inf: it has no weight; all of them: NaN, as 0 / 0."""
    q, pools, table, rows = make(6, [40, 300], 2, 1, 64, 16, "heads", dtype)
    q = np.abs(q) + np.asarray(0.5, q.dtype)
    for s in range(2):
        for p in range(40 if s == 0 else 299):
            rows[s][0][0, p, 0] = -np.inf
            pools[0][table[s, p // 16], 0, p % 16, 0] = -np.inf
    got = run(ctx, engine, q, pools, table, [40, 300], "heads", dtype)
    assert np.all(np.isnan(got[0]))
    want, tol = truth(q[1:], [[r[:, 299:] for r in rows[1]]], 1 / 8, dtype == "f16")
    check(got[1:], want, tol, "one left")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("scale", [-0.3, 1e-30, 4.0])
def test_scale(ctx, engine, dtype, scale):
    q, pools, table, rows = make(8, [90, 5], 6, 3, 64, 32, "positions", dtype)
    want, tol = truth(q, rows, np.float64(np.float32(scale)), dtype == "f16")
    check(run(ctx, engine, q, pools, table, [90, 5], "positions", dtype, scale=scale), want, tol, f"scale {scale}")


def test_rows_and_tables_of_other_strides(ctx, engine):
    """q in the rows of a fused product, out with gaps, a table wider than its sequences, the
    pages of K and V inside larger ones."""
    n, heads, kv, dim, page = [100, 3, 77], 8, 2, 64, 16
    q, pools, table, rows = make(9, n, heads, kv, dim, page, "heads", "f16")
    want, tol = truth(q, rows, 1 / 8, True)
    wide = [np.full((p.shape[0], 2, kv, page, dim + 8), NAN, np.float16) for p in pools]
    for w, p in zip(wide, pools):
        w[:, 1, ..., :dim] = p
    K, V = (dev(ctx, w) for w in wide)
    first = kv * page * (dim + 8) * 2
    view = lambda t: UnifiedTensor(ctx, t.ptr + first, pools[0].shape, DType.FP16, owner=False)  # noqa: E731
    strides = (2 * kv * page * (dim + 8), page * (dim + 8), dim + 8)
    T = dev(ctx, np.concatenate([table, np.full((3, 5), 3, np.int32)], 1), DType.I32)
    narrow = UnifiedTensor(ctx, T.ptr, table.shape, DType.I32, owner=False)
    cache = PagedCache(view(K), view(V), narrow, strides=strides)
    cache.descriptor.table_row = T.shape[1]
    row, orow = (heads + 2 * kv) * dim, heads * dim + 24
    fused = np.full((3, row), NAN, np.float16)
    fused[:, :heads * dim] = q.reshape(3, -1)
    F, out = dev(ctx, fused), dev(ctx, np.full((3, orow), 7.0, np.float16))
    L = dev(ctx, np.array(n, np.int32), DType.I32)
    as_rows = lambda t: UnifiedTensor(ctx, t.ptr, q.shape, DType.FP16, owner=False)  # noqa: E731
    engine.attn_paged(ctx, as_rows(F), cache, L, as_rows(out), q_row=row, out_row=orow)
    got = out.to_vec()
    check(got[:, :heads * dim].reshape(q.shape), want, tol, "strided")
    assert np.all(got[:, heads * dim:] == 7.0)


def test_graph_two_calls_and_stream(ctx, engine):
    """Two captured calls with workspaces of their own, replayed in turn as the lengths
    grow, between eager calls."""
    stream = Stream()
    n = [900, 40, 3]
    q, pools, table, rows = make(10, n, 8, 2, 64, 16, "heads", "f16")
    cache = PagedCache(dev(ctx, pools[0]), dev(ctx, pools[1]), dev(ctx, table, DType.I32))
    Q, L = dev(ctx, q), dev(ctx, np.zeros(3, np.int32), DType.I32)
    outs = [dev(ctx, np.full(q.shape, 7.0, np.float16)) for _ in range(3)]
    works = [engine.attn_paged_workspace(ctx, Q, cache) for _ in range(3)]
    ctx.sync()
    graphs = [Graph(stream.h, lambda i=i: engine.attn_paged(ctx, Q, cache, L, outs[i], workspace=works[i], stream=stream.h))
              for i in range(2)]
    for lengths in ([1, 1, 1], [700, 0, 2], [900, 40, 3], [33, 40, 0]):
        h = np.array(lengths, np.int32)
        call("rq_memcpy_h2d", ctx.handle, L.ptr, h.ctypes.data, h.nbytes, None)
        ctx.sync()
        want, tol = truth(q, [[r[:, :m] for r in rows[s]] for s, m in enumerate(lengths)], 1 / 8, True)
        graphs[0].launch()
        graphs[1].launch()
        stream.synchronize()
        engine.attn_paged(ctx, Q, cache, L, outs[2], workspace=works[2])
        eager = outs[2].to_vec()
        check(eager, want, tol, f"eager {lengths}")
        for o in outs[:2]:
            assert np.array_equal(o.to_vec(), eager)


def test_same_result_every_time(ctx, engine):
    q, pools, table, _ = make(11, [5000, 17, 800], 8, 2, 128, 16, "heads", "f16")
    first = run(ctx, engine, q, pools, table, [5000, 17, 800], "heads", "f16")
    for _ in range(3):
        assert np.array_equal(run(ctx, engine, q, pools, table, [5000, 17, 800], "heads", "f16"), first)


def test_refusals(ctx, engine):
    q, pools, table, _ = make(12, [5, 6], 4, 2, 64, 16, "heads", "f16")
    K, T = dev(ctx, pools[0]), dev(ctx, table, DType.I32)
    cache, Q, L = PagedCache(K, K, T), dev(ctx, q), dev(ctx, np.array([5, 6], np.int32), DType.I32)
    for bad in (lambda: PagedCache(K, K, L), lambda: PagedCache(K, dev(ctx, pools[0].astype(np.float32)), T),
                lambda: PagedCache(K, K, T, "pages"), lambda: engine.attn_paged(ctx, Q, cache, dev(ctx, np.zeros(3, np.int32), DType.I32), Q),
                lambda: engine.attn_paged(ctx, dev(ctx, q.astype(np.float32)), cache, L, dev(ctx, q.astype(np.float32))),
                lambda: engine.attn_paged(ctx, dev(ctx, q[:1]), cache, L, dev(ctx, q[:1]))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim,lengths,page", [(8, 2, 64, [9000, 5, 130, 700], 64), (16, 1, 128, [3000, 2000], 16),
                                                       (40, 2, 64, [2500], 8), (6, 6, 128, [900, 800, 0, 700], 32)])
def test_on_a_callers_stream(ctx, engine, dtype, heads, kv, dim, lengths, page):
    """Cut sequences on another stream than the context's, where their pieces are joined by a launch of its own."""
    stream = Stream()
    q, pools, table, rows = make(13, lengths, heads, kv, dim, page, "heads", dtype)
    want, tol = truth(q, rows, 1 / np.sqrt(dim), dtype == "f16")
    kind = KIND[dtype][1]
    cache = PagedCache(dev(ctx, pools[0], kind), dev(ctx, pools[1], kind), dev(ctx, table, DType.I32))
    Q, out, L = dev(ctx, q, kind), dev(ctx, np.full(q.shape, 7.0), kind), dev(ctx, np.array(lengths, np.int32), DType.I32)
    work = engine.attn_paged_workspace(ctx, Q, cache)
    call("rq_memset", ctx.handle, work.ptr, 0xFF, work.nbytes, None)
    ctx.sync()
    for _ in range(2):
        engine.attn_paged(ctx, Q, cache, L, out, workspace=work, stream=stream.h)
        stream.synchronize()
        check(out.to_vec(), want, tol, f"caller's stream {lengths} {dtype}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_graphs_on_the_contexts_stream(ctx, engine, dtype):
    """Two calls captured on the context's own stream, whose cut sequences are joined through the context's counters,
    with workspaces of their own: replayed in turn, with a product that uses the same counters and eager calls between."""
    n = [4000, 40, 2500]
    q, pools, table, rows = make(14, n, 8, 2, 64, 16, "heads", dtype)
    kind = KIND[dtype][1]
    cache = PagedCache(dev(ctx, pools[0], kind), dev(ctx, pools[1], kind), dev(ctx, table, DType.I32))
    Q, L = dev(ctx, q, kind), dev(ctx, np.zeros(3, np.int32), DType.I32)
    outs = [dev(ctx, np.full(q.shape, 7.0), kind) for _ in range(3)]
    works = [engine.attn_paged_workspace(ctx, Q, cache) for _ in range(3)]
    g = np.random.default_rng(15)
    w = QuantizedTensor.rowwise(ctx, g.integers(-127, 128, (512, 4096)).astype(np.int8), np.full(512, 0.01, np.float32))
    X = dev(ctx, g.standard_normal((64, 4096)).astype(np.float16))
    Y = [dev(ctx, np.zeros((64, 512), np.float32)) for _ in range(2)]
    engine.qmatmul(ctx, X, w, Y[0])
    first = Y[0].to_vec()
    ctx.sync()
    graphs = [Graph(ctx.stream, lambda i=i: engine.attn_paged(ctx, Q, cache, L, outs[i], workspace=works[i])) for i in range(2)]
    for lengths in ([4000, 40, 2500], [1, 0, 2], [3999, 1, 700], [33, 40, 2500]):
        h = np.array(lengths, np.int32)
        call("rq_memcpy_h2d", ctx.handle, L.ptr, h.ctypes.data, h.nbytes, None)
        ctx.sync()
        want, tol = truth(q, [[r[:, :m] for r in rows[s]] for s, m in enumerate(lengths)], 1 / 8, dtype == "f16")
        graphs[0].launch()
        engine.qmatmul(ctx, X, w, Y[1])
        graphs[1].launch()
        engine.attn_paged(ctx, Q, cache, L, outs[2], workspace=works[2])
        eager = outs[2].to_vec()
        check(eager, want, tol, f"eager {lengths}")
        for o in outs[:2]:
            assert np.array_equal(o.to_vec(), eager)
        assert np.array_equal(Y[1].to_vec(), first)
