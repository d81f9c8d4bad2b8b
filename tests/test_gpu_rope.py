"""rq_rope_rows and rq_rope_append against a plain computation in 64 bits and more.

Tolerance of a turned value m (x_a cos t -+ x_b sin t), S = |m| (|x_a| + |x_b|), u = 2^-24:
  * the angle: a fraction of a turn of at most 1/2, rounded to f32 (pi u), formed from a
    product of two roundings in 64 bits (2^-51 of it, which tells for far positions);
  * sine and cosine of it within 2 ulp (2 u each, values up to 1), the product with m (u);
  * one product and one fused multiply-add (u each of values up to S, both):
    together (3.2 + 2 + 1 + 2) u S, taken as 9 u S;
  * the result's own rounding, half a step: 2^-11 (fp16, at least 2^-25) or u of it.
Copied elements are equal bit for bit."""
import numpy as np
import pytest

from rusty_amd import DType, PagedCache, Rope, UnifiedTensor
from rusty_amd.hiprt import Graph, Stream

pytestmark = pytest.mark.gpu

KIND = {"f16": (np.float16, DType.FP16), "f32": (np.float32, DType.FP32)}
U = 2.0 ** -24


def pairs(rot, layout):
    i = np.arange(rot // 2)
    return (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)


def turned(x, positions, freqs, magnitude, rot, layout, sign=1):
    """(result, tolerance) [tokens, heads, dim] in 64 bits, the angles in 80."""
    angle = np.asarray(positions, np.longdouble)[:, None] * np.asarray(freqs, np.longdouble)
    c, s = (np.asarray(f(angle), np.float64)[:, None] * magnitude for f in (np.cos, np.sin))
    x64 = x.astype(np.float64)
    y, tol = x64.copy(), np.zeros(x.shape)
    a, b = pairs(rot, layout)
    xa, xb = x64[..., a], x64[..., b]
    y[..., a], y[..., b] = xa * c - sign * xb * s, xb * c + sign * xa * s
    S = abs(magnitude) * (np.abs(xa) + np.abs(xb))
    e = (9 * U + np.abs(np.asarray(angle, np.float64))[:, None] * 2.0 ** -51) * S
    half, least = (2.0 ** -11, 2.0 ** -25) if x.dtype == np.float16 else (U, 2.0 ** -149)
    for i in (a, b):
        tol[..., i] = e + np.maximum(half * np.abs(y[..., i]), least)
    return y, tol


def check(got, want, tol, what):
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    worst = float(np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300))) if got.size and tol.any() else 0.0
    print(f"[{what}] worst {worst:.3f} of the tolerance", flush=True)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside, first at {np.argwhere(bad)[0]}"


def values(seed, shape, dtype):
    return np.random.default_rng(seed).standard_normal(shape).astype(KIND[dtype][0])


def dev(ctx, a, dtype=None):
    return UnifiedTensor.new(ctx, a, dtype=dtype)


def run_rows(ctx, engine, x, positions, rope, dtype, **kw):
    out = dev(ctx, np.full(x.shape, 7.0), KIND[dtype][1])
    engine.rope(ctx, dev(ctx, x, KIND[dtype][1]), rope, dev(ctx, np.asarray(positions, np.int32), DType.I32), out, **kw)
    return out.to_vec()


SHAPES = [(64, 64), (128, 64), (80, 80), (96, 26), (2, 2), (6, 4), (256, 254), (1024, 1024), (33, 8), (64, 2)]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", SHAPES)
@pytest.mark.parametrize("backward", [False, True])
def test_rows(ctx, engine, dtype, layout, dim, rot, backward):
    tokens, heads = 11, 3
    x = values(dim + rot, (tokens, heads, dim), dtype)
    positions = np.array([0, 1, 2, 5, 100, 4095, 131071, -3, 7, 7, 2 ** 31 - 1])
    rope = Rope(ctx, dim, rot, layout)
    f, m = Rope.frequencies_of(rot)
    want, tol = turned(x, positions, f, m, rot, layout, -1 if backward else 1)
    got = run_rows(ctx, engine, x, positions, rope, dtype, backward=backward)
    check(got, want, tol, f"{dtype} {layout} {dim}/{rot}")


@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 32), (1, 700), (3, 40), (513, 1), (1030, 5), (2500, 2)])
def test_row_counts(ctx, engine, tokens, heads):
    x = values(tokens, (tokens, heads, 64), "f16")
    positions = np.random.default_rng(1).integers(0, 5000, tokens)
    f, m = Rope.frequencies_of(64)
    want, tol = turned(x, positions, f, m, 64, "half")
    check(run_rows(ctx, engine, x, positions, Rope(ctx, 64), "f16"), want, tol, f"{tokens} x {heads}")


@pytest.mark.parametrize("scaling", ["linear", "stretch", "bands", "ramp"])
def test_scalings(ctx, engine, scaling):
    kw = dict(theta=500000.0, scaling=scaling, factor=8.0, trained=8192.0, low=1.0, high=4.0)
    x = values(5, (9, 2, 128), "f32")
    positions = np.arange(9) * 14563
    f, m = Rope.frequencies_of(128, **kw)
    want, tol = turned(x, positions, f, m, 128, "half")
    check(run_rows(ctx, engine, x, positions, Rope(ctx, 128, **kw), "f32"), want, tol, scaling)


def test_own_frequencies(ctx, engine):
    f = np.array([2.0, 0.25, 0.0, -1.0])
    x = values(6, (5, 2, 16), "f32")
    rope = Rope(ctx, 16, 8, "interleaved", frequencies=f, magnitude=-1.5)
    want, tol = turned(x, np.arange(5), f, -1.5, 8, "interleaved")
    check(run_rows(ctx, engine, x, np.arange(5), rope, "f32"), want, tol, "own")
    with pytest.raises(ValueError):
        Rope(ctx, 16, 8, frequencies=f[:3])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("x_row,out_row,shift", [(0, 0, 0), (205, 0, 1), (192 + 8, 192 + 2, 0), (240, 216, 4)])
def test_strides_and_in_place(ctx, engine, dtype, layout, x_row, out_row, shift):
    """Rows of other strides and alignments; what lies between them stays; in place."""
    tokens, heads, dim, rot = 6, 3, 64, 40
    t, kind = KIND[dtype]
    xr, orow = x_row or heads * dim, out_row or heads * dim
    buf = values(8, (tokens * xr + shift,), dtype)
    x = buf[shift:].reshape(tokens, xr)[:, :heads * dim].reshape(tokens, heads, dim)
    positions = np.arange(tokens) * 77
    f, m = Rope.frequencies_of(rot)
    rope, P = Rope(ctx, dim, rot, layout), dev(ctx, positions.astype(np.int32), DType.I32)
    want, tol = turned(x, positions, f, m, rot, layout)
    src, dst = dev(ctx, buf, kind), dev(ctx, np.full(tokens * orow + shift, 7.0), kind)
    size = kind.itemsize
    view = lambda b: UnifiedTensor(ctx, b.ptr + shift * size, (tokens, heads, dim), kind, owner=False)  # noqa: E731
    engine.rope(ctx, view(src), rope, P, view(dst), x_row=x_row or None, out_row=out_row or None)
    got = dst.to_vec()
    assert np.all(got[:shift] == 7.0)
    got = got[shift:].reshape(tokens, orow)
    check(got[:, :heads * dim].reshape(x.shape), want, tol, "out of place")
    assert np.all(got[:, heads * dim:] == 7.0)
    engine.rope(ctx, view(src), rope, P, x_row=x_row or None)
    got = src.to_vec()
    assert np.array_equal(got[:shift], buf[:shift])
    got = got[shift:].reshape(tokens, xr)
    check(got[:, :heads * dim].reshape(x.shape), want, tol, "in place")
    assert np.array_equal(got[:, heads * dim:], buf[shift:].reshape(tokens, xr)[:, heads * dim:])


def test_copied_elements_keep_their_bits(ctx, engine):
    """Past rot_dim: infinities, NaN and signed zeros as they are."""
    x = values(9, (4, 2, 64), "f16")
    x[..., 30:34] = [np.inf, -np.inf, np.nan, -0.0]
    for layout in ("half", "interleaved"):
        got = run_rows(ctx, engine, x, np.arange(4), Rope(ctx, 64, 30, layout), "f16")
        assert np.array_equal(got[..., 30:].view(np.uint16), x[..., 30:].view(np.uint16))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_by_differences(ctx, engine, layout):
    """The backward turn of a direction d is the gradient of sum(d * rope(x)): linear, so differences are exact."""
    x, d = values(10, (7, 2, 32), "f32"), values(11, (7, 2, 32), "f32")
    positions = np.arange(7) * 13
    rope = Rope(ctx, 32, 24, layout, magnitude=1.25)
    grad = run_rows(ctx, engine, d, positions, rope, "f32", backward=True).astype(np.float64)
    for seed in range(4):
        step = values(20 + seed, x.shape, "f32")
        a = run_rows(ctx, engine, x, positions, rope, "f32").astype(np.float64)
        b = run_rows(ctx, engine, (x + step).astype(np.float32), positions, rope, "f32").astype(np.float64)
        moved = (x + step).astype(np.float32).astype(np.float64) - x
        lhs, rhs = (d * (b - a)).sum(), (grad * moved).sum()
        # each of the terms is off by the tolerances above
        bound = 30 * U * 1.25 * 2 * (np.abs(d).sum() * (np.abs(x) + np.abs(step)).max())
        assert abs(lhs - rhs) <= bound


def test_forward_then_backward(ctx, engine):
    """The turn and its gradient with magnitude 1 give x back, up to both tolerances."""
    x = values(12, (50, 3, 64), "f32")
    positions = np.arange(50) * 1000
    rope = Rope(ctx, 64)
    there = run_rows(ctx, engine, x, positions, rope, "f32")
    back = run_rows(ctx, engine, there, positions, rope, "f32", backward=True)
    f, _ = Rope.frequencies_of(64)
    _, tol = turned(x, positions, f, 1.0, 64, "half")
    a, b = pairs(64, "half")
    both = np.empty_like(tol)
    both[..., a] = both[..., b] = tol[..., a] + tol[..., b]
    check(back, x.astype(np.float64), both + tol + 4 * U * np.abs(x).max(), "there and back")


# ---- into the cache ----------------------------------------------------------------


def pool(seed, n_pages, kv, page, dim, order, dtype):
    shape = (n_pages, kv, page, dim) if order == "heads" else (n_pages, page, kv, dim)
    return values(seed, shape, dtype), values(seed + 1, shape, dtype)


def appended(k_pool, v_pool, k, v, table, where, page, order, tol):
    """The pools (in 64 bits, with tolerances) after tokens t at where[t] = (sequence, position) or None."""
    outs = [k_pool.astype(np.float64), v_pool.astype(np.float64)]
    tols = [np.zeros(k_pool.shape), np.zeros(k_pool.shape)]
    for t, w in enumerate(where):
        if w is None or not 0 <= w[1] < table.shape[1] * page:
            continue
        e = table[w[0], w[1] // page]
        if not 0 <= e < k_pool.shape[0]:
            continue
        at = (e, slice(None), w[1] % page) if order == "heads" else (e, w[1] % page)
        outs[0][at], outs[1][at], tols[0][at] = k[t], v[t], tol[t]
    return outs, tols


def run_append(ctx, engine, q, k, v, rope, positions, pools, table, order, starts, dtype, fused=False, in_place=False):
    kind = KIND[dtype][1]
    P = lambda a: dev(ctx, np.asarray(a, np.int32), DType.I32)  # noqa: E731
    K, V = dev(ctx, pools[0], kind), dev(ctx, pools[1], kind)
    cache = PagedCache(K, V, P(table), order)
    kw = {}
    if fused:
        rows = np.concatenate([a.reshape(a.shape[0], -1) for a in (q, k, v)], 1)
        buf, size = dev(ctx, rows, kind), kind.itemsize
        n = rows.shape[1]
        views, first = [], 0
        for a in (q, k, v):
            views.append(UnifiedTensor(ctx, buf.ptr + first * size, a.shape, kind, owner=False))
            first += a[0].size
        kw = dict(q_row=n, k_row=n, v_row=n)
        Q, Kn, Vn = views
    else:
        Q, Kn, Vn = (dev(ctx, a, kind) for a in (q, k, v))
    out = Q if in_place else dev(ctx, np.full(q.shape, 7.0), kind)
    if in_place and fused:
        kw["out_row"] = n
    engine.rope_append(ctx, Q, Kn, Vn, rope, P(positions), cache, out, starts=None if starts is None else P(starts), **kw)
    got = buf.to_vec()[:, :q[0].size].reshape(q.shape) if in_place and fused else out.to_vec()
    return got, K.to_vec(), V.to_vec()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim,rot,layout", [(4, 4, 64, 64, "half"), (8, 2, 128, 64, "interleaved"),
                                                     (3, 1, 64, 26, "half"), (5, 1, 128, 126, "interleaved")])
@pytest.mark.parametrize("page,order", [(1, "heads"), (16, "positions"), (8, "heads"), (64, "heads")])
@pytest.mark.parametrize("fused", [False, True])
def test_append(ctx, engine, dtype, heads, kv, dim, rot, layout, page, order, fused):
    """Sequences of 0 to 40 new tokens behind some cached ones, in random pages; nothing else moves."""
    g = np.random.default_rng(page + heads)
    counts, before = [3, 0, 40, 1, 17], [5, 9, 0, 63, 30]
    starts = np.concatenate([[0], np.cumsum(counts)])
    need = [-(-(a + b) // page) for a, b in zip(counts, before)]
    table = np.full((5, max(need)), -1, np.int32)
    order_of = g.permutation(sum(need) + 3)
    first = 0
    for s, n in enumerate(need):
        table[s, :n] = order_of[first:first + n]
        first += n
    total = int(starts[-1])
    positions = np.concatenate([b + np.arange(c) for b, c in zip(before, counts)])
    where = [(s, b + i) for s, (b, c) in enumerate(zip(before, counts)) for i in range(c)]
    q, k, v = (values(20 + i, (total, n, dim), dtype) for i, n in enumerate((heads, kv, kv)))
    pools = pool(30, sum(need) + 3, kv, page, dim, order, dtype)
    rope, (f, m) = Rope(ctx, dim, rot, layout), Rope.frequencies_of(rot)
    wq, tq = turned(q, positions, f, m, rot, layout)
    wk, tk = turned(k, positions, f, m, rot, layout)
    outs, tols = appended(*pools, wk, v.astype(np.float64), table, where, page, order, tk)
    for in_place in (False, True):
        got, K, V = run_append(ctx, engine, q, k, v, rope, positions, pools, table, order, starts, dtype, fused, in_place)
        check(got, wq, tq, "q")
        check(K, outs[0], tols[0], "k pages")
        assert np.array_equal(V, outs[1].astype(V.dtype))


def test_append_bad_places(ctx, engine):
    """Positions below zero or past the capacity and entries of no page cache nothing; q is
    turned all the same.  Tokens of no sequence: nothing at all, their rows stay."""
    table = np.array([[2, -1, 9], [0, 5, 2 ** 31 - 1]], np.int32)  # 6 pages of 8
    starts = [2, 10, 13]
    positions = np.array([0, 1, 0, 7, 8, 15, 16, -1, 24, 3, 9, 23, -2 ** 31, 4, 5])
    where = [None, None] + [(0, p) for p in positions[2:10]] + [(1, p) for p in positions[10:13]] + [None, None]
    q, k, v = (values(40 + i, (15, n, 64), "f16") for i, n in enumerate((4, 2, 2)))
    pools = pool(50, 6, 2, 8, 64, "heads", "f16")
    f, m = Rope.frequencies_of(64)
    wq, tq = turned(q, positions, f, m, 64, "half")
    wk, tk = turned(k, positions, f, m, 64, "half")
    outs, tols = appended(*pools, wk, v.astype(np.float64), table, where, 8, "heads", tk)
    got, K, V = run_append(ctx, engine, q, k, v, Rope(ctx, 64), positions, pools, table, "heads", starts, "f16")
    assert np.all(got[:2] == 7.0) and np.all(got[13:] == 7.0)
    check(got[2:13], wq[2:13], tq[2:13], "q")
    check(K, outs[0], tols[0], "k pages")
    assert np.array_equal(V, outs[1].astype(V.dtype))


@pytest.mark.parametrize("n_seqs", [1, 63, 64, 65, 300])
def test_append_many_sequences(ctx, engine, n_seqs):
    """One token per sequence, with starts and without; and sequences of 0 to 2 tokens."""
    g = np.random.default_rng(n_seqs)
    table = g.permutation(2 * n_seqs).reshape(n_seqs, 2).astype(np.int32)
    f, m = Rope.frequencies_of(64)
    for counts in (np.ones(n_seqs, int), g.integers(0, 3, n_seqs)):
        starts = np.concatenate([[0], np.cumsum(counts)])
        total = int(starts[-1])
        if not total:
            continue
        seq = np.repeat(np.arange(n_seqs), counts)
        at = g.integers(0, 30, n_seqs)
        positions = np.concatenate([at[s] + np.arange(c) for s, c in enumerate(counts)])
        q, k, v = (values(60 + i, (total, n, 64), "f16") for i, n in enumerate((2, 1, 1)))
        pools = pool(70, 2 * n_seqs, 1, 16, 64, "heads", "f16")
        wk, tk = turned(k, positions, f, m, 64, "half")
        outs, tols = appended(*pools, wk, v.astype(np.float64), table, list(zip(seq, positions)), 16, "heads", tk)
        for st in ([starts, None] if counts.min() == counts.max() == 1 else [starts]):
            got, K, V = run_append(ctx, engine, q, k, v, Rope(ctx, 64), positions, pools, table, "heads", st, "f16")
            check(got, *turned(q, positions, f, m, 64, "half"), "q")
            check(K, outs[0], tols[0], "k pages")
            assert np.array_equal(V, outs[1].astype(V.dtype))


def test_graph_and_stream(ctx, engine):
    """Captured on a caller's stream and replayed with other positions."""
    stream, rope = Stream(), Rope(ctx, 64)
    f, m = Rope.frequencies_of(64)
    x = values(80, (5, 4, 64), "f16")
    X, out = dev(ctx, x), dev(ctx, np.zeros_like(x))
    P = dev(ctx, np.zeros(5, np.int32), DType.I32)
    ctx.sync()
    graph = Graph(stream.h, lambda: engine.rope(ctx, X, rope, P, out, stream=stream.h))
    from rusty_amd._lib import call
    for i in range(4):
        positions = np.arange(5, dtype=np.int32) * (i + 1)
        call("rq_memcpy_h2d", ctx.handle, P.ptr, positions.ctypes.data, positions.nbytes, None)
        ctx.sync()
        graph.launch()
        stream.synchronize()
        check(out.to_vec(), *turned(x, positions, f, m, 64, "half"), f"replay {i}")


def test_refusals(ctx, engine):
    x, P = dev(ctx, np.zeros((3, 2, 64), np.float16)), dev(ctx, np.zeros(3, np.int32), DType.I32)
    rope = Rope(ctx, 64)
    for args in ((x, rope, dev(ctx, np.zeros(4, np.int32), DType.I32), None), (x, Rope(ctx, 32), P, None),
                 (x, rope, dev(ctx, np.zeros(3, np.uint32)), None), (x, rope, P, dev(ctx, np.zeros((3, 2, 64), np.float32)))):
        with pytest.raises(ValueError):
            engine.rope(ctx, *args)
    with pytest.raises(ValueError):
        Rope(ctx, 64, layout="other")
