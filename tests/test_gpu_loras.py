"""rq_qmatmul_loras against a plain computation in 64 bits.

Tolerance, per output, u = 2^-24, W the shared weight, P = sum |x| |W|, T_r = sum |x| |A_r|:
  * the shared product in f32: (k + 16) u P; f32 rows of up to 16 carried as two fp16 terms, 2^-21 P
    more; past 16 rows f32 X and affine weights are rounded to fp16, half a step each: 2^-10 P;
  * t_r = x . A_r, f32 sums of exact or rounded products: (k + 8) u T_r;
  * factor t . B, f32: (rank + 8) u of sum |f t_r b_r|, and t's error in it;
  * their sum (u) and the rounding to the output's type: 2^-11 (fp16, at least 2^-25) or u."""
import ctypes

import numpy as np
import pytest

from rusty_amd import DType, LoraSet, QuantizedTensor, UnifiedTensor, _lib, synth
from rusty_amd._lib import call
from rusty_amd.hiprt import Graph, Stream

pytestmark = pytest.mark.gpu

KIND = {"f16": (np.float16, DType.FP16), "f32": (np.float32, DType.FP32)}
U = 2.0 ** -24


def dev(ctx, a, dtype=None):
    return UnifiedTensor.new(ctx, a, dtype=dtype)


def weight(ctx, g, n, k, form):
    """(the device weight, its values in 64 bits)"""
    if form == "rowwise8":
        q, s = g.integers(-127, 128, (n, k)).astype(np.int8), (g.random(n) * 0.01).astype(np.float32)
        return QuantizedTensor.rowwise(ctx, q, s), q * s.astype(np.float64)[:, None]
    bits = 4 if form == "affine4" else 8
    u = g.integers(0, 1 << bits, (n, k)).astype(np.uint8)
    s = ((g.random((n, k // 64)) + 0.5) * 0.1 / (1 << bits)).astype(np.float32)
    b = (-s * (1 << (bits - 1))).astype(np.float32)
    w = u * np.repeat(s.astype(np.float64), 64, 1) + np.repeat(b.astype(np.float64), 64, 1)
    make = QuantizedTensor.affine4 if bits == 4 else QuantizedTensor.affine
    return make(ctx, u, s, b, 64), w


def truth(x, w, a, b, factors, ids, ranks, out, rounded):
    """(y, tolerance); a [n, rank, k], b [n, rank, n_out]."""
    x = x.astype(np.float64)
    k = x.shape[1]
    P = np.abs(x) @ np.abs(w).T
    y = x @ w.T
    tol = ((k + 16) * U + 2.0 ** -21 + (2.0 ** -10 if rounded else 0.0)) * P
    for t, i in enumerate(ids):
        if not 0 <= i < len(a):
            continue
        r = ranks[i]
        ai, bi, f = a[i, :r].astype(np.float64), b[i, :r].astype(np.float64), float(factors[i])
        v, T = ai @ x[t], np.abs(ai) @ np.abs(x[t])
        y[t] += f * (v @ bi)
        tol[t] += ((k + 8) * U * abs(f)) * (T @ np.abs(bi)) + (r + 8) * U * abs(f) * (T @ np.abs(bi))
    tol += U * np.abs(y)
    half, least = (2.0 ** -11, 2.0 ** -25) if out == "f16" else (U, 2.0 ** -149)
    return y, tol * (1 + half) + np.maximum(half * np.abs(y), least)


def check(got, want, tol, what):
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    worst = float(np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300))) if got.size else 0.0
    print(f"[{what}] worst {worst:.3f} of the tolerance", flush=True)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside, first at {np.argwhere(bad)[0]}"


def adapters(g, n, rank, k, n_out, dtype):
    t = KIND[dtype][0]
    return (g.standard_normal((n, rank, k)) / max(k, 1) ** 0.5).astype(t), (g.standard_normal((n, rank, n_out)) * 0.1).astype(t)


def run(ctx, engine, x, w, a, b, factors, ids, ranks, x_t, y_t, a_t, **kw):
    s = LoraSet(dev(ctx, a, KIND[a_t][1]), dev(ctx, b, KIND[a_t][1]),
                None if factors is None else dev(ctx, factors, DType.FP32),
                None if ranks is None else dev(ctx, np.asarray(ranks, np.int32), DType.I32))
    X = dev(ctx, x, KIND[x_t][1])
    out = dev(ctx, np.full((len(ids), w.n_out), 7.0), KIND[y_t][1])
    work = engine.qmatmul_loras_workspace(ctx, X, w, s, out)
    call("rq_memset", ctx.handle, work.ptr, 0xFF, work.nbytes, None)  # NaN
    engine.qmatmul_loras(ctx, X, w, s, dev(ctx, np.asarray(ids, np.int32), DType.I32), out, workspace=work, **kw)
    return out.to_vec()


def case(ctx, engine, seed, m, n, k, count, rank, form, x_t, y_t, a_t, ids=None, some_ranks=False):
    g = np.random.default_rng(seed)
    w, w64 = weight(ctx, g, n, k, form)
    a, b = adapters(g, count, rank, k, n, a_t)
    factors = (g.random(count) + 0.5).astype(np.float32)
    x = g.standard_normal((m, k)).astype(KIND[x_t][0])
    ids = g.integers(-1, count, m) if ids is None else np.asarray(ids)
    ranks = g.integers(0, rank + 1, count) if some_ranks else np.full(count, rank)
    if some_ranks:
        for i, r in enumerate(ranks):
            a[i, r:], b[i, r:] = np.nan, np.inf  # never read
    rounded = m > 16 and (x_t == "f32" or form == "affine8") or (form == "affine4" and m > 48)
    want, tol = truth(x, w64, a, b, factors, ids, ranks, y_t, rounded)
    got = run(ctx, engine, x, w, a, b, factors, ids, ranks if some_ranks else None, x_t, y_t, a_t)
    check(got, want, tol, f"{m}x{n}x{k} {count} of rank {rank} {form} {x_t}/{y_t}/{a_t}")


TYPES = [("f16", "f16", "f16"), ("f32", "f32", "f32"), ("f16", "f32", "f32"), ("f32", "f16", "f16")]


@pytest.mark.parametrize("x_t,y_t,a_t", TYPES)
@pytest.mark.parametrize("m", [1, 2, 3, 15, 16, 17, 48, 64, 65, 256, 257, 330])
@pytest.mark.parametrize("rank", [1, 4, 16, 21, 40])
def test_rows_and_ranks(ctx, engine, x_t, y_t, a_t, m, rank):
    case(ctx, engine, m + rank, m, 256, 512, 5, rank, "rowwise8", x_t, y_t, a_t)


@pytest.mark.parametrize("x_t,y_t,a_t", TYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (5, 7), (8, 64), (100, 100), (2056, 1032), (40, 2500), (333, 1024), (4100, 8)])
@pytest.mark.parametrize("m", [3, 70, 270])
def test_odd_sizes(ctx, engine, x_t, y_t, a_t, n, k, m):
    case(ctx, engine, n + k, m, n, k, 3, 9, "rowwise8", x_t, y_t, a_t)


@pytest.mark.parametrize("form", ["rowwise8", "affine8", "affine4"])
@pytest.mark.parametrize("m", [1, 8, 33, 200, 400])
def test_weights(ctx, engine, form, m):
    case(ctx, engine, m, m, 512, 1024, 6, 16, form, "f16", "f16", "f16")


@pytest.mark.parametrize("x_t,y_t,a_t", TYPES)
@pytest.mark.parametrize("m", [7, 90, 300])
@pytest.mark.parametrize("rank", [16, 100, 256])
def test_adapters_of_other_ranks(ctx, engine, x_t, y_t, a_t, m, rank):
    """What lies past an adapter's rank is not read; rank 0 adds nothing."""
    case(ctx, engine, rank, m, 136, 264, 9, rank, "rowwise8", x_t, y_t, a_t, some_ranks=True)


@pytest.mark.parametrize("m", [20, 100, 290])
@pytest.mark.parametrize("kind", ["one", "none", "foreign", "every", "runs"])
def test_ids(ctx, engine, m, kind):
    """One adapter, none, numbers of none (below zero, past the set), a new one each row, runs across tiles."""
    ids = {"one": [3] * m, "none": [-1] * m, "foreign": [[-2 ** 31, 40, 2 ** 31 - 1, 0, 39][t % 5] for t in range(m)],
           "every": [t % 40 for t in range(m)], "runs": [t // 23 for t in range(m)]}[kind]
    case(ctx, engine, m, m, 264, 520, 40, 8, "rowwise8", "f16", "f16", "f16", ids=ids)


@pytest.mark.parametrize("x_t,y_t,a_t", TYPES)
@pytest.mark.parametrize("m", [16, 80, 280])
def test_foreign_adapters_do_not_reach_a_row(ctx, engine, x_t, y_t, a_t, m):
    """Adapters of infinities and NaN: their rows have them, the others' bits are those without them."""
    g = np.random.default_rng(2)
    w, _ = weight(ctx, g, 128, 256, "rowwise8")
    a, b = adapters(g, 3, 8, 256, 128, a_t)
    x = g.standard_normal((m, 256)).astype(KIND[x_t][0])
    ids = g.integers(-1, 3, m)
    f = np.ones(3, np.float32)
    clean = run(ctx, engine, x, w, a, b, f, ids, None, x_t, y_t, a_t)
    a[1], b[1, 3] = np.inf, np.nan
    got = run(ctx, engine, x, w, a, b, f, ids, None, x_t, y_t, a_t)
    other = ids != 1
    assert np.array_equal(got[other], clean[other]) and np.all(np.isnan(got[~other]))
    x[ids == 1] = np.nan  # rows of NaN likewise
    got = run(ctx, engine, x, w, a, b, f, ids, None, x_t, y_t, a_t)
    if not (x_t == "f32" and 2 < m <= 16):  # (the shared product's rows of one tile have a power of two in common there)
        assert np.array_equal(got[other], clean[other])


@pytest.mark.parametrize("x_t,y_t,a_t", TYPES)
@pytest.mark.parametrize("m", [9, 77, 273])
def test_whole_numbers_are_exact(ctx, engine, x_t, y_t, a_t, m):
    """Small whole numbers: every sum is exact, so every value is."""
    g = np.random.default_rng(3)
    n, k, rank, count = 72, 2080, 12, 5
    q = g.integers(-1, 2, (n, k)).astype(np.int8)
    w = QuantizedTensor.rowwise(ctx, q, np.ones(n, np.float32))
    a, b = (g.integers(-1, 2, (count, rank, d)).astype(KIND[a_t][0]) for d in (k, n))
    x = (g.integers(0, 8, (m, k)) == 0).astype(KIND[x_t][0])
    ids = g.integers(-1, count, m)
    want = x.astype(np.float64) @ q.T
    for t, i in enumerate(ids):
        if i >= 0:
            want[t] += 2.0 * ((a[i].astype(np.float64) @ x[t]) @ b[i].astype(np.float64))
    got = run(ctx, engine, x, w, a, b, np.full(count, 2.0, np.float32), ids, None, x_t, y_t, a_t)
    assert np.abs(want).max() < 2048 and np.array_equal(got.astype(np.float64), want)


def test_no_weight_no_reduction(ctx, engine):
    """No factors (all 1), k_in = 0 (zeros), an empty set (the shared product alone), no rows."""
    g = np.random.default_rng(4)
    w, w64 = weight(ctx, g, 64, 128, "rowwise8")
    a, b = adapters(g, 2, 8, 128, 64, "f32")
    x = g.standard_normal((4, 128)).astype(np.float32)
    want, tol = truth(x, w64, a, b, np.ones(2), [0, 1, 1, -1], [8, 8], "f32", False)
    check(run(ctx, engine, x, w, a, b, None, [0, 1, 1, -1], None, "f32", "f32", "f32"), want, tol, "no factors")
    empty = QuantizedTensor.rowwise(ctx, np.zeros((64, 0), np.int8), np.ones(64, np.float32))
    got = run(ctx, engine, np.zeros((4, 0), np.float32), empty, np.zeros((2, 8, 0), np.float32), b, None, [0, 1, 1, -1],
              None, "f32", "f32", "f32")
    assert np.all(got == 0)
    want, tol = truth(x, w64, a[:0], b[:0], [], [0, 1, 1, -1], [], "f16", False)
    check(run(ctx, engine, x, w, np.zeros((0, 8, 128), np.float32), np.zeros((0, 8, 64), np.float32), None, [0, 1, 1, -1],
              None, "f32", "f16", "f32"), want, tol, "empty set")


def test_stack(ctx, engine):
    """Adapters as the reference holds them, of different ranks."""
    g = np.random.default_rng(5)
    w, w64 = weight(ctx, g, 96, 160, "rowwise8")
    pairs = [(g.standard_normal((160, r)).astype(np.float32) * 0.1, g.standard_normal((r, 96)).astype(np.float32)) for r in (4, 16, 7)]
    s = LoraSet.stack(ctx, pairs, factors=[1.0, 0.5, 2.0], dtype=DType.FP32)
    x = g.standard_normal((5, 160)).astype(np.float32)
    ids = np.array([2, 0, 1, -1, 2], np.int32)
    X, out = dev(ctx, x), dev(ctx, np.zeros((5, 96), np.float32))
    engine.qmatmul_loras(ctx, X, w, s, dev(ctx, ids, DType.I32), out)
    a, b = np.zeros((3, 16, 160)), np.zeros((3, 16, 96))
    for i, (p, q) in enumerate(pairs):
        a[i, :p.shape[1]], b[i, :p.shape[1]] = p.T, q
    check(out.to_vec(), *truth(x, w64, a, b, [1.0, 0.5, 2.0], ids, [4, 16, 7], "f32", False), "stack")


def test_graph_and_stream(ctx, engine):
    """Captured on a caller's stream, replayed with other ids, between eager calls."""
    g = np.random.default_rng(6)
    stream = Stream()
    w, w64 = weight(ctx, g, 256, 512, "rowwise8")
    a, b = adapters(g, 4, 16, 512, 256, "f16")
    s = LoraSet(dev(ctx, a), dev(ctx, b))
    for m in (5, 100, 300):
        x = g.standard_normal((m, 512)).astype(np.float16)
        X, I = dev(ctx, x), dev(ctx, np.zeros(m, np.int32), DType.I32)
        outs = [dev(ctx, np.zeros((m, 256), np.float16)) for _ in range(2)]
        works = [engine.qmatmul_loras_workspace(ctx, X, w, s, outs[0]) for _ in range(2)]
        ctx.sync()
        graph = Graph(stream.h, lambda: engine.qmatmul_loras(ctx, X, w, s, I, outs[0], workspace=works[0], stream=stream.h))
        for i in range(4):
            ids = g.integers(-1, 4, m).astype(np.int32)
            call("rq_memcpy_h2d", ctx.handle, I.ptr, ids.ctypes.data, ids.nbytes, None)
            ctx.sync()
            graph.launch()
            stream.synchronize()
            want, tol = truth(x, w64, a, b, np.ones(4), ids, [16] * 4, "f16", False)
            check(outs[0].to_vec(), want, tol, f"replay {i}")
            engine.qmatmul_loras(ctx, X, w, s, I, outs[1], workspace=works[1])
            check(outs[1].to_vec(), want, tol, f"eager {i}")


def test_refusals(ctx, engine):
    g = np.random.default_rng(7)
    w, _ = weight(ctx, g, 64, 128, "rowwise8")
    a, b = adapters(g, 2, 8, 128, 64, "f16")
    A, B = dev(ctx, a), dev(ctx, b)
    X, I, out = dev(ctx, np.zeros((3, 128), np.float16)), dev(ctx, np.zeros(3, np.int32), DType.I32), dev(ctx, np.zeros((3, 64), np.float16))
    s = LoraSet(A, B)
    for bad in (lambda: LoraSet(A, dev(ctx, b.astype(np.float32))), lambda: LoraSet(A, dev(ctx, b[:1])),
                lambda: LoraSet(A, B, factors=dev(ctx, np.zeros(3, np.float32))), lambda: LoraSet(A, B, ranks=I),
                lambda: engine.qmatmul_loras(ctx, X, w, s, dev(ctx, np.zeros(2, np.int32), DType.I32), out),
                lambda: engine.qmatmul_loras(ctx, X, w, LoraSet(B, A), I, out),
                lambda: engine.qmatmul_loras(ctx, X, w, s, I, X)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("m", [4, 300])
@pytest.mark.parametrize("exp", [-60, -20, 14, 40])
def test_large_and_small_products(ctx, engine, m, exp):
    """x . A_i^T far outside fp16's range, and far below it, in rows side by side: f32 adapters and fp16
    ones keep f32 accuracy whatever t's magnitude."""
    g = np.random.default_rng(8)
    k, n, rank, count = 256, 128, 24, 4
    w = QuantizedTensor.rowwise(ctx, np.zeros((n, k), np.int8), np.ones(n, np.float32))
    a, b = adapters(g, count, rank, k, n, "f16")
    f = np.array([1.0, 2.0 ** exp, 2.0 ** (exp // 2), -1.0], np.float32)
    x = g.standard_normal((m, k)).astype(np.float16)
    ids = np.arange(m) % count
    want, tol = truth(x, np.zeros((n, k)), a, b, f, ids, [rank] * count, "f32", False)
    check(run(ctx, engine, x, w, a, b, f, ids, None, "f16", "f32", "f16"), want, tol, f"factors 2^{exp}")


def test_infinite_products(ctx, engine):
    """t beyond f32: the row's results are what plain f32 arithmetic gives, infinite, the others' unchanged."""
    g = np.random.default_rng(9)
    k, n, m = 64, 64, 300
    w = QuantizedTensor.rowwise(ctx, np.zeros((n, k), np.int8), np.ones(n, np.float32))
    a, b = np.ones((2, 8, k), np.float16), np.ones((2, 8, n), np.float16)
    f = np.array([1.0, 3e38], np.float32)
    x = np.full((m, k), 4.0, np.float16)
    ids = np.arange(m) % 2
    for rows in (m, 8):
        got = run(ctx, engine, x[:rows], w, a, b, f, ids[:rows], None, "f16", "f32", "f16")
        assert np.all(got[0::2] == 8 * 256.0) and np.all(got[1::2] == np.inf)


@pytest.mark.parametrize("m", [8, 300])
def test_infinite_beside_large(ctx, engine, m):
    """A t with an infinite entry (one rank's sum is past f32) and entries past fp16's range: columns where the
    infinite entry's B is 1 are infinite, whatever the sign of the finite one's, and no NaN appears."""
    k, n = 64, 64
    w = QuantizedTensor.rowwise(ctx, np.zeros((n, k), np.int8), np.ones(n, np.float32))
    a, b = np.full((1, 2, k), 6e4, np.float16), np.ones((1, 2, n), np.float16)
    a[0, 1], b[0, 1, ::2] = 1e-3, -1.0
    x = np.full((m, k), 1e34, np.float32)  # 1e34 6e4 > 3.4e38 > 64 1e34 1e-3 > 65504
    got = run(ctx, engine, x, w, a, b, None, np.zeros(m, int), None, "f32", "f32", "f16")
    assert np.all(got == np.inf)


@pytest.mark.parametrize("x_t,y_t,a_t", TYPES)
@pytest.mark.parametrize("form", ["rowwise8", "affine8"])
@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("n,k,rank", [(40, 16384, 100), (16400, 64, 256), (131, 2048, 65), (2056, 4160, 16), (7, 1024, 3)])
def test_one_and_two_rows(ctx, engine, x_t, y_t, a_t, form, m, n, k, rank):
    """The decode form: many slices of k, ranks of more than a wave, tall weights, adapters of fewer ranks (0 among them)."""
    g = np.random.default_rng(n)
    for ids in ([0, 2], [1, 1], [-1, 1], [2, 5]):
        case(ctx, engine, n + k + ids[0] + 7, m, n, k, 3, rank, form, x_t, y_t, a_t, ids=ids[:m], some_ranks=bool(g.integers(2)))


def tile(form, m, n, k):
    f = _lib.lib().rusty_gemm_tile
    f.argtypes, f.restype = [ctypes.c_int] + [ctypes.c_int64] * 3 + [ctypes.c_int] * 2, ctypes.c_int
    return f(int(form != "rowwise8"), m, n, k, 256, 2)


@pytest.mark.parametrize("x_t,y_t", [("f16", "f16"), ("f32", "f32"), ("f16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("form,m,n,k,rank,want", [("rowwise8", 1100, 5640, 192, 32, 128256), ("rowwise8", 515, 10264, 64, 70, 128256),
                                                  ("affine8", 900, 6152, 192, 21, 128256), ("affine8", 700, 3712, 128, 40, 128128),
                                                  ("rowwise8", 1024, 4096, 1024, 16, 128128)])
def test_in_the_products_tiles(ctx, engine, form, m, n, k, rank, want, x_t, y_t):
    """Where the shared product takes tiles of 128 rows and 8 waves, its kernel adds the adapters: prompts of one adapter
    behind another, and every row another one, with ranks that differ."""
    assert tile(form, m, n, k) == want
    g = np.random.default_rng(m)
    prompts = np.repeat(g.integers(-1, 5, m // 90 + 1), 90)[:m]
    case(ctx, engine, m, m, n, k, 5, rank, form, x_t, y_t, "f16", ids=prompts)
    case(ctx, engine, m + 1, m, n, k, 5, rank, form, x_t, y_t, "f16", ids=g.integers(-1, 6, m), some_ranks=True)


def test_in_the_products_tiles_not_finite(ctx, engine):
    """Adapters that hold infinities and NaN, in the same tiles as rows of others: those rows are as without them."""
    g = np.random.default_rng(16)
    m, n, k = 1100, 5640, 192
    w, w64 = weight(ctx, g, n, k, "rowwise8")
    a, b = adapters(g, 4, 40, k, n, "f16")
    a[1], b[1], b[2, :, ::3], b[3, 33] = np.nan, np.inf, np.inf, np.nan
    x = g.standard_normal((m, k)).astype(np.float16)
    ids = g.integers(-1, 4, m)
    want, tol = truth(x, w64, a[:1], b[:1], np.ones(4), np.where(ids == 0, 0, -1), [40], "f16", False)
    got = run(ctx, engine, x, w, a, b, None, ids, [40, 40, 40, 33], "f16", "f16", "f16")
    own = (ids == 0) | (ids == -1)
    check(got[own], want[own], tol[own], "rows beside")
    assert not np.isfinite(got[ids == 1]).any() and not np.isfinite(got[ids == 2][:, ::3]).any()
    assert np.isfinite(got[ids == 3]).all()


@pytest.mark.parametrize("x_t,y_t", [("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("form,m,n,k,rank,want", [("rowwise8", 1100, 5640, 192, 32, 128256), ("affine8", 700, 3712, 128, 90, 128128)])
@pytest.mark.parametrize("count", [8, 16, 17, 60])
def test_in_the_products_tiles_many_adapters(ctx, engine, form, m, n, k, rank, want, count, x_t, y_t):
    """More adapters in a tile's rows than are taken one after another."""
    assert tile(form, m, n, k) == want
    g = np.random.default_rng(count)
    case(ctx, engine, m, m, n, k, count, rank, form, x_t, y_t, "f16", ids=g.integers(-1, count, m), some_ranks=count == 60)


def test_tiles_that_add_adapters():
    """Where the product's tiles add the adapters, and where they are added in a pass of their own."""
    assert [tile("rowwise8", m, n, 4096) for m, n in ((2048, 4096), (1024, 4096), (1293, 4096))] == [128256, 128128, 128256]
    assert [tile("rowwise8", m, n, 4096) for m, n in ((300, 4096), (512, 4096), (777, 11008))] == [-1, -1, -1]


@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (2, 256, 512), (1100, 5640, 192)])
@pytest.mark.parametrize("own", [True, False])
def test_graph_of_two_launches(ctx, engine, m, n, k, own):
    """The forms in which the product's kernel adds the adapters, captured on the context's stream or another, replayed with
    other ids between eager calls."""
    g = np.random.default_rng(m)
    other = Stream()
    stream = ctx.stream if own else other.h
    w, w64 = weight(ctx, g, n, k, "rowwise8")
    a, b = adapters(g, 4, 16, k, n, "f16")
    s = LoraSet(dev(ctx, a), dev(ctx, b))
    x = g.standard_normal((m, k)).astype(np.float16)
    X, I = dev(ctx, x), dev(ctx, np.zeros(m, np.int32), DType.I32)
    outs = [dev(ctx, np.zeros((m, n), np.float16)) for _ in range(2)]
    works = [engine.qmatmul_loras_workspace(ctx, X, w, s, outs[0]) for _ in range(2)]
    ctx.sync()
    graph = Graph(stream, lambda: engine.qmatmul_loras(ctx, X, w, s, I, outs[0], workspace=works[0],
                                                       stream=None if own else stream))
    for i in range(3):
        ids = g.integers(-1, 4, m).astype(np.int32)
        call("rq_memcpy_h2d", ctx.handle, I.ptr, ids.ctypes.data, ids.nbytes, None)
        ctx.sync()
        graph.launch()
        if not own:
            other.synchronize()
        want, tol = truth(x, w64, a, b, np.ones(4), ids, [16] * 4, "f16", False)
        check(outs[0].to_vec(), want, tol, f"replay {i}")
        engine.qmatmul_loras(ctx, X, w, s, I, outs[1], workspace=works[1])
        assert np.array_equal(outs[1].to_vec(), outs[0].to_vec())


@pytest.mark.parametrize("m,n,k", [(1, 128, 256), (2, 128, 256), (1100, 5640, 192)])
@pytest.mark.parametrize("exp", [-60, -20, 14, 40])
def test_large_and_small_products_of_two_launches(ctx, engine, m, n, k, exp):
    """t far outside fp16's range, and far below it, in rows side by side."""
    g = np.random.default_rng(18)
    rank, count = 40, 4
    w = QuantizedTensor.rowwise(ctx, np.zeros((n, k), np.int8), np.ones(n, np.float32))
    a, b = adapters(g, count, rank, k, n, "f16")
    f = np.array([2.0 ** exp, 1.0, 2.0 ** (exp // 2), -1.0], np.float32)
    x = g.standard_normal((m, k)).astype(np.float16)
    ids = np.arange(m) % count
    want, tol = truth(x, np.zeros((n, k)), a, b, f, ids, [rank] * count, "f32", False)
    check(run(ctx, engine, x, w, a, b, f, ids, None, "f16", "f32", "f16"), want, tol, f"factors 2^{exp}")


@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (2, 64, 64), (1100, 5640, 64)])
def test_infinite_beside_large_of_two_launches(ctx, engine, m, n, k):
    w = QuantizedTensor.rowwise(ctx, np.zeros((n, k), np.int8), np.ones(n, np.float32))
    a, b = np.full((2, 2, k), 6e4, np.float16), np.ones((2, 2, n), np.float16)
    a[0, 1], b[0, 1, ::2] = 1e-3, -1.0
    a[1] = 1e-30  # (zero in fp16)
    x = np.full((m, k), 1e34, np.float32)
    ids = np.arange(m) % 2
    got = run(ctx, engine, x, w, a, b, None, ids, None, "f32", "f32", "f16")
    assert np.all(got[0::2] == np.inf) and np.all(got[1::2] == 0.0)


def test_one_row_off_its_alignment(ctx, engine):
    """Activations and results in whatever place their elements allow: the decode form is left for others."""
    g = np.random.default_rng(19)
    w, w64 = weight(ctx, g, 72, 128, "rowwise8")
    a, b = adapters(g, 2, 8, 128, 72, "f16")
    s = LoraSet(dev(ctx, a), dev(ctx, b))
    x = g.standard_normal((2, 128)).astype(np.float16)
    held, out = dev(ctx, np.concatenate([np.zeros(1, np.float16), x.ravel()])), dev(ctx, np.zeros(145, np.float16))
    X, Y = UnifiedTensor(ctx, held.ptr + 2, (2, 128), DType.FP16, owner=False), UnifiedTensor(ctx, out.ptr + 2, (2, 72), DType.FP16, owner=False)
    engine.qmatmul_loras(ctx, X, w, s, dev(ctx, np.array([1, 0], np.int32), DType.I32), Y)
    got = out.to_vec()
    check(got[1:].reshape(2, 72), *truth(x, w64, a, b, np.ones(2), [1, 0], [8, 8], "f16", False), "off alignment")
    assert got[0] == 0.0


@pytest.mark.parametrize("x_t,y_t,a_t", TYPES)
@pytest.mark.parametrize("m", [200, 270])
@pytest.mark.parametrize("n,k,rank", [(7, 130, 33), (5001, 130, 100), (130, 131, 256), (518, 260, 17)])
def test_widths_that_pieces_do_not_divide(ctx, engine, x_t, y_t, a_t, m, n, k, rank):
    """Rows of B and Y that begin anywhere, several steps of ranks, adapters of fewer ranks."""
    case(ctx, engine, n, m, n, k, 3, rank, "rowwise8", x_t, y_t, a_t, some_ranks=True)
