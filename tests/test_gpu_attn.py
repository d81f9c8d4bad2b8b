"""rq_attn_packed and rq_attn_tree against a plain computation in 64 bits.

Tolerance, per output value o = sum_j p_j v_j / l (p_j = exp(s_j - max), l =
sum p_j >= 1, A = sum_j p_j |v_j| / l, n keys, u = 2^-24):
  * a score is a sum of at most head_dim + 2 rounded terms, then scaled and
    shifted by the maximum: its error is at most
    e = (dim + 4) u |scale| sum|q||k| + 4 u (|s| + |max|), and the exponential
    adds 2^-21 relative.  Numerator and denominator each move by that;
  * sums over n keys in f32, rescaled now and then: (2 n + 32) u each;
  * fp16: p is rounded to fp16, half a step 2^-11 relative, below 2^-14 at most
    2^-25 absolute: 2^-11 A + n 2^-25 max|v| / l;
  * the output's own rounding, half a step: 2^-11 |o| (fp16; at least 2^-25), u |o| (f32).
"""
import numpy as np
import pytest

from rusty_amd import DType, UnifiedTensor
from rusty_amd.hiprt import Graph, Stream

pytestmark = pytest.mark.gpu

KIND = {"f16": (np.float16, DType.FP16), "f32": (np.float32, DType.FP32)}
U = 2.0 ** -24


def attend(q, k, v, keep, scale, f16):
    """(o, tolerance) in 64 bits: q [rows, dim], k, v [keys, dim], keep [rows, keys]."""
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    dim, n = q.shape[1], k.shape[0]
    o, tol = np.zeros_like(q), np.full(q.shape, 2.0 ** -25 if f16 else 2.0 ** -140)
    for r in range(q.shape[0]):
        c = np.nonzero(keep[r])[0]
        if not c.size:
            tol[r] = 0.0
            continue
        s = k[c] @ q[r] * scale
        top = s.max()
        p = np.exp(s - top)
        l, av = p.sum(), np.abs(v[c])
        o[r], A = p @ v[c] / l, p @ av / l
        e = (dim + 4) * U * abs(scale) * (np.abs(k[c]) @ np.abs(q[r])).max() + 4 * U * (np.abs(s).max() + abs(top))
        rel = 2 * np.expm1(e + 2.0 ** -21) + 2 * (2 * n + 32) * U
        tol[r] += rel * A + (2.0 ** -11 if f16 else U) * np.abs(o[r])
        if f16:
            tol[r] += 2.0 ** -11 * A + n * 2.0 ** -25 * av.max(0) / l
    return o, tol


def check(got, want, tol, what):
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    worst = np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300)) if got.size else 0.0
    print(f"[{what}] worst {worst:.3f} of the tolerance", flush=True)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} values outside, first at {np.argwhere(bad)[0]}"


# ---- packed prompts ------------------------------------------------------------------


def packed_inputs(seed, total, heads, kv, dim, dtype, std=1.0):
    g = np.random.default_rng(seed)
    t = KIND[dtype][0]
    return [(g.standard_normal((total, n, dim)) * std).astype(t) for n in (heads, kv, kv)]


def packed_truth(q, k, v, starts, scale, f16):
    heads, kv = q.shape[1], k.shape[1]
    o, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for a, b in zip(starts[:-1], starts[1:]):
        keep = np.tril(np.ones((b - a, b - a), bool))
        for h in range(heads):
            g = h // (heads // kv)
            o[a:b, h], tol[a:b, h] = attend(q[a:b, h], k[a:b, g], v[a:b, g], keep, scale, f16)
    return o, tol


def run_packed(ctx, engine, q, k, v, starts, dtype, fill=7.0, **kw):
    T = lambda a, d: UnifiedTensor.new(ctx, a, dtype=d)  # noqa: E731
    kind = KIND[dtype][1]
    out = T(np.full(q.shape, fill), kind)
    engine.attn_packed(ctx, T(q, kind), T(k, kind), T(v, kind), T(np.asarray(starts, np.int32), DType.I32), out, **kw)
    return out.to_vec()


LENGTHS = {"one": [1], "empties": [0, 1, 0, 0, 3, 0], "edges": [31, 32, 33, 1, 63, 64, 65], "tiles": [129, 128, 127],
           "long": [257, 5], "longer": [700]}


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 1, 64), (6, 2, 128), (5, 1, 128)])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_packed(ctx, engine, dtype, heads, kv, dim, lengths):
    starts = np.concatenate([[0], np.cumsum(LENGTHS[lengths])])
    q, k, v = packed_inputs(1 + len(lengths) + heads, int(starts[-1]), heads, kv, dim, dtype)
    want, tol = packed_truth(q, k, v, starts, 1 / np.sqrt(dim), dtype == "f16")
    got = run_packed(ctx, engine, q, k, v, starts, dtype)
    check(got, want, tol, f"packed {lengths} {heads}/{kv}x{dim} {dtype}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_packed_rows_of_no_sequence_stay(ctx, engine, dtype):
    """Rows before the first start and behind the last one are left as they
    were, and starts outside the tokens are clamped."""
    q, k, v = packed_inputs(3, 90, 4, 2, 64, dtype)
    starts = np.array([9, 40, 40, 77])
    got = run_packed(ctx, engine, q, k, v, starts, dtype)
    assert np.all(got[:9] == 7.0) and np.all(got[77:] == 7.0)
    want, tol = packed_truth(q, k, v, starts, 1 / 8, dtype == "f16")
    check(got[9:77], want[9:77], tol[9:77], "inner rows")
    clamped = run_packed(ctx, engine, q, k, v, [-5, 40, 1000], dtype)
    want, tol = packed_truth(q, k, v, [0, 40, 90], 1 / 8, dtype == "f16")
    check(clamped, want, tol, "clamped starts")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
def test_packed_fused_rows(ctx, engine, dtype, dim):
    """q, k and v read in place from the rows of one fused product, out
    written into wider rows whose other columns stay."""
    heads, kv, total = 6, 2, 150
    starts = [0, 70, 71, 150]
    q, k, v = packed_inputs(4, total, heads, kv, dim, dtype)
    row = (heads + 2 * kv) * dim
    kind = KIND[dtype]
    qkv = UnifiedTensor.new(ctx, np.concatenate([q, k, v], 1).reshape(total, row), dtype=kind[1])
    at = lambda n, shape: UnifiedTensor(ctx, qkv.ptr + n * dim * kind[1].itemsize, shape, kind[1], owner=False)  # noqa: E731
    out = UnifiedTensor.new(ctx, np.full((total, heads + 1, dim), 7.0), dtype=kind[1])
    view = UnifiedTensor(ctx, out.ptr, q.shape, kind[1], owner=False)
    engine.attn_packed(ctx, at(0, q.shape), at(heads, k.shape), at(heads + kv, v.shape),
                       UnifiedTensor.new(ctx, np.array(starts, np.int32), dtype=DType.I32), view, q_row=row, k_row=row,
                       v_row=row, out_row=(heads + 1) * dim)
    got = out.to_vec()
    assert np.all(got[:, heads] == 7.0)
    want, tol = packed_truth(q, k, v, starts, dim ** -0.5, dtype == "f16")
    check(got[:, :heads], want, tol, f"fused {dim} {dtype}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_packed_nonfinite_keys_stay_hidden(ctx, engine, dtype, dim, bad):
    """A key or value that is not finite reaches the tokens that see it, and no
    other: neither earlier tokens nor other sequences."""
    starts = [0, 40, 110, 150]
    q, k, v = packed_inputs(5, 150, 4, 2, dim, dtype)
    want, tol = packed_truth(q, k, v, starts, dim ** -0.5, dtype == "f16")
    k[75, 0], v[77, 1, 3], v[100, 1, 5], v[39, 0, :] = bad, bad, bad, bad
    got = run_packed(ctx, engine, q, k, v, starts, dtype)
    hit = np.zeros(got.shape, bool)
    hit[75:110, 0:2] = True       # scores against k[75]
    hit[77:110, 2:4, 3] = True    # the value's own dimension
    hit[100:110, 2:4, 5] = True
    hit[39, 0:2] = True
    check(np.where(hit, 0, got), np.where(hit, 0, want), np.where(hit, 1, tol), f"hidden {bad} {dim} {dtype}")
    assert not np.isfinite(got[39, 0:2].astype(np.float64)).any()
    for d in (3, 5):
        assert not np.isfinite(got[100:110, 2:4, d].astype(np.float64)).any()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("std,scale", [(8.0, None), (1.0, -0.3), (0.02, 1.0), (1.0, 1e-6)])
def test_packed_scales(ctx, engine, dtype, std, scale):
    """Sharp and flat softmaxes, a negative scale."""
    starts = [0, 200, 233]
    q, k, v = packed_inputs(6, 233, 2, 1, 64, dtype, std)
    want, tol = packed_truth(q, k, v, starts, 1 / 8 if scale is None else np.float64(np.float32(scale)), dtype == "f16")
    check(run_packed(ctx, engine, q, k, v, starts, dtype, scale=scale), want, tol, f"std {std} scale {scale} {dtype}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_packed_streams_and_graphs(ctx, engine, dtype):
    """The same bits on a stream of the caller's and from a captured call
    replayed with other inputs between eager calls."""
    starts = [0, 33, 160]
    q, k, v = packed_inputs(7, 160, 4, 2, 64, dtype)
    kind = KIND[dtype][1]
    T = lambda a, d=kind: UnifiedTensor.new(ctx, a, dtype=d)  # noqa: E731
    Q, K, V, S = T(q), T(k), T(v), T(np.array(starts, np.int32), DType.I32)
    one, two = T(np.zeros(q.shape)), T(np.zeros(q.shape))
    engine.attn_packed(ctx, Q, K, V, S, one)
    ref = one.to_vec()
    st = Stream()
    ctx.sync()
    engine.attn_packed(ctx, Q, K, V, S, two, stream=st.h)
    st.synchronize()
    assert np.array_equal(two.to_vec(), ref)
    graph = Graph(ctx.stream, lambda: engine.attn_packed(ctx, Q, K, V, S, two))
    for i in range(4):
        Q2 = T(packed_inputs(20 + i, 160, 4, 2, 64, dtype)[0])
        from rusty_amd import _lib
        _lib.call("rq_memcpy_d2d", ctx.handle, Q.ptr, Q2.ptr, Q.nbytes, None)
        two.zero_()
        graph.launch()
        got = two.to_vec()
        engine.attn_packed(ctx, Q, K, V, S, one)
        assert np.array_equal(got, one.to_vec()) and not np.array_equal(got, ref)


# ---- drafted trees over a cache ----------------------------------------------------------


def tree_masks(g, nodes):
    rows = []
    for n in nodes:
        m = []
        for i in range(n):
            parent = int(g.integers(-1, i)) if i else -1
            m.append((m[parent] if parent >= 0 else 0) | 1 << i)
        rows += m
    return np.array(rows, dtype=np.uint64)


def tree_inputs(seed, lengths, nodes, capacity, heads, kv, dim, dtype):
    g = np.random.default_rng(seed)
    t = KIND[dtype][0]
    q = g.standard_normal((sum(nodes), heads, dim)).astype(t)
    k, v = (g.standard_normal((len(lengths), kv, capacity, dim)).astype(t) for _ in range(2))
    return q, k, v, tree_masks(g, nodes)


def tree_truth(q, k, v, lengths, nodes, mask, scale, f16):
    heads, kv, cap = q.shape[1], k.shape[1], k.shape[2]
    o, tol, first = np.zeros(q.shape), np.zeros(q.shape), 0
    for s, (length, n) in enumerate(zip(lengths, nodes)):
        end = min(length + n, cap)
        keep = np.zeros((n, end), bool)
        keep[:, :length] = True
        for i in range(n):
            bits = int(mask[first + i]) if mask is not None else (2 << i) - 1
            for j in range(min(n, end - length)):
                keep[i, length + j] = bits >> j & 1
        for h in range(heads):
            g = h // (heads // kv)
            o[first:first + n, h], tol[first:first + n, h] = attend(q[first:first + n, h], k[s, g, :end], v[s, g, :end],
                                                                    keep, scale, f16)
        first += n
    return o, tol


def run_tree(ctx, engine, q, k, v, lengths, nodes, mask, dtype, max_nodes=None, tokens=None, starts=None, **kw):
    kind = KIND[dtype][1]
    T = lambda a, d=kind: UnifiedTensor.new(ctx, a, dtype=d)  # noqa: E731
    starts = np.concatenate([[0], np.cumsum(nodes)]) if starts is None else starts
    out = T(np.full(q.shape, 7.0))
    engine.attn_tree(ctx, T(q), T(k), T(v), T(np.asarray(starts, np.int32), DType.I32),
                     T(np.asarray(lengths, np.int32), DType.I32), None if mask is None else T(mask, DType.U64), out,
                     max_nodes or max(nodes), **kw)
    return out.to_vec()


TREES = {  # lengths, nodes, capacity
    "one": ([0], [1], 4), "first": ([5], [1], 6), "step": ([512], [1], 640), "steps": ([0, 31, 32, 33, 200], [1] * 5, 256),
    "chats": ([61, 0, 127, 300], [16, 3, 1, 13], 320), "wide": ([97, 500], [64, 33], 600), "long": ([2300], [5], 2400),
    "empty": ([10, 7, 90], [0, 4, 0], 100), "full": ([60], [4], 64),
}


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 1, 64), (6, 2, 128), (5, 1, 128)])
@pytest.mark.parametrize("name", list(TREES))
def test_tree(ctx, engine, dtype, heads, kv, dim, name):
    lengths, nodes, cap = TREES[name]
    q, k, v, mask = tree_inputs(11 + heads, lengths, nodes, cap, heads, kv, dim, dtype)
    for m in (mask, None):
        want, tol = tree_truth(q, k, v, lengths, nodes, m, dim ** -0.5, dtype == "f16")
        got = run_tree(ctx, engine, q, k, v, lengths, nodes, m, dtype)
        check(got, want, tol, f"tree {name} {heads}/{kv}x{dim} {dtype} {'chain' if m is None else ''}")


# Few and many sequences, rows and keys: each way in which a call's rows and keys are cut into blocks.
CUTS = {  # sequences, capacity, most nodes of one, heads, key/value heads, dim
    "many row tiles": (260, 30, 8, 34, 2, 64), "row tiles": (70, 150, 10, 32, 4, 64), "many small": (130, 40, 9, 16, 4, 64),
    "half tiles": (33, 300, 20, 16, 4, 128), "half tiles, fewer": (9, 230, 33, 32, 4, 64),
    "pieces": (3, 1000, 20, 8, 2, 128), "pieces of tiles": (5, 1700, 64, 16, 8, 128), "one long": (1, 20000, 40, 4, 1, 64),
}


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("name", list(CUTS))
def test_tree_cuts(ctx, engine, dtype, name):
    seqs, cap, most, heads, kv, dim = CUTS[name]
    g = np.random.default_rng(31)
    nodes = [most] + [int(x) for x in g.integers(0, most + 1, seqs - 1)]
    lengths = [cap - most] + [int(x) for x in g.integers(0, cap - most + 1, seqs - 1)]
    q, k, v, mask = tree_inputs(30, lengths, nodes, cap, heads, kv, dim, dtype)
    want, tol = tree_truth(q, k, v, lengths, nodes, mask, dim ** -0.5, dtype == "f16")
    check(run_tree(ctx, engine, q, k, v, lengths, nodes, mask, dtype), want, tol, f"tree {name} {dtype}")


# With q = 0 every weight is 1, and whole values below 9 have exact sums: a result is a
# mean with one rounding of 1 / l, one of the product and the output's own, so a key
# lost or taken twice among thousands shows.
def check_means(got, sums, counts, f16, what):
    want = sums / np.maximum(counts, 1)
    check(got, want, ((2.0 ** -11 if f16 else U) + 3 * U) * np.abs(want) + (2.0 ** -25 if f16 else 0.0), what)


RAGGED = [int(x) for x in np.random.default_rng(5).integers(0, 60, 65)]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 64), (4, 2, 128), (32, 4, 64), (24, 3, 128)])
@pytest.mark.parametrize("lengths", [[1], [5, 0, 70, 1], [1000, 3], [129] * 9, [2500], [300, 290], RAGGED[:64], RAGGED,
                                     [0, 700, 1, 300, 0, 530, 64], [1, 2, 1500]], ids=lambda v: str(v[:7]))
def test_packed_takes_every_key_once(ctx, engine, dtype, heads, kv, dim, lengths):
    starts = np.concatenate([[0], np.cumsum(lengths)])
    q, k, v = packed_inputs(3, int(starts[-1]), heads, kv, dim, dtype)
    v = np.random.default_rng(4).integers(-8, 9, v.shape).astype(v.dtype)
    got = run_packed(ctx, engine, 0 * q, k, v, starts, dtype)
    sums = np.concatenate([np.cumsum(v[a:b].astype(np.float64), 0) for a, b in zip(starts, starts[1:])])
    counts = np.concatenate([np.arange(1, n + 1) for n in lengths])[:, None, None]
    check_means(got, np.repeat(sums, heads // kv, 1), counts, dtype == "f16", f"means {lengths[:3]} {dtype}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("name", list(CUTS))
def test_tree_takes_every_key_once(ctx, engine, dtype, name):
    seqs, cap, most, heads, kv, dim = CUTS[name]
    g = np.random.default_rng(41)
    nodes = [most] + [int(x) for x in g.integers(0, most + 1, seqs - 1)]
    lengths = [cap - most] + [int(x) for x in g.integers(0, cap - most + 1, seqs - 1)]
    q, k, v, mask = tree_inputs(42, lengths, nodes, cap, heads, kv, dim, dtype)
    v = g.integers(-8, 9, v.shape).astype(v.dtype)
    got = run_tree(ctx, engine, 0 * q, k, v, lengths, nodes, mask, dtype)
    sums, counts, t = np.zeros(q.shape), np.zeros((len(q), 1, 1)), 0
    for s, (length, n) in enumerate(zip(lengths, nodes)):
        cached = v[s, :, :length].sum(1, dtype=np.float64)
        for i in range(n):
            seen = [j for j in range(n) if int(mask[t]) >> j & 1]
            sums[t] = np.repeat(cached + v[s][:, [length + j for j in seen]].sum(1, dtype=np.float64), heads // kv, 0)
            counts[t] = length + len(seen)
            t += 1
    check_means(got, sums, counts, dtype == "f16", f"means {name} {dtype}")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_tree_masks_that_leave_nothing(ctx, engine, dtype):
    """No cached position and no set bit: zeros.  Bits past the sequence's
    tokens, or past the capacity, name nothing."""
    lengths, nodes, cap = [0, 0, 30, 62], [3, 2, 2, 4], 64
    q, k, v, _ = tree_inputs(12, lengths, nodes, cap, 4, 2, 64, dtype)
    k[3, :, 63], v[3, :, 63] = np.nan, np.nan  # not named by the masks that reach it
    mask = np.array([0, 1 << 63 | 1 << 3, 1, 0, 2, 0, 1 << 40, 1, 1 << 2, 1 << 3, 0], np.uint64)
    want, tol = tree_truth(q, k, v, lengths, nodes, mask, 1 / 8, dtype == "f16")
    got = run_tree(ctx, engine, q, k, v, lengths, nodes, mask, dtype)
    check(got, want, tol, "empty masks")
    assert np.all(got[[0, 1, 3]] == 0) and np.isfinite(got.astype(np.float64)).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_tree_stale_rows_and_hidden_nodes(ctx, engine, dtype, dim, bad):
    """Cache rows past the drafted tokens, and drafted tokens a node does not
    see, may hold anything."""
    lengths, nodes, cap = [45, 3, 200], [6, 40, 2], 256
    q, k, v, mask = tree_inputs(13, lengths, nodes, cap, 4, 2, dim, dtype)
    mask[:6] = [1, 3, 5, 9, 17, 33]  # node 0, its five children
    mask[6:46] = [1 << i for i in range(40)]
    want, tol = tree_truth(q, k, v, lengths, nodes, mask, dim ** -0.5, dtype == "f16")
    for s, (a, n) in enumerate(zip(lengths, nodes)):
        k[s, :, a + n:], v[s, :, a + n:] = bad, bad
    k[0, :, 45 + 3], v[0, :, 45 + 4, 1], v[1, :, 3 + 17] = bad, bad, bad
    got = run_tree(ctx, engine, q, k, v, lengths, nodes, mask, dtype)
    hit = np.zeros(got.shape, bool)
    hit[3], hit[4, :, 1], hit[6 + 17] = True, True, True
    check(np.where(hit, 0, got), np.where(hit, 0, want), np.where(hit, 1, tol), f"hidden nodes {bad} {dim} {dtype}")
    assert not np.isfinite(got[6 + 17].astype(np.float64)).any()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_tree_clamps_and_untouched_rows(ctx, engine, dtype):
    """Lengths outside 0..capacity are clamped; rows past max_nodes of a
    sequence and behind the last one stay as they were."""
    lengths, nodes, cap = [-4, 900, 20], [3, 3, 9], 64
    q, k, v, mask = tree_inputs(14, lengths, nodes, cap, 4, 2, 64, dtype)
    more = np.concatenate([q, q[:5]])
    got = run_tree(ctx, engine, more, k, v, lengths, nodes, np.concatenate([mask, mask[:5]]), dtype, max_nodes=4,
                   starts=[0, 3, 6, 15])
    want, tol = tree_truth(q, k, v, [0, 64, 20], [3, 3, 9], mask & np.uint64(0xFFFF), 1 / 8, dtype == "f16")
    lim = mask.copy()
    lim[6:] &= np.uint64(15)  # tokens past max_nodes are not there
    want, tol = tree_truth(q, k, v, [0, 64, 20], [3, 3, 9], lim, 1 / 8, dtype == "f16")
    check(got[:10], want[:10], tol[:10], "clamped lengths")
    assert np.all(got[10:] == 7.0)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
def test_tree_cache_layouts(ctx, engine, dtype, dim):
    """[n_seqs, capacity, n_kv, dim] caches and strided q and out rows give the
    same bits as the default layout."""
    lengths, nodes, cap, heads, kv = [100, 3, 260], [7, 2, 12], 288, 6, 2
    q, k, v, mask = tree_inputs(15, lengths, nodes, cap, heads, kv, dim, dtype)
    ref = run_tree(ctx, engine, q, k, v, lengths, nodes, mask, dtype)
    kind = KIND[dtype][1]
    T = lambda a, d=kind: UnifiedTensor.new(ctx, np.ascontiguousarray(a), dtype=d)  # noqa: E731
    kt, vt = T(k.transpose(0, 2, 1, 3)).reshaped(k.shape), T(v.transpose(0, 2, 1, 3)).reshaped(v.shape)
    wide = T(np.concatenate([q, q[:, :2] * 0], 1))
    out = T(np.full((sum(nodes), heads + 1, dim), 7.0))
    see = lambda t: UnifiedTensor(ctx, t.ptr, q.shape, kind, owner=False)  # noqa: E731
    engine.attn_tree(ctx, see(wide), kt, vt, T(np.array([0, 7, 9, 21], np.int32), DType.I32),
                     T(np.array(lengths, np.int32), DType.I32), T(mask, DType.U64), see(out), 12,
                     q_row=(heads + 2) * dim, out_row=(heads + 1) * dim, strides=(cap * kv * dim, dim, kv * dim))
    got = out.to_vec()
    assert np.array_equal(got[:, :heads], ref) and np.all(got[:, heads] == 7.0)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_tree_streams_and_graphs(ctx, engine, dtype):
    """The same bits on a caller's stream, from a second call that shares the
    workspace after it, and from a captured call whose lengths change between
    replays."""
    lengths, nodes, cap = [700, 50], [5, 9], 1024
    q, k, v, mask = tree_inputs(16, lengths, nodes, cap, 8, 2, 64, dtype)
    kind = KIND[dtype][1]
    T = lambda a, d=kind: UnifiedTensor.new(ctx, a, dtype=d)  # noqa: E731
    Q, K, V, M = T(q), T(k), T(v), T(mask, DType.U64)
    S, L = T(np.array([0, 5, 14], np.int32), DType.I32), T(np.array(lengths, np.int32), DType.I32)
    one, two = T(np.zeros(q.shape)), T(np.zeros(q.shape))
    W = engine.attn_tree_workspace(ctx, Q, K, 9)
    W2 = engine.attn_tree_workspace(ctx, Q, K, 9)
    engine.attn_tree(ctx, Q, K, V, S, L, M, one, 9, workspace=W)
    ref = one.to_vec()
    st = Stream()
    ctx.sync()
    engine.attn_tree(ctx, Q, K, V, S, L, M, two, 9, workspace=W2, stream=st.h)
    st.synchronize()
    assert np.array_equal(two.to_vec(), ref)
    graph = Graph(ctx.stream, lambda: engine.attn_tree(ctx, Q, K, V, S, L, M, two, 9, workspace=W2))
    from rusty_amd import _lib
    for now in ([700, 50], [0, 1015], [33, 0], [1, 64]):
        L2 = T(np.array(now, np.int32), DType.I32)
        _lib.call("rq_memcpy_d2d", ctx.handle, L.ptr, L2.ptr, L.nbytes, None)
        two.zero_()
        graph.launch()
        got = two.to_vec()
        engine.attn_tree(ctx, Q, K, V, S, L, M, one, 9, workspace=W)
        assert np.array_equal(got, one.to_vec())
        want, tol = tree_truth(q, k, v, now, nodes, mask, 1 / 8, dtype == "f16")
        check(got, want, tol, f"replay {now} {dtype}")


def test_tree_follows_packed(ctx, engine):
    """Prompts through rq_attn_packed, their keys copied into a cache, then one
    more token each through rq_attn_tree: what rq_attn_packed gives for the
    prompts with that token."""
    heads, kv, dim, lengths = 8, 2, 64, [37, 1, 130]
    full = [n + 1 for n in lengths]
    starts = np.concatenate([[0], np.cumsum(full)])
    q, k, v = packed_inputs(17, int(starts[-1]), heads, kv, dim, "f16")
    want, tol = packed_truth(q, k, v, starts, 1 / 8, True)
    both = run_packed(ctx, engine, q, k, v, starts, "f16")
    cap = 136
    kc, vc = np.zeros((3, kv, cap, dim), np.float16), np.zeros((3, kv, cap, dim), np.float16)
    for s, a in enumerate(starts[:-1]):
        kc[s, :, :full[s]] = k[a:a + full[s]].transpose(1, 0, 2)
        vc[s, :, :full[s]] = v[a:a + full[s]].transpose(1, 0, 2)
    last = starts[1:] - 1
    step = run_tree(ctx, engine, q[last], kc, vc, lengths, [1, 1, 1], None, "f16")
    check(both[last], want[last], tol[last], "packed")
    check(step, want[last], tol[last], "tree")
