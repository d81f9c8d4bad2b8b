"""rq_attn_paged in fp16 carries its weights in two fp16 terms, at 2^8 of their place below the
running maximum: a weight p (of 1 for the largest key) is off by at most 2^-22 p + 2^-33.
Tolerance: as in test_gpu_attn.py, with that in the place of one fp16 rounding of each weight:
2^-22 A + n 2^-33 max|v| / l, A = sum p |v| / l."""
import numpy as np
import pytest

from test_gpu_attn import attend, check
from test_gpu_paged import make, run

pytestmark = pytest.mark.gpu


def truth(q, rows, scale):
    o, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s, (k, v) in enumerate(rows):
        n, grp = k.shape[1], q.shape[1] // k.shape[0]
        for g in range(k.shape[0]):
            h = slice(g * grp, (g + 1) * grp)
            if not n:
                continue
            o[s, h], tol[s, h] = attend(q[s, h], k[g], v[g], np.ones((grp, n), bool), scale, False)
            x = k[g].astype(np.float64) @ q[s, h].astype(np.float64).T * scale
            p = np.exp(x - x.max(0))
            l, av = p.sum(0)[:, None], np.abs(v[g].astype(np.float64))
            tol[s, h] += 2.0 ** -22 * (p.T @ av) / l + n * 2.0 ** -33 * av.max(0) / l
    return o, tol + np.maximum(2.0 ** -11 * np.abs(o), 2.0 ** -25)


def put(pools, places, order, page, k, v):
    for pool, r in zip(pools, (k, v)):
        pool = pool if order == "heads" else pool.transpose(0, 2, 1, 3)
        for p in range(r.shape[1]):
            pool[places[p // page], :, p % page] = r[:, p]


@pytest.mark.parametrize("heads,kv,dim,page,order", [(4, 2, 64, 16, "heads"), (5, 1, 128, 64, "positions"), (6, 6, 128, 4, "heads")])
def test_values_that_cancel(ctx, engine, heads, kv, dim, page, order):
    """Pairs of like keys with values of 1 and -1: the sums are far below the values, and what the weights lose shows."""
    lengths = [2, 4, 8, 0, 16, 32, 1, 34, 700]
    q, pools, table, rows = make(21, lengths, heads, kv, dim, page, order, "f16")
    g = np.random.default_rng(22)
    for s, (k, v) in enumerate(rows):
        k[:, 1::2] = k[:, :lengths[s] - 1:2]
        k[:, :, 0] = g.standard_normal(k.shape[:2]) * 0.1  # (but for one element, so that the weights differ a little)
        v[:, 0::2], v[:, 1::2] = -1.0, 1.0
        put(pools, table[s], order, page, k, v)
    want, tol = truth(q, rows, 1 / np.sqrt(dim))
    check(run(ctx, engine, q, pools, table, lengths, order, "f16"), want, tol, f"{heads}/{kv}x{dim}")


@pytest.mark.parametrize("n", [96, 768, 5000])
@pytest.mark.parametrize("low", [12, 20, 24, 26])
def test_many_light_keys_beside_a_heavy_one(ctx, engine, n, low):
    """One key of weight 1 whose value is 0, all others of weights from 2^-low to a quarter of it: they are the
    whole result, however light."""
    heads, dim, page = 2, 64, 16
    q, pools, table, rows = make(23, [n], heads, 1, dim, page, "heads", "f16", fill=0.0)
    g = np.random.default_rng(24)
    q[...] = 0.0
    q[..., 0] = 8.0  # with a scale of 1/8, the score is the key's first element
    k, v = np.zeros((1, n, dim), np.float16), np.ones((1, n, dim), np.float16)
    k[0, :, 0] = -np.log(2.0) * (low + 2 * g.random(n))
    k[0, n // 3, 0], v[0, n // 3] = 0.0, 0.0
    v[0, :, 1] *= 1.0 + g.random(n).astype(np.float16)
    put(pools, table[0], "heads", page, k, v)
    want, tol = truth(q, [[k, v]], 1 / 8)
    check(run(ctx, engine, q, pools, table, [n], "heads", "f16"), want, tol, f"{n} keys of 2^-{low}")


@pytest.mark.parametrize("heads,kv,dim,n", [(4, 2, 64, 64), (3, 1, 128, 128), (8, 1, 64, 3000)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_infinite_values(ctx, engine, heads, kv, dim, n, sign):
    """An infinity in V, at every place of a unit of keys, reaches its dimension as itself, and no other."""
    q, pools, table, rows = make(25, [n], heads, kv, dim, 16, "heads", "f16")
    k, v = rows[0]
    g = np.random.default_rng(26)
    hit = g.random(dim) < 0.8
    for d in np.nonzero(hit)[0]:
        v[:, (d * 37 + n // 2) % n, d] = sign * np.inf
    put(pools, table[0], "heads", 16, k, v)
    got = run(ctx, engine, q, pools, table, [n], "heads", "f16")[0]
    assert np.all(got[:, hit] == sign * np.inf) and np.isfinite(got[:, ~hit]).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("scale", [1e-3, 1.0, 30.0, 1e3, -1e3])
@pytest.mark.parametrize("n", [5, 70, 3000])
def test_scores_past_the_exponentials_reach(ctx, engine, dtype, scale, n):
    """Scores so large that a step of f32 between them is many times the exponential's range: the largest has all
    the weight, two alike share it."""
    q, pools, table, rows = make(27, [n], 4, 2, 64, 16, "heads", dtype)
    g = np.random.default_rng(28)
    k, v = rows[0]
    q[...], k[...] = 0.0, 0.0
    q[..., 0] = np.sign(scale) * (5e4 + 1e4 * g.random(q.shape[:2]))
    k[:, :, 0] = np.linspace(1e4, 4e4, n)  # (fp16: steps of 8 to 32, alike in places; the largest two are not)
    top = [n // 3, n - 2]
    k[:, top, 0] = 6e4
    put(pools, table[0], "heads", 16, k, v)
    want = np.repeat(v[:, top].astype(np.float64).mean(1), 2, 0)
    got = run(ctx, engine, q, pools, table, [n], "heads", dtype, scale=scale)[0]
    half, u = (2.0 ** -11 if dtype == "f16" else 2.0 ** -24), 2.0 ** -24
    # the two weights are equal; a sum, a quotient and the output's rounding
    tol = (half + 4 * u) * np.abs(want) + 4 * u * np.abs(v[:, top].astype(np.float64)).max(1).repeat(2, 0) + 2.0 ** -25
    check(got, want, tol, f"{n} keys, scale {scale}")
