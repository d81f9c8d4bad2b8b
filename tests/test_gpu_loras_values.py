"""rq_qmatmul_loras: adapters whose ranks differ far in size, and infinite factors; the tolerances are those derived in
test_gpu_loras.py."""
import numpy as np
import pytest

from rusty_amd import QuantizedTensor
from test_gpu_loras import KIND, adapters, check, run, truth

pytestmark = pytest.mark.gpu


def zeros(ctx, n, k):
    return QuantizedTensor.rowwise(ctx, np.zeros((n, k), np.int8), np.ones(n, np.float32))


# a row, rows one by one, tiles of rows, the product's own tiles
SIZES = [(1, 256, 256), (2, 256, 256), (16, 256, 256), (256, 256, 256), (257, 256, 256), (300, 331, 256), (1100, 5640, 192)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("rank", [4, 40, 100])
@pytest.mark.parametrize("spread", [20, 29])
def test_ranks_of_very_different_size(ctx, engine, m, n, k, rank, spread):
    """x . A's entries 2^spread apart within a row, and columns that only the small ones reach: each column has the
    accuracy of its own terms."""
    g = np.random.default_rng(31)
    a, b = adapters(g, 3, rank, k, n, "f16")
    size = np.array([0, -spread / 3, -2 * spread / 3, -spread])[np.arange(rank) % 4]
    # all of one sign, so that no sum cancels; fp16's normal numbers
    a[...] = (1 + g.random(a.shape)) * 2.0 ** np.round(size + 14)[:, None]
    x = (1 + g.random((m, k))).astype(np.float16)
    b[...] = np.where(np.arange(rank)[:, None] % 4 == np.arange(n) % 4, 1 + g.random(b.shape), 0.0)
    ids = np.repeat(g.integers(-1, 3, m // 50 + 1), 50)[:m]
    for who in (ids, g.integers(-1, 3, m)):
        want, tol = truth(x, np.zeros((n, k)), a, b, np.ones(3), who, [rank] * 3, "f32", False)
        check(run(ctx, engine, x, zeros(ctx, n, k), a, b, None, who, None, "f16", "f32", "f16"), want, tol, f"{m} rows, 2^{spread}")


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("many", [False, True])
def test_one_rank_far_above_the_others(ctx, engine, m, n, k, many):
    """One entry of f32's upper range and one of its lower in the same row."""
    g = np.random.default_rng(32)
    count = 60 if many else 2
    a, b = np.zeros((count, 9, k), np.float16), np.zeros((count, 9, n), np.float16)
    a[:, 2], a[:, 7] = 2.0 ** 15, 2.0 ** -24
    b[:, 2, ::2], b[:, 7, 1::2] = 1 + g.random((count, (n + 1) // 2)), 1 + g.random((count, n // 2))
    x = ((1 + g.random((m, k))) * 2.0 ** g.integers(-100, 100, m)[:, None]).astype(np.float32)
    ids = g.integers(-1, count, m)
    want, tol = truth(x, np.zeros((n, k)), a, b, np.ones(count), ids, [9] * count, "f32", False)
    check(run(ctx, engine, x, zeros(ctx, n, k), a, b, None, ids, None, "f32", "f32", "f16"), want, tol, f"{m} rows")


@pytest.mark.parametrize("x_t,y_t,a_t", [("f16", "f16", "f16"), ("f32", "f32", "f32"), ("f16", "f32", "f16")])
@pytest.mark.parametrize("m,n,k,count", [(1, 64, 64, 2), (2, 64, 64, 2), (7, 72, 64, 2), (100, 64, 64, 60), (256, 65, 64, 2),
                                         (300, 64, 64, 60), (1100, 5640, 64, 2), (1100, 5640, 64, 60)])
@pytest.mark.parametrize("rank,own", [(5, 5), (40, 33), (16, 1)])
def test_infinite_factor(ctx, engine, x_t, y_t, a_t, m, n, k, count, rank, own):
    """A factor of infinity over positive sums is infinity in every column, whatever the rank leaves of a kernel's step;
    rows of the other adapters are as ever."""
    a, b = np.ones((count, rank, k), KIND[a_t][0]), np.ones((count, rank, n), KIND[a_t][0])
    f = np.where(np.arange(count) % 2, np.inf, 1.0).astype(np.float32)
    x = np.full((m, k), 2.0, KIND[x_t][0])
    ids = (np.arange(m) + 1) % count
    got = run(ctx, engine, x, zeros(ctx, n, k), a, b, f, ids, [own] * count, x_t, y_t, a_t)
    assert np.all(got[ids % 2 == 1] == np.inf) and np.all(got[ids % 2 == 0] == own * 128.0)


@pytest.mark.parametrize("m,n,k", [(2, 64, 64), (100, 64, 64), (300, 64, 64), (300, 65, 64), (1100, 5640, 64)])
def test_infinite_adapter(ctx, engine, m, n, k):
    """An infinity in B reaches its column as itself, with its sign, in rows of any number."""
    a, b = np.ones((2, 40, k), np.float16), np.ones((2, 40, n), np.float16)
    b[1, 3, ::3], b[1, 35, 1::3] = np.inf, -np.inf
    a[:, 35] = 1.0 / 3.0
    x = np.full((m, k), 2.0, np.float16)
    ids = (np.arange(m) + 1) % 2
    got = run(ctx, engine, x, zeros(ctx, n, k), a, b, None, ids, None, "f16", "f32", "f16")
    assert np.isfinite(got[ids == 0]).all() and np.isfinite(got[ids == 1][:, 2::3]).all()
    assert np.all(got[ids == 1][:, ::3] == np.inf) and np.all(got[ids == 1][:, 1::3] == -np.inf)
