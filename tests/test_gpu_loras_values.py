"""rq_qmatmul_loras with infinite factors."""
import numpy as np
import pytest

from rusty_amd import QuantizedTensor
from test_gpu_loras import KIND, run

pytestmark = pytest.mark.gpu


def zeros(ctx, n, k):
    return QuantizedTensor.rowwise(ctx, np.zeros((n, k), np.int8), np.ones(n, np.float32))


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
