"""rq_qmatmul_loras where the shared product's tiles add many adapters, of many ranks; the tolerances are those of
test_gpu_loras.py."""
import numpy as np
import pytest

from rusty_amd import QuantizedTensor
from test_gpu_loras import case, run
from test_lora_tiles import tile

pytestmark = pytest.mark.gpu

WIDE, NARROW = (8000, 1000, 192, 128256), (8192, 512, 64, 128128)


@pytest.mark.parametrize("form,x_t,y_t", [("rowwise8", "f16", "f16"), ("rowwise8", "f32", "f32"), ("affine8", "f16", "f32")])
@pytest.mark.parametrize("shape,count,rank", [(WIDE, 3, 150), (WIDE, 16, 40), (WIDE, 17, 33), (WIDE, 60, 70), (NARROW, 16, 40), (NARROW, 17, 33)])
def test_many_adapters(ctx, engine, form, x_t, y_t, shape, count, rank):
    """In turn up to 16 adapters a tile, row by row above, several steps of ranks each."""
    m, n, k, want = shape
    assert tile(m, n, k, rank, count, form == "affine8") == want
    g = np.random.default_rng(count)
    case(ctx, engine, rank, m, n, k, count, rank, form, x_t, y_t, "f16", ids=g.integers(-1, count, m), some_ranks=count == 17)


@pytest.mark.parametrize("count,rank,own", [(4, 5, 5), (60, 5, 5), (60, 40, 33)])
def test_infinite_factor(ctx, engine, count, rank, own):
    m, n, k, want = WIDE
    assert tile(m, n, k, rank, count) == want
    w = QuantizedTensor.rowwise(ctx, np.zeros((n, k), np.int8), np.ones(n, np.float32))
    a, b = np.ones((count, rank, k), np.float16), np.ones((count, rank, n), np.float16)
    f = np.where(np.arange(count) % 2, np.inf, 1.0).astype(np.float32)
    ids = np.arange(m) % count
    got = run(ctx, engine, np.full((m, k), 2.0, np.float16), w, a, b, f, ids, [own] * count, "f16", "f16", "f16")
    assert np.all(got[ids % 2 == 1] == np.inf) and np.all(got[ids % 2 == 0] == own * 384.0)
