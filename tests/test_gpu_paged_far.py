"""Paged caches whose offsets pass 32 bits: pages past 4 GiB of a pool, rows far apart
within a page.  Only the pages that a call names are written."""
import numpy as np
import pytest

from rusty_amd import DType, PagedCache, Rope, UnifiedTensor
from rusty_amd._lib import call
from test_gpu_attn import check
from test_gpu_paged import truth

pytestmark = pytest.mark.gpu


def put(ctx, base, offset, a):
    call("rq_memcpy_h2d", ctx.handle, base + offset, a.ctypes.data, a.nbytes, None)


def get(ctx, base, offset, shape):
    a = np.empty(shape, np.float16)
    call("rq_memcpy_d2h", ctx.handle, a.ctypes.data, base + offset, a.nbytes, None)
    return a


@pytest.mark.parametrize("n_pages,page,strides", [(40000, 512, (0, 0, 0)), (3, 16, (1 << 31, 1 << 29, 1 << 24)),
                                                  (3, 64, (128, 64, 1 << 26))], ids=["far pages", "far rows", "pages within rows"])
def test_far(ctx, engine, n_pages, page, strides):
    """A pool of 4 to 8 GiB (K and V in one memory): the last page, or its last rows, lie past 4 GiB."""
    kv, dim = 2, 64
    ps, hs, xs = strides if any(strides) else (page * kv * dim, page * dim, dim)
    size = 2 * ((n_pages - 1) * ps + (kv - 1) * hs + (page - 1) * xs + dim)
    assert size > 1 << 32
    pool = UnifiedTensor.empty(ctx, [size], DType.U8)
    view = UnifiedTensor(ctx, pool.ptr, (n_pages, kv, page, dim), DType.FP16, owner=False)
    n = [page + 5, 3]
    table = np.array([[n_pages - 1, 1], [n_pages - 2 if n_pages > 3 else 0, -1]], np.int32)
    g = np.random.default_rng(1)
    rows = [[g.standard_normal((kv, m, dim)).astype(np.float16)] * 2 for m in n]  # K and V alike: one memory
    for s, (k, _) in enumerate(rows):
        for h in range(kv):
            for p in range(n[s]):
                put(ctx, pool.ptr, 2 * (int(table[s, p // page]) * ps + h * hs + p % page * xs), np.ascontiguousarray(k[h, p]))
    cache = PagedCache(view, view, UnifiedTensor.new(ctx, table, dtype=DType.I32), strides=strides)
    q = g.standard_normal((2, 4, dim)).astype(np.float16)
    Q, out = UnifiedTensor.new(ctx, q), UnifiedTensor.new(ctx, np.zeros_like(q))
    engine.attn_paged(ctx, Q, cache, UnifiedTensor.new(ctx, np.array(n), dtype=DType.I32), out)
    check(out.to_vec(), *truth(q, rows, 1 / 8, True), "far")
    # a token's key and value into the far pages, at position 0: the turn by 0 leaves the key as it is
    new = g.standard_normal((2, kv, dim)).astype(np.float16)
    N, Z = UnifiedTensor.new(ctx, new), UnifiedTensor.new(ctx, np.zeros(2, np.int32), dtype=DType.I32)
    engine.rope_append(ctx, Q, N, N, Rope(ctx, dim), Z, cache, out)
    assert np.array_equal(out.to_vec(), q)
    for s in range(2):
        for h in range(kv):
            assert np.array_equal(get(ctx, pool.ptr, 2 * (int(table[s, 0]) * ps + h * hs), (dim,)), new[s, h])
