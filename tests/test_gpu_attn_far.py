"""Attention over rows that lie more than 4 GiB apart: the same bits as over packed ones."""
import numpy as np
import pytest
from test_gpu_attn import KIND, packed_inputs, run_packed, run_tree, tree_inputs

from rusty_amd import DType, UnifiedTensor, _lib

pytestmark = pytest.mark.gpu


def put(ctx, base, at, rows):
    """rows[i] to the device at byte at[i] of base."""
    for a, r in zip(at, rows):
        r = np.ascontiguousarray(r)
        _lib.call("rq_memcpy_h2d", ctx.handle, base.ptr + int(a), r.ctypes.data, r.nbytes, None)


def test_packed_rows_far_apart(ctx, engine):
    """q, k and v in rows of 2^21 elements, the widest allowed."""
    total, heads, kv, dim, row = 1100, 2, 1, 64, 1 << 21
    starts = [0, 700, 1100]
    q, k, v = packed_inputs(50, total, heads, kv, dim, "f16")
    ref = run_packed(ctx, engine, q, k, v, starts, "f16")
    far = UnifiedTensor.empty(ctx, [(total - 1) * row + 4096], DType.FP16)
    put(ctx, far, np.arange(total) * row * 2, np.concatenate([q, k, v], 1))
    see = lambda t, at, h: UnifiedTensor(ctx, t.ptr + at * dim * 2, [total, h, dim], DType.FP16, owner=False)  # noqa: E731
    engine.attn_packed(ctx, see(far, 0, heads), see(far, heads, kv), see(far, heads + kv, kv),
                       UnifiedTensor.new(ctx, np.array(starts, np.int32), dtype=DType.I32), see(far, 8, heads), q_row=row,
                       k_row=row, v_row=row, out_row=row)
    got = np.empty((total, heads, dim), np.float16)
    for i in range(total):
        _lib.call("rq_memcpy_d2h", ctx.handle, got[i].ctypes.data, far.ptr + i * row * 2 + 8 * dim * 2, got[i].nbytes, None)
    assert np.array_equal(got, ref)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("far", ["positions", "heads", "sequences"])
def test_tree_cache_far_apart(ctx, engine, dtype, far):
    """A cache whose positions, heads or sequences reach past 4 GiB, k and v side by side in one buffer."""
    heads, kv, dim, size = 4, 2, 64, KIND[dtype][1].itemsize
    lengths, nodes, cap = ([9000], [7], 9100) if far == "positions" else ([300, 21], [7, 3], 320)
    q, k, v, mask = tree_inputs(51, lengths, nodes, cap, heads, kv, dim, dtype)
    ref = run_tree(ctx, engine, q, k, v, lengths, nodes, mask, dtype)
    near, wide = 2 * dim, (9 << 28) // size  # elements: a row of k and of v; 2.25 GiB
    pos = {"positions": (1 << 19) // size, "heads": near, "sequences": near}[far]  # 512 KiB: 4.4 GiB over the cache
    head = {"positions": near, "heads": 2 * wide, "sequences": near * cap}[far]
    seq = {"positions": 0, "heads": near * cap, "sequences": 2 * wide}[far]
    where = (np.arange(len(lengths))[:, None, None] * seq + np.arange(kv)[:, None] * head + np.arange(cap) * pos) * size
    buf = UnifiedTensor.empty(ctx, [int(where.max()) + near * size], DType.U8)
    assert where.max() > 1 << 32
    rows = np.concatenate([k, v], -1)
    if far == "positions":
        # (a position's heads lie side by side)
        put(ctx, buf, where[0, 0], rows[0].transpose(1, 0, 2))
    else:
        put(ctx, buf, where[:, :, 0].ravel(), rows.reshape(-1, cap, near))
    kind = KIND[dtype][1]
    T = lambda a, d=kind: UnifiedTensor.new(ctx, a, dtype=d)  # noqa: E731
    out = T(np.zeros(q.shape))
    K, V = (UnifiedTensor(ctx, buf.ptr + i * dim * size, k.shape, kind, owner=False) for i in (0, 1))
    engine.attn_tree(ctx, T(q), K, V, T(np.concatenate([[0], np.cumsum(nodes)]), DType.I32), T(np.array(lengths), DType.I32),
                     T(mask, DType.U64), out, max(nodes), strides=(seq, head, pos))
    assert np.array_equal(out.to_vec(), ref)
