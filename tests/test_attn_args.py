"""The attention entry points' argument checks and workspace size (host
arithmetic, no device; no pointer is read)."""
import ctypes

import pytest

from rusty_amd import _lib

INV, SHAPE, UNSUP = _lib.RQ_ERR_INVALID_ARGUMENT, _lib.RQ_ERR_SHAPE, _lib.RQ_ERR_UNSUPPORTED
P = 0x10000  # an aligned address
WS = 1 << 40


def _check():
    fn = _lib.lib().rusty_attn_check
    p = ctypes.c_void_p
    fn.argtypes = [p, p, p, p, p, p, p, p, ctypes.c_int32, ctypes.c_int64, ctypes.c_int32, p, p, ctypes.c_size_t]
    fn.restype = ctypes.c_int
    return fn


def attn(heads=8, kv=2, dim=64, dtype=_lib.RQ_F16, scale=0.0, reserved=0, q_row=0, k_row=0, v_row=0, out_row=0):
    return _lib.rq_attn(heads, kv, dim, dtype, scale, reserved, q_row, k_row, v_row, out_row)


def packed(a=None, q=P, k=P, v=P, starts=P, n_seqs=3, tokens=10, out=P):
    a = a or attn()
    return _check()(ctypes.byref(a), None, q, k, v, starts, None, None, n_seqs, tokens, 0, out, None, 0)


def tree(a=None, k=P, v=P, strides=(0, 0, 0), n_seqs=3, capacity=640, q=P, starts=P, lengths=P, mask=P, tokens=10,
         max_nodes=16, out=P, work=P, work_bytes=WS):
    a = a or attn()
    c = _lib.rq_kv_cache(k, v, *strides, n_seqs, capacity)
    return _check()(ctypes.byref(a), ctypes.byref(c), q, None, None, starts, lengths, mask, 0, tokens, max_nodes, out,
                    work, work_bytes)


BOTH = [(dict(dtype=2), INV), (dict(dtype=-1), INV), (dict(reserved=1), INV), (dict(scale=float("nan")), INV),
        (dict(scale=float("inf")), INV), (dict(dim=96), UNSUP), (dict(dim=0), UNSUP), (dict(heads=0), SHAPE),
        (dict(kv=0), SHAPE), (dict(heads=8, kv=3), SHAPE), (dict(heads=-8, kv=-2), SHAPE), (dict(q_row=511), SHAPE),
        (dict(out_row=-512), SHAPE), (dict(q_row=516), UNSUP), (dict(out_row=514), UNSUP),
        (dict(q_row=1 << 41), SHAPE), (dict(heads=1 << 17, kv=2), SHAPE)]


@pytest.mark.parametrize("kw,want", BOTH, ids=lambda v: str(v))
def test_descriptor_refusals(kw, want):
    assert packed(attn(**kw)) == want
    assert tree(attn(**kw)) == want


def test_packed_refusals():
    assert packed() == 0 and packed(attn(scale=-1.5)) == 0
    for a, want in ((attn(k_row=127), SHAPE), (attn(v_row=100), SHAPE), (attn(k_row=132), UNSUP),
                    (attn(v_row=130), UNSUP)):
        assert packed(a) == want
    assert packed(attn(k_row=768, v_row=768, q_row=768)) == 0
    assert packed(attn(dtype=_lib.RQ_F32, q_row=516)) == 0  # 4 elements are 16 bytes
    assert packed(n_seqs=-1) == SHAPE and packed(tokens=-1) == SHAPE and packed(tokens=1 << 31) == SHAPE
    for name in ("q", "k", "v", "starts", "out"):
        assert packed(**{name: None}) == INV
        assert packed(**{name: P + 2}) == UNSUP
    # nothing to do: no pointer is needed
    assert packed(q=None, k=None, v=None, starts=None, out=None, n_seqs=0) == 0
    assert packed(q=None, k=None, v=None, starts=None, out=None, tokens=0) == 0


def test_tree_refusals():
    assert tree() == 0 and tree(mask=None) == 0
    assert tree(max_nodes=0) == SHAPE and tree(max_nodes=65) == SHAPE and tree(max_nodes=64) == 0
    assert tree(n_seqs=-1) == SHAPE and tree(capacity=-1) == SHAPE and tree(tokens=-1) == SHAPE
    for strides, want in (((81920, 40960, 32), SHAPE), ((81920, 32, 64), SHAPE), ((32, 40960, 64), SHAPE),
                          ((-8, 40960, 64), SHAPE), ((81924, 40960, 64), UNSUP), ((81920, 40964, 64), UNSUP),
                          ((81920, 40960, 68), UNSUP), ((1 << 41, 40960, 64), SHAPE), ((81920, 1 << 41, 64), SHAPE),
                          ((81920, 64, 1 << 25), SHAPE), ((81920, 64, 128), 0)):
        assert tree(strides=strides) == want, strides
    assert tree(attn(kv=1), strides=(40960, 0, 64)) == 0 and tree(strides=(0, 40960, 64), n_seqs=1) == 0
    for name in ("q", "starts", "lengths", "out", "k", "v"):
        assert tree(**{name: None}) == INV
        assert tree(**{name: P + 2}) == UNSUP
    assert tree(mask=P + 4) == UNSUP
    # an empty cache needs no K or V; no tokens need nothing
    assert tree(k=None, v=None, capacity=0) == 0
    assert tree(k=None, v=None, q=None, starts=None, lengths=None, out=None, tokens=0) == 0
    assert tree(k=None, v=None, q=None, starts=None, lengths=None, out=None, n_seqs=0) == 0


def test_workspace():
    """A call with less than the queried bytes, or a misaligned workspace, is refused where any is needed."""
    fn = _lib.lib().rq_attn_tree_workspace
    a = attn(32, 4)
    for n_seqs, tokens, nodes, cap in ((1, 1, 1, 640), (1, 64, 64, 32768), (8, 100, 16, 2048), (0, 0, 1, 0)):
        need = fn(ctypes.byref(a), n_seqs, tokens, nodes, cap)
        assert need % 16 == 0
        kw = dict(n_seqs=n_seqs, tokens=tokens, max_nodes=nodes, capacity=cap)
        assert tree(a, work=P, work_bytes=need, **kw) == 0
        if need:
            assert tree(a, work=P, work_bytes=need - 1, **kw) == INV
            assert tree(a, work=None, work_bytes=need, **kw) == INV
            assert tree(a, work=P + 8, work_bytes=need, **kw) == UNSUP
    for bad in (attn(dim=96), attn(heads=0)):
        assert fn(ctypes.byref(bad), 1, 1, 1, 640) == 0
    assert fn(None, 1, 1, 1, 640) == 0 and fn(ctypes.byref(a), 1, 1, 65, 640) == 0
    assert fn(ctypes.byref(a), -1, 1, 1, 640) == 0 and fn(ctypes.byref(a), 1, -1, 1, 640) == 0
