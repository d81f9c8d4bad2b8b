"""Argument checks of the rotary, paged-cache and adapter-batch entry points, the
rotary frequencies, and where a paged cache keeps a position (host arithmetic,
no device; no pointer is read but the page table)."""
import ctypes
import math

import numpy as np
import pytest

from rusty_amd import Rope, _lib

INV, SHAPE, UNSUP = _lib.RQ_ERR_INVALID_ARGUMENT, _lib.RQ_ERR_SHAPE, _lib.RQ_ERR_UNSUPPORTED
P = 0x10000  # an aligned address
WS = 1 << 40
p, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64


def _fn(name, args, res=ctypes.c_int):
    fn = getattr(_lib.lib(), name)
    fn.argtypes, fn.restype = args, res
    return fn


def ref(s):
    return None if s is None else ctypes.byref(s)


def rope(freqs=P, dim=64, rot=64, layout=0, magnitude=1.0):
    return _lib.rq_rope(freqs, dim, rot, layout, magnitude)


def attn(heads=8, kv=2, dim=64, dtype=_lib.RQ_F16, scale=0.0, q_row=0, k_row=0, v_row=0, out_row=0):
    return _lib.rq_attn(heads, kv, dim, dtype, scale, 0, q_row, k_row, v_row, out_row)


def pages(k=P, v=P, table=P, strides=(0, 0, 0), table_row=0, n_seqs=3, max_pages=40, n_pages=100, page=16):
    return _lib.rq_kv_pages(k, v, table, *strides, table_row, n_seqs, max_pages, n_pages, page)


def rows(r=rope(), x=P, x_row=0, positions=P, tokens=10, heads=4, dtype=_lib.RQ_F16, out=2 * P, out_row=0, flags=0):
    return _fn("rusty_rope_check", [p, p, p, p, p, p, i64, p, p, i64, i32, ctypes.c_int, p, i64, ctypes.c_uint])(
        ref(r), None, None, x, None, None, x_row, None, positions, tokens, heads, dtype, out, out_row, flags)


def append(r=rope(), a=attn(), c=pages(), q=P, k=P, v=P, starts=P, positions=P, tokens=10, out=2 * P):
    return _fn("rusty_rope_check", [p, p, p, p, p, p, i64, p, p, i64, i32, ctypes.c_int, p, i64, ctypes.c_uint])(
        ref(r), ref(a), ref(c), q, k, v, 0, starts, positions, tokens, 0, 0, out, 0, 0)


def paged(a=attn(), c=pages(), q=P, lengths=P, out=P, work=P, work_bytes=WS):
    return _fn("rusty_paged_check", [p, p, p, p, p, p, ctypes.c_size_t])(ref(a), ref(c), q, lengths, out, work, work_bytes)


def test_limits():
    """Sizes up to the documented ones are taken, one past them refused before anything is launched."""
    assert paged(c=pages(n_seqs=65536)) == 0 and paged(c=pages(n_seqs=65537)) == SHAPE
    assert append(c=pages(n_seqs=65537)) == 0
    most = (1 << 24) - 256
    for kw in (dict(m=most), dict(w=weight(n=most)), dict(w=weight(k=most))):
        assert loras(work_bytes=1 << 62, **kw) == 0
    for kw in (dict(m=most + 1), dict(w=weight(n=most + 1)), dict(w=weight(k=most + 128))):
        assert loras(work_bytes=1 << 62, **kw) == SHAPE


# ---- rotary rows -------------------------------------------------------------------


def test_rows_refusals():
    assert rows() == 0 and rows(out=P) == 0 and rows(rope(rot=2)) == 0 and rows(rope(dim=6, rot=4, layout=1)) == 0
    assert rows(None) == INV and rows(rope(layout=2)) == INV and rows(rope(layout=-1)) == INV
    assert rows(rope(magnitude=float("nan"))) == INV and rows(rope(magnitude=float("inf"))) == INV
    for dim, rot in ((64, 0), (64, 3), (64, 66), (64, -2), (0, 0), (1, 1), (1026, 64)):
        assert rows(rope(dim=dim, rot=rot)) == SHAPE, (dim, rot)
    assert rows(dtype=2) == INV and rows(flags=2) == INV and rows(flags=1) == 0
    assert rows(tokens=-1) == SHAPE and rows(tokens=1 << 31) == SHAPE and rows(heads=-1) == SHAPE
    assert rows(heads=65537) == SHAPE
    assert rows(x_row=255) == SHAPE and rows(out_row=255) == SHAPE and rows(x_row=257) == 0
    assert rows(x_row=-512) == SHAPE and rows(x_row=1 << 32) == SHAPE
    assert rows(out=P, x_row=512) == SHAPE and rows(out=P, x_row=512, out_row=512) == 0
    for name in ("x", "positions", "out"):
        assert rows(**{name: None}) == INV and rows(**{name: P + 1}) == UNSUP
    assert rows(rope(freqs=None)) == INV and rows(rope(freqs=P + 4)) == UNSUP
    assert rows(x=P + 2) == 0 and rows(x=P + 2, dtype=_lib.RQ_F32) == UNSUP
    # nothing to do: no pointer is needed
    for kw in (dict(tokens=0), dict(heads=0)):
        assert rows(rope(freqs=None), x=None, positions=None, out=None, **kw) == 0


# ---- the paged cache -----------------------------------------------------------------

CACHES = [(dict(n_seqs=-1), SHAPE), (dict(max_pages=-1), SHAPE), (dict(n_pages=-1), SHAPE), (dict(page=0), UNSUP),
          (dict(page=24), UNSUP), (dict(page=-16), UNSUP), (dict(page=1 << 17), UNSUP), (dict(max_pages=1 << 27), SHAPE),
          (dict(n_seqs=1 << 20, max_pages=1 << 16), SHAPE), (dict(n_seqs=1 << 30, max_pages=0), SHAPE),
          (dict(strides=(2048, 32, 64)), SHAPE), (dict(strides=(2048, 1024, 32)), SHAPE),
          (dict(strides=(32, 1024, 64)), SHAPE), (dict(strides=(-2048, 1024, 64)), SHAPE),
          (dict(strides=(2052, 1024, 64)), UNSUP), (dict(strides=(2048, 1028, 64)), UNSUP),
          (dict(strides=(2048, 1024, 68)), UNSUP), (dict(strides=(1 << 41, 1024, 64)), SHAPE),
          (dict(table_row=39), SHAPE), (dict(table_row=-1), SHAPE), (dict(table_row=1 << 32), SHAPE),
          (dict(k=None), INV), (dict(v=None), INV), (dict(table=None), INV), (dict(k=P + 8), UNSUP), (dict(v=P + 2), UNSUP),
          (dict(table=P + 2), UNSUP)]


@pytest.mark.parametrize("kw,want", CACHES, ids=lambda v: str(v))
def test_cache_refusals(kw, want):
    assert paged(c=pages(**kw)) == want
    assert append(c=pages(**kw)) == want


def test_cache_accepted():
    for c in (pages(), pages(page=1), pages(strides=(2048, 64, 128)), pages(table_row=64), pages(n_pages=1, strides=(0, 1024, 64)),
              pages(max_pages=0, table=None), pages(n_pages=0, k=None, v=None)):
        assert paged(c=c) == 0 and append(c=c) == 0
    one = attn(8, 1)
    assert paged(one, pages(strides=(1024, 0, 64))) == 0


@pytest.mark.parametrize("kw,want", [(dict(dtype=2), INV), (dict(scale=float("nan")), INV), (dict(dim=96), UNSUP),
                                     (dict(heads=8, kv=3), SHAPE), (dict(heads=0), SHAPE), (dict(q_row=511), SHAPE),
                                     (dict(q_row=516), UNSUP), (dict(out_row=514), UNSUP), (dict(q_row=1 << 22), SHAPE)],
                         ids=lambda v: str(v))
def test_heads_refusals(kw, want):
    assert paged(attn(**kw)) == want
    assert append(a=attn(**kw)) == want


def test_append_refusals():
    assert append() == 0 and append(out=P) == 0
    assert append(None) == INV and append(c=None) == INV
    assert append(rope(dim=128, rot=64)) == SHAPE and append(rope(rot=32)) == 0
    assert append(a=attn(k_row=127)) == SHAPE and append(a=attn(v_row=132)) == UNSUP
    assert append(out=P, a=attn(q_row=768)) == SHAPE and append(out=P, a=attn(q_row=768, out_row=768)) == 0
    for name in ("q", "k", "v", "positions", "out"):
        assert append(**{name: None}) == INV and append(**{name: P + 2}) == UNSUP
    assert append(starts=P + 2) == UNSUP
    # without starts a token is a sequence
    assert append(starts=None) == SHAPE and append(starts=None, tokens=3) == 0
    assert append(tokens=-1) == SHAPE and append(tokens=1 << 31) == SHAPE
    none = dict(q=None, k=None, v=None, starts=None, positions=None, out=None)
    assert append(tokens=0, **none) == 0 and append(c=pages(n_seqs=0, k=None, v=None, table=None), tokens=0, **none) == 0


def test_paged_refusals():
    assert paged() == 0 and paged(None) == INV and paged(c=None) == INV
    for name in ("q", "lengths", "out"):
        assert paged(**{name: None}) == INV and paged(**{name: P + 2}) == UNSUP
    assert paged(c=pages(n_seqs=0, k=None, v=None, table=None), q=None, lengths=None, out=None, work=None, work_bytes=0) == 0


def test_paged_workspace():
    fn = _lib.lib().rq_attn_paged_workspace
    for a in (attn(), attn(32, 8, 128), attn(96, 2), attn(128, 128), attn(8192, 8192)):
        c = pages()
        need = fn(ref(a), ref(c))
        assert need % 8 == 0
        assert paged(a, c, work=P, work_bytes=need) == 0
        if need:
            assert paged(a, c, work=P, work_bytes=need - 1) == INV
            assert paged(a, c, work=None, work_bytes=need) == INV
            assert paged(a, c, work=P + 8, work_bytes=need) == UNSUP
    assert fn(None, ref(pages())) == 0 and fn(ref(attn()), None) == 0 and fn(ref(attn(dim=96)), ref(pages())) == 0


@pytest.mark.parametrize("page", [1, 8, 16, 256])
def test_where_a_position_lies(page):
    """Every position of a table with missing and foreign entries, and some outside it."""
    at = _fn("rusty_paged_at", [p, p, ctypes.c_int, ctypes.c_int], i64)
    g = np.random.default_rng(page)
    table = g.integers(-2, 9, (3, 5)).astype(np.int32)  # n_pages 7: -2, -1, 7 and 8 name none
    table[0, 0], table[1, 1] = 2 ** 31 - 1, -2 ** 31
    a = attn()
    for strides, row in (((0, 0, 0), 0), ((page * 128 + 64, 64, 128), 0)):
        c = pages(table=table.ctypes.data, strides=strides, table_row=row, max_pages=5, n_pages=7, page=page)
        ps, _, pos = strides if any(strides) else (page * 2 * 64, 0, 64)
        for s in range(3):
            for x in (-2 ** 31, -1, *range(5 * page), 5 * page, 2 ** 31 - 1):
                e = table[s, x // page] if 0 <= x < 5 * page else -1
                want = 2 * (int(e) * ps + x % page * pos) if 0 <= e < 7 else -1
                assert at(ref(a), ref(c), s, x) == want, (s, x)


def test_where_a_far_page_lies():
    """Offsets past 32 bits."""
    at = _fn("rusty_paged_at", [p, p, ctypes.c_int, ctypes.c_int], i64)
    table = np.array([[2 ** 30]], np.int32)
    c = pages(table=table.ctypes.data, n_seqs=1, max_pages=1, n_pages=2 ** 31 - 1)
    assert at(ref(attn()), ref(c), 0, 3) == 2 * (2 ** 30 * 16 * 2 * 64 + 3 * 64)


# ---- adapters --------------------------------------------------------------------------


def weight(n=64, k=128):
    return _lib.rq_qweight(P, P, None, n, k, _lib.RQ_Q_ROWWISE_I8, 0, None)


def lora_set(a=P, b=P, factors=P, ranks=P, n=4, rank=16, dtype=_lib.RQ_F16, reserved=0):
    return _lib.rq_lora_set(a, b, factors, ranks, n, rank, dtype, reserved)


def loras(w=weight(), s=lora_set(), ids=P, x=P, xt=_lib.RQ_F16, y=P, yt=_lib.RQ_F16, m=5, work=P, work_bytes=WS):
    return _fn("rusty_loras_check", [p, p, p, p, ctypes.c_int, p, ctypes.c_int, i64, p, ctypes.c_size_t])(
        ref(w), ref(s), ids, x, xt, y, yt, m, work, work_bytes)


def test_loras_refusals():
    assert loras() == 0 and loras(s=lora_set(factors=None, ranks=None)) == 0
    assert loras(None) == INV and loras(s=None) == INV
    for kw, want in ((dict(dtype=2), INV), (dict(reserved=1), INV), (dict(n=-1), SHAPE), (dict(rank=0), SHAPE),
                     (dict(rank=257), SHAPE), (dict(a=None), INV), (dict(b=None), INV), (dict(a=P + 1), UNSUP),
                     (dict(b=P + 1), UNSUP), (dict(factors=P + 2), UNSUP), (dict(ranks=P + 2), UNSUP)):
        assert loras(s=lora_set(**kw)) == want, kw
    assert loras(s=lora_set(a=P + 2)) == 0 and loras(s=lora_set(a=P + 2, dtype=_lib.RQ_F32)) == UNSUP
    assert loras(s=lora_set(a=None, b=None, n=0)) == 0
    assert loras(xt=2) == INV and loras(yt=-1) == INV and loras(m=-1) == SHAPE and loras(m=1 << 31) == SHAPE
    for name in ("ids", "x", "y"):
        assert loras(**{name: None}) == INV and loras(**{name: P + 1}) == UNSUP
    assert loras(x=P + 2) == 0 and loras(x=P + 2, xt=_lib.RQ_F32) == UNSUP
    assert loras(weight(1 << 41, 128), m=1) == SHAPE and loras(weight(k=1 << 41), m=1) == SHAPE
    assert loras(s=lora_set(n=2 ** 31 - 1, rank=256), w=weight(1 << 24, 16)) == SHAPE
    for kw in (dict(m=0), dict(w=weight(n=0))):
        assert loras(ids=None, x=None, y=None, work=None, work_bytes=0, **kw) == 0
    assert loras(weight(k=0), s=lora_set(a=None), x=None) == 0


def test_loras_workspace():
    fn = _lib.lib().rq_qmatmul_loras_workspace
    for m, k, n, yt in ((1, 128, 64, 0), (5, 4096, 1000, 1), (2048, 11008, 33, 1), (3, 0, 7, 0)):
        s = lora_set()
        need = fn(ref(s), m, k, n, 1, yt)
        kw = dict(w=weight(n, k), s=s, m=m, yt=yt)
        assert loras(work=P, work_bytes=need, **kw) == 0 and loras(work=P, work_bytes=need - 1, **kw) == INV
        assert loras(work=None, work_bytes=need, **kw) == INV and loras(work=P + 16, work_bytes=need, **kw) == UNSUP
    assert fn(None, 1, 1, 1, 1, 1) == 0 and fn(ref(lora_set(rank=0)), 1, 1, 1, 1, 1) == 0
    assert fn(ref(lora_set()), -1, 1, 1, 1, 1) == 0 and fn(ref(lora_set()), 1 << 40, 1 << 40, 1, 1, 1) == 0


# ---- frequencies -------------------------------------------------------------------------


def turns(f, trained):
    return trained * f / (2 * math.pi)


@pytest.mark.parametrize("rot", [2, 4, 26, 64, 128])
@pytest.mark.parametrize("theta", [10000.0, 500000.0])
def test_frequencies(rot, theta):
    plain, m = Rope.frequencies_of(rot, theta)
    want = [theta ** (-2 * i / rot) for i in range(rot // 2)]
    np.testing.assert_allclose(plain, want, rtol=1e-14)
    assert m == 1.0
    linear, m = Rope.frequencies_of(rot, theta, "linear", factor=4.0)
    np.testing.assert_allclose(linear, np.array(want) / 4, rtol=1e-14)
    # the base grows: the first pair is kept, the last divided by the factor (where there are two)
    stretch, m = Rope.frequencies_of(rot, theta, "stretch", factor=4.0)
    assert stretch[0] == 1.0 and m == 1.0
    if rot > 2:
        np.testing.assert_allclose(stretch[-1], want[-1] / 4, rtol=1e-13)
    bands, m = Rope.frequencies_of(rot, theta, "bands", factor=8.0, trained=8192, low=1.0, high=4.0)
    assert m == 1.0
    for f, g in zip(want, bands):
        n = turns(f, 8192)
        kept = min(max((n - 1) / 3, 0), 1)
        assert math.isclose(g, f * kept + f / 8 * (1 - kept), rel_tol=1e-13)
    ramp, m = Rope.frequencies_of(rot, theta, "ramp", factor=8.0, trained=4096, low=1.0, high=32.0)
    assert math.isclose(m, 0.1 * math.log(8) + 1, rel_tol=1e-6)
    index = lambda n: rot / 2 * math.log(4096 / (2 * math.pi * n)) / math.log(theta)  # noqa: E731
    lo, hi = max(math.floor(index(32)), 0), min(math.ceil(index(1)), rot - 1)
    for i, (f, g) in enumerate(zip(want, ramp)):
        slow = min(max((i - lo) / max(hi - lo, 0.001), 0), 1)
        assert math.isclose(g, f * (1 - slow) + f / 8 * slow, rel_tol=1e-13)


def test_frequency_refusals():
    def go(f=True, m=True, **kw):
        c = dict(theta=1e4, factor=2.0, trained=100.0, low=1.0, high=4.0, scaling=3, rot_dim=64, **{})
        c.update(kw)
        out, mag = (ctypes.c_double * 512)(), ctypes.c_float()
        return _lib.lib().rq_rope_frequencies(ctypes.byref(_lib.rq_rope_config(**c)), out if f else None,
                                              ctypes.byref(mag) if m else None)

    nan, inf = float("nan"), float("inf")
    assert go() == 0 and go(f=False) == INV and go(m=False) == INV
    assert _lib.lib().rq_rope_frequencies(None, None, None) == INV
    for kw, want in ((dict(scaling=5), INV), (dict(scaling=-1), INV), (dict(rot_dim=0), SHAPE), (dict(rot_dim=63), SHAPE),
                     (dict(rot_dim=1026), SHAPE), (dict(theta=1.0), INV), (dict(theta=nan), INV), (dict(theta=inf), INV),
                     (dict(factor=0.5), INV), (dict(factor=nan), INV), (dict(factor=inf), INV), (dict(trained=0.0), INV),
                     (dict(trained=inf), INV), (dict(low=0.0), INV), (dict(low=4.0), INV), (dict(high=inf), INV),
                     (dict(high=nan), INV)):
        assert go(**kw) == want, kw
    assert go(scaling=0, factor=nan, trained=nan) == 0 and go(scaling=1, trained=nan) == 0


def test_struct_layouts(tmp_path):
    """The ctypes mirrors have the sizes and field offsets a C compiler gives the header's structs."""
    import shutil
    import subprocess
    from pathlib import Path

    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    structs = [_lib.rq_rope, _lib.rq_rope_config, _lib.rq_kv_pages, _lib.rq_lora_set]
    body = "".join(f'printf("%zu ", sizeof({s.__name__}));' + "".join(
        f'printf("%zu ", offsetof({s.__name__}, {f[0]}));' for f in s._fields_) for s in structs)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "rusty_hip.h"\nint main(void) {' + body + "return 0;}\n")
    root = Path(__file__).resolve().parent.parent
    subprocess.run([gcc, "-std=c99", "-I", str(root / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [v for s in structs for v in (ctypes.sizeof(s), *(getattr(s, f[0]).offset for f in s._fields_))]
    assert got == want
