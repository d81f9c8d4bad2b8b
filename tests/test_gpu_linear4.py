"""4-bit affine weights (RQ_Q_AFFINE_U4) through the public entry points,
against a plain computation in 64 bits.

Tolerance of y = sum_k x_k (u_k s + b), u = 2^-24: the kernels add products of
x with codes (or codes + 16) and sums of x, scaled by s and b per group, in
f32.  With S = sum_k |x_k| (|s| (u_k + 32) + |b|), each partial sum is at most S,
the longest chain of additions one value passes is K / 32 + 64 long, and
f32 activations enter as two fp16 terms that lose at most 2^-21 of them:
|dy| <= (K / 32 + 64) u S + 2^-21 S, and half a step of the output, 2^-11 |y|
(fp16) or u |y|.  Past 16 rows each product loses half an fp16 step of the
weight and (f32 rows) of the activation, the documented accuracy there:
2 * 2^-11 sum_k |x_k| |w_k|, and a weight below fp16's normal range half its spacing.
"""
import ctypes

import numpy as np
import pytest

from rusty_amd import DType, QuantizedTensor, RqError, UnifiedTensor, _lib
from rusty_amd.hiprt import Graph, Stream

pytestmark = pytest.mark.gpu

KIND = {"f16": (np.float16, DType.FP16), "f32": (np.float32, DType.FP32)}
U = 2.0 ** -24


def weight(g, n, k, group, biases=True):
    u = g.integers(0, 16, size=(n, k), dtype=np.uint8)
    s = (g.uniform(0.5, 1.5, size=(n, k // group)) * 0.02 / 4.61).astype(np.float32)
    b = (-7.5 * s * g.uniform(0.95, 1.05, size=s.shape)).astype(np.float32) if biases else None
    return u, s, b, group


def parts(w):
    """(W, |s| (u + 32) + |b|) in 64 bits."""
    u, s, b, group = w
    rep = lambda a: np.repeat(a.astype(np.float64), group, axis=1)  # noqa: E731
    bb = rep(b) if b is not None else 0.0
    return u * rep(s) + bb, np.abs(rep(s)) * (u + 32.0) + np.abs(bb)


def truth(x, w, y_f16):
    W, S = parts(w)
    x = x.astype(np.float64)
    y, size = x @ W.T, np.abs(x) @ S.T
    K = W.shape[1]
    tol = ((K / 32 + 64) * U + 2.0 ** -21) * size + (2.0 ** -11 if y_f16 else U) * np.abs(y) + (2.0 ** -25 if y_f16 else 0)
    if x.shape[0] > 16:
        tol = tol + 2.0 ** -10 * np.abs(x) @ np.abs(W).T + 2.0 ** -25 * np.abs(x).sum(1, keepdims=True)
    return y, tol


def check(got, want, tol, what):
    d = np.abs(got.astype(np.float64) - want)
    worst = float((d / np.maximum(tol, 1e-300)).max()) if d.size else 0.0
    print(f"[{what}] worst {worst:.3f} of the tolerance", flush=True)
    assert np.all(d <= tol), f"{what}: {np.count_nonzero(~(d <= tol))} of {d.size} outside"


def run(ctx, engine, x, w, xt, yt, stream=None):
    qt = w if isinstance(w, QuantizedTensor) else QuantizedTensor.affine4(ctx, *w)
    X = UnifiedTensor.new(ctx, x, dtype=KIND[xt][1])
    Y = UnifiedTensor.new(ctx, np.full((x.shape[0], qt.n_out), 7.0), dtype=KIND[yt][1])
    ctx.sync()
    engine.qmatmul(ctx, X, qt, Y, stream=stream.h if stream else None)
    if stream:
        stream.synchronize()
    return Y.to_vec()


def acts(g, m, k, t, std=1.0):
    return (g.standard_normal((m, k)) * std).astype(KIND[t][0])


@pytest.mark.parametrize("n,k,group", [(37, 256, 64), (16, 6, 2), (5, 30, 10), (130, 96, 32)])
@pytest.mark.parametrize("biases", [True, False])
def test_dequantize_bit_exact(ctx, engine, n, k, group, biases):
    g = np.random.default_rng(n)
    u, s, b, _ = w = weight(g, n, k, group, biases)
    out = UnifiedTensor.empty(ctx, [n, k])
    engine.dequantize_weight(ctx, QuantizedTensor.affine4(ctx, *w), out)
    rep = lambda a: np.repeat(a, group, axis=1)  # noqa: E731
    want = u.astype(np.float32) * rep(s) + (rep(b) if biases else np.float32(0))
    assert np.array_equal(out.to_vec(), want)


SHAPES = [(1, 2, 2), (7, 128, 128), (64, 256, 64), (257, 320, 32), (33, 1088, 64), (96, 4096, 64), (40, 2048, 128),
          (24, 11008, 32), (19, 16384, 128), (11, 20480, 64), (50, 360, 24), (3, 96, 96), (1000, 64, 64)]


@pytest.mark.parametrize("xt,yt", [("f16", "f16"), ("f32", "f32"), ("f16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("n,k,group", SHAPES, ids=lambda v: str(v))
def test_rows(ctx, engine, n, k, group, xt, yt):
    """1 to 16 rows and some more, every dtype, odd shapes and groups."""
    g = np.random.default_rng(n + k)
    w = weight(g, n, k, group)
    qt = QuantizedTensor.affine4(ctx, *w)
    for m in (1, 2, 3, 4, 5, 8, 9, 13, 16, 17, 40):
        x = acts(g, m, k, xt)
        want, tol = truth(x, w, yt == "f16")
        check(run(ctx, engine, x, qt, xt, yt), want, tol, f"{m}x{n}x{k}/{group} {xt}->{yt}")


@pytest.mark.parametrize("xt", ["f16", "f32"])
@pytest.mark.parametrize("n,k,group", SHAPES + [(4133, 320, 64), (9000, 256, 32), (16411, 128, 64), (37, 20480, 32),
                                                (4133, 17408, 32)], ids=lambda v: str(v))
def test_whole_numbers(ctx, engine, n, k, group, xt):
    """Activations, scales and biases of small whole numbers: every sum, in any
    order and with the codes offset by 16, stays a whole number below
    3 * 4 * 31 * 20480 < 2^24, so results are exact -- no element lost or taken twice."""
    g = np.random.default_rng(n + k + 7)
    u = g.integers(0, 16, (n, k), dtype=np.uint8)
    s = 2.0 ** g.integers(0, 3, (n, k // group)) * g.choice([-1, 1], (n, k // group))
    b = g.integers(-8, 9, s.shape).astype(np.float64)
    qt = QuantizedTensor.affine4(ctx, u, s, b, group)
    at = np.unique(g.integers(0, n, 200))
    W = u[at] * np.repeat(s[at], group, 1) + np.repeat(b[at], group, 1)
    for m in (1, 2, 3, 7, 8, 9, 15, 16, 18, 60):
        x = g.integers(-3, 4, (m, k)).astype(KIND[xt][0])
        got = run(ctx, engine, x, qt, xt, "f32")
        assert np.array_equal(got[:, at], x.astype(np.float64) @ W.T), m


@pytest.mark.parametrize("xt", ["f16", "f32"])
@pytest.mark.parametrize("n,k,group", [(4133, 320, 64), (9000, 256, 32), (16411, 128, 64), (37, 20480, 32),
                                       (4133, 17408, 32), (16411, 1056, 32)])
def test_tall_and_long(ctx, engine, n, k, group, xt):
    """Weights of many rows (two row tiles per block) and of more than 512
    groups per row; some rows of each are checked."""
    g = np.random.default_rng(n + k)
    u, s, b, _ = w = weight(g, n, k, group)
    qt = QuantizedTensor.affine4(ctx, *w)
    at = np.unique(np.concatenate([np.arange(40), n // 2 + np.arange(40), n - 1 - np.arange(40)]) % n)
    for m in (2, 3, 8, 9, 16, 18):
        x = acts(g, m, k, xt)
        want, tol = truth(x, (u[at], s[at], b[at], group), False)
        got = run(ctx, engine, x, qt, xt, "f32")
        assert np.isfinite(got).all() and np.count_nonzero(got == 7.0) <= 1
        check(got[:, at], want, tol, f"{m}x{n}x{k}/{group} {xt}")


@pytest.mark.parametrize("xt,yt", [("f16", "f16"), ("f32", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("m", [33, 130, 515])
@pytest.mark.parametrize("n,k,group", [(300, 512, 64), (129, 1088, 64), (72, 640, 128), (100, 512, 32)])
def test_prompts(ctx, engine, m, n, k, group, xt, yt):
    """Many rows, on the context's stream (codes widened to bytes where the
    8-bit GEMM serves the shape) and on a caller's."""
    g = np.random.default_rng(m + n)
    w = weight(g, n, k, group)
    qt = QuantizedTensor.affine4(ctx, *w)
    x = acts(g, m, k, xt)
    want, tol = truth(x, w, yt == "f16")
    check(run(ctx, engine, x, qt, xt, yt), want, tol, f"{m}x{n}x{k}/{group} {xt}->{yt}")
    check(run(ctx, engine, x, qt, xt, yt, Stream()), want, tol, f"stream {m}x{n}x{k}/{group} {xt}->{yt}")


@pytest.mark.parametrize("m", [1, 2, 7, 16, 33])
def test_without_biases(ctx, engine, m):
    g = np.random.default_rng(m)
    w = weight(g, 100, 512, 64, biases=False)
    x = acts(g, m, 512, "f16")
    want, tol = truth(x, w, False)
    check(run(ctx, engine, x, w, "f16", "f32"), want, tol, f"no biases m={m}")


@pytest.mark.parametrize("m", [1, 2, 3, 11, 16])
def test_f32_rows_keep_their_range(ctx, engine, m):
    """f32 rows past fp16's range, tiny ones, and both in one row."""
    g = np.random.default_rng(m + 40)
    w = weight(g, 70, 1024, 64)
    x = acts(g, m, 1024, "f32")
    x[0, :] *= 1e30
    x[-1, 512:] *= np.float32(1e6)
    want, tol = truth(x, w, False)
    check(run(ctx, engine, x, w, "f32", "f32"), want, tol, f"large m={m}")
    x = acts(g, m, 1024, "f32") * np.float32(1e-20 if m <= 2 else 6.2e-5)
    want, tol = truth(x, w, False)
    if m > 2:  # 3 to 16 rows keep fp16-subnormal precision below 6.1e-5
        tol = tol + 2.0 ** -24 * parts(w)[1].sum(1)
    check(run(ctx, engine, x, w, "f32", "f32"), want, tol, f"tiny m={m}")


@pytest.mark.parametrize("m", [1, 2, 5, 16, 20])
def test_misaligned(ctx, engine, m):
    """Codes and activations at odd addresses are served."""
    g = np.random.default_rng(m + 60)
    w = weight(g, 50, 256, 64)
    x = acts(g, m, 256, "f16")
    qt = QuantizedTensor.affine4(ctx, *w)
    raw = qt.codes.to_vec().ravel()
    codes = UnifiedTensor.new(ctx, np.concatenate([[0] * 3, raw]).astype(np.uint8), dtype=DType.U8)
    xs = UnifiedTensor.new(ctx, np.concatenate([[0], x.ravel()]).astype(np.float16), dtype=DType.FP16)
    Y = UnifiedTensor.empty(ctx, [m, 50], DType.FP32)
    odd = QuantizedTensor.from_affine4(UnifiedTensor(ctx, codes.ptr + 3, qt.codes.shape, DType.U8, owner=False),
                                       qt.scales, qt.biases, 64)
    engine.qmatmul(ctx, UnifiedTensor(ctx, xs.ptr + 2, x.shape, DType.FP16, owner=False), odd, Y)
    want, tol = truth(x, w, False)
    check(Y.to_vec(), want, tol, f"misaligned m={m}")


def test_degenerate_sizes(ctx, engine):
    g = np.random.default_rng(5)
    w = QuantizedTensor.affine4(ctx, *weight(g, 6, 64, 64))
    engine.qmatmul(ctx, UnifiedTensor.empty(ctx, [0, 64], DType.FP16), w, UnifiedTensor.empty(ctx, [0, 6], DType.FP16))
    empty = QuantizedTensor.affine4(ctx, np.zeros((5, 0), np.uint8), np.zeros((5, 0)), None)
    empty.scales = w.scales
    Y = UnifiedTensor.new(ctx, np.full((2, 5), 7.0), dtype=DType.FP16)
    engine.qmatmul(ctx, UnifiedTensor.empty(ctx, [2, 0], DType.FP16), empty, Y)
    assert np.all(Y.to_vec() == 0)


@pytest.mark.parametrize("m", [1, 4, 24, 130])
def test_streams_and_graphs(ctx, engine, m):
    g = np.random.default_rng(m + 80)
    w = weight(g, 300, 1024, 64)
    qt = QuantizedTensor.affine4(ctx, *w)
    x = acts(g, m, 1024, "f16")
    ref = run(ctx, engine, x, qt, "f16", "f32")
    want, tol = truth(x, w, False)
    check(run(ctx, engine, x, qt, "f16", "f32", Stream()), want, tol, f"stream m={m}")
    X = UnifiedTensor.new(ctx, x, dtype=DType.FP16)
    Y = UnifiedTensor.empty(ctx, [m, 300], DType.FP32)
    graph = Graph(ctx.stream, lambda: engine.qmatmul(ctx, X, qt, Y))
    for i in range(4):
        Y.zero_()
        graph.launch()
        assert np.array_equal(Y.to_vec(), ref)
        x2 = acts(g, m, 1024, "f16")
        new = UnifiedTensor.new(ctx, x2, dtype=DType.FP16)
        _lib.call("rq_memcpy_d2d", ctx.handle, X.ptr, new.ptr, X.nbytes, None)
        ref = run(ctx, engine, x2, qt, "f16", "f32")


@pytest.mark.parametrize("m", [1, 2, 6, 16, 40, 70])
@pytest.mark.parametrize("xt", ["f16", "f32"])
def test_mlp_and_lora(ctx, engine, m, xt):
    """The SwiGLU MLP and the LoRA linear over 4-bit weights."""
    g = np.random.default_rng(m + 100)
    H, I = 256, 448
    gate, up, down = weight(g, I, H, 64), weight(g, I, H, 64), weight(g, H, I, 64)
    x = acts(g, m, H, xt)
    Q = [QuantizedTensor.affine4(ctx, *w) for w in (gate, up, down)]
    X = UnifiedTensor.new(ctx, x, dtype=KIND[xt][1])
    Y = UnifiedTensor.empty(ctx, [m, H], DType.FP32)
    h = engine.mlp_swiglu(ctx, X, *Q, Y).to_vec().ravel()[:m * I].reshape(m, I)
    (a, ta), (b, tb) = truth(x, gate, True), truth(x, up, True)
    silu = a / (1 + np.exp(-a))
    # |silu'| < 1.1; g, u and h each rounded to fp16
    th = 1.1 * ta * (np.abs(b) + tb) + np.abs(silu) * tb + 2.0 ** -11 * np.abs(silu * b) * 1.01 + 2.0 ** -24
    check(h, silu * b, th, f"h m={m} {xt}")
    want, tol = truth(h, down, False)
    check(Y.to_vec(), want, tol, f"mlp m={m} {xt}")
    if m * I * 4 <= 8 << 20:
        Y2 = UnifiedTensor.empty(ctx, [m, H], DType.FP32)
        d = [w.descriptor() for w in Q]
        _lib.call("rq_mlp_swiglu_noalloc", ctx.handle, *(ctypes.byref(v) for v in d), X.ptr,
                  _lib.RQ_F16 if xt == "f16" else _lib.RQ_F32, Y2.ptr, _lib.RQ_F32, m, None)
        check(Y2.to_vec(), want, tol + np.abs(parts(down)[0]) .sum(1) * 2.0 ** -10 * np.abs(h).max(), f"noalloc m={m} {xt}")
    rank = 8
    A, B = acts(g, H, rank, "f32", H ** -0.5), acts(g, rank, I, "f32", 0.02)
    T = lambda v: UnifiedTensor.new(ctx, v, dtype=DType.FP32)  # noqa: E731
    for tree in (False, True):
        Z = UnifiedTensor.empty(ctx, [m, I], DType.FP32)
        engine.qmatmul_lora(ctx, X, Q[0], T(A), T(B), Z, tree=tree)
        base, tol = truth(x, gate, False)
        x64, A64, B64 = x.astype(np.float64), A.astype(np.float64), B.astype(np.float64)
        tol = tol + 2 * (H + rank + 8) * U * (np.abs(x64) @ np.abs(A64) @ np.abs(B64)) + 2 * U * np.abs(base)
        check(Z.to_vec(), base + x64 @ A64 @ B64, tol, f"lora m={m} {xt} tree={tree}")


def test_refusals(ctx, engine):
    g = np.random.default_rng(6)
    w = QuantizedTensor.affine4(ctx, *weight(g, 64, 128, 64))
    d = w.descriptor()
    lib = _lib.lib()
    assert lib.rq_qweight_prep_bytes(ctypes.byref(d)) == 0 and lib.rq_qweight_dx_table_bytes(ctypes.byref(d)) == 0
    dy, dx = UnifiedTensor.empty(ctx, [2, 64]), UnifiedTensor.empty(ctx, [2, 128])
    with pytest.raises(RqError, match="RQ_ERR_UNSUPPORTED"):
        engine.qmatmul_dx(ctx, dy, w, dx)
    X, Y = UnifiedTensor.empty(ctx, [1, 128], DType.FP16), UnifiedTensor.empty(ctx, [1, 64], DType.FP16)
    for field, value, err in (("group", 0, "INVALID"), ("group", 48, "SHAPE"), ("k_in", 127, "SHAPE"),
                              ("format", 3, "INVALID"), ("codes", None, "INVALID"), ("scales", None, "INVALID"),
                              ("prep", 4096, "INVALID")):
        bad = w.descriptor()
        setattr(bad, field, value)
        with pytest.raises(RqError, match=err):
            _lib.call("rq_qmatmul", ctx.handle, ctypes.byref(bad), X.ptr, 1, Y.ptr, 1, 1, None)
    for bad in ((np.zeros((2, 3), np.uint8), np.zeros((2, 1)), None, 3), (np.full((2, 64), 16), np.zeros((2, 1)), None, 64),
                (np.zeros((2, 64), np.uint8), np.zeros((2, 2)), None, 64)):
        with pytest.raises(ValueError):
            QuantizedTensor.affine4(ctx, *bad)
