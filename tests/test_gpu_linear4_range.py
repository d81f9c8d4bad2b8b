"""4-bit Linears at the ends of their types' range.

Tolerance as in test_gpu_linear4.py without its fp16 term, |dy| <= ((K / 32 +
64) u + 2^-21) S and half a step of the output: the two fp16 terms of an f32
activation are it to 2^-22, or where the row's largest magnitude in the 256 k
is 1 or more (or else scaled to 2^14 and more) to 2^-25 of that, half the
spacing of fp16's subnormals: 2^-25 of the largest times the weights' sizes.
"""
import numpy as np
import pytest
from test_gpu_linear4 import KIND, U, acts, check, parts, run, truth, weight

from rusty_amd import DType, QuantizedTensor, UnifiedTensor
from rusty_amd.hiprt import Stream

pytestmark = pytest.mark.gpu


def tight(x, w, y_f16):
    """truth() of 16 rows at a time: exact codes, f32 rows as two terms."""
    p = [truth(x[i:i + 16], w, y_f16) for i in range(0, len(x), 16)]
    return np.concatenate([a for a, _ in p]), np.concatenate([b for _, b in p])


def peaks(x, S):
    """sum over k of S[n, k] times the largest |x| of the row in the 256 k around k."""
    out = np.zeros((x.shape[0], S.shape[0]))
    for k in range(0, x.shape[1], 256):
        out += np.abs(x[:, k:k + 256]).max(1, keepdims=True).astype(np.float64) * S[:, k:k + 256].sum(1)
    return out


@pytest.mark.parametrize("std", [1.0, 0.3, 1e-2, 1e-3, 1e-4, 1e-6, 1e-20, 1e-37])
@pytest.mark.parametrize("n,k,group", [(70, 1024, 64), (19, 20480, 128), (600, 320, 32)], ids=lambda v: str(v))
def test_small_f32_rows(ctx, engine, n, k, group, std):
    """f32 rows of any magnitude keep f32 accuracy in 1 to 48 rows: the error is relative to the row."""
    g = np.random.default_rng(k)
    w = weight(g, n, k, group)
    qt = QuantizedTensor.affine4(ctx, *w)
    S = parts(w)[1]
    for m in (1, 2, 3, 8, 9, 16, 17, 40):
        x = acts(g, m, k, "f32", std)
        want, tol = tight(x, w, False)
        tol = tol + 2.0 ** -25 * peaks(x, S) + 2.0 ** -149 * k
        check(run(ctx, engine, x, qt, "f32", "f32"), want, tol, f"std {std} {m}x{n}x{k}")


@pytest.mark.parametrize("m", [1, 2, 3, 8, 13, 16])
def test_small_rows_typical_error(ctx, engine, m):
    """The rms error relative to the rms of S x: f32 rounding of K / 32 sums and 2^-22 of the activations stay below
    2^-20 of the typical size at any magnitude (a row rounded to fp16's subnormals: 1e-5 and more at 1e-3)."""
    g = np.random.default_rng(m + 9)
    w = weight(g, 96, 2048, 64)
    qt = QuantizedTensor.affine4(ctx, *w)
    S = parts(w)[1]
    for std in (1.0, 1e-2, 1e-3, 1e-4, 1e-5):
        x = acts(g, m, 2048, "f32", std)
        want, _ = tight(x, w, False)
        err = run(ctx, engine, x, qt, "f32", "f32") - want
        size = np.sqrt((x.astype(np.float64) ** 2) @ (S ** 2).T)
        r = float(np.sqrt((err ** 2).mean()) / np.sqrt((size ** 2).mean()))
        print(f"[m {m} std {std}] rms {r:.2e}", flush=True)
        assert r < 2.0 ** -20


@pytest.mark.parametrize("m", [1, 2, 3, 8, 9, 16, 33])
@pytest.mark.parametrize("xt", ["f16", "f32"])
def test_tiny_fp16_rows(ctx, engine, m, xt):
    """Values of fp16's subnormals are exact activations, in either type."""
    g = np.random.default_rng(m + 21)
    w = weight(g, 40, 512, 64)
    x = (g.integers(-64, 65, (m, 512)) * 2.0 ** -24).astype(KIND[xt][0])
    want, tol = tight(x, w, False)
    check(run(ctx, engine, x, w, xt, "f32"), want, tol, f"subnormal m={m} {xt}")


@pytest.mark.parametrize("xt,yt", [("f16", "f16"), ("f32", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("n,k,group", [(300, 512, 64), (72, 640, 128), (100, 512, 32)], ids=lambda v: str(v))
def test_sixteen_at_a_time(ctx, engine, n, k, group, xt, yt):
    """17 to 48 rows, and any number on a caller's stream or in groups of 32, keep the codes exact."""
    g = np.random.default_rng(n + k)
    w = weight(g, n, k, group)
    qt = QuantizedTensor.affine4(ctx, *w)
    for m, stream in ((17, None), (33, None), (48, None), (49, Stream()), (130, Stream())) + (((130, None),) if group == 32 else ()):
        x = acts(g, m, k, xt)
        want, tol = tight(x, w, yt == "f16")
        check(run(ctx, engine, x, qt, xt, yt, stream), want, tol, f"{m}x{n}x{k}/{group} {xt}->{yt}")


@pytest.mark.parametrize("m", [1, 2, 3, 8, 9, 16, 33])
@pytest.mark.parametrize("big", [1e36, 1e37])
def test_sums_that_fit_while_their_parts_do_not(ctx, engine, m, big):
    """f32 rows whose products with 16 + u pass f32's range though the result does not."""
    g = np.random.default_rng(m)
    w = weight(g, 48, 512, 64)
    x = np.clip(acts(g, m, 512, "f32"), -3, 3) * np.float32(big)
    want, tol = tight(x, w, False)
    assert np.abs(want).max() < 1e38
    check(run(ctx, engine, x, w, "f32", "f32"), want, tol, f"{big} m={m}")


@pytest.mark.parametrize("m", [1, 2, 3, 8, 9, 16, 20, 60])
@pytest.mark.parametrize("xt", ["f16", "f32"])
@pytest.mark.parametrize("n,k,group", [(37, 320, 32), (300, 512, 64), (20, 20480, 64), (50, 360, 24)], ids=lambda v: str(v))
def test_infinities_and_nan(ctx, engine, n, k, group, m, xt):
    """An infinite activation gives the infinity of x w, whatever the other terms; NaN, and infinities of both signs or
    against a zero weight, give NaN (f32 rows of the 8-bit GEMM all NaN); other rows keep their values."""
    g = np.random.default_rng(n + m)
    u, s, b, _ = w = weight(g, n, k, group)
    s[:, 0], b[:, 0], u[3, 2] = 2.0 ** -6, -2.0 ** -4, 4  # W[3, 2] = 0
    u[:, 1] |= 8
    x = acts(g, m, k, xt)
    x[0, k - 1] = np.inf
    if m > 2:
        x[1, 5], x[2, 2] = np.nan, -np.inf
    if m > 8:
        x[7, 1], x[7, 0], x[8, 1] = np.inf, 0.0, -np.inf
    W = parts(w)[0]
    with np.errstate(invalid="ignore"):
        want = np.stack([(x[i].astype(np.float64) * W).sum(1) for i in range(m)])
    for stream in (None, Stream()) if m in (3, 60) else (None,):
        got = run(ctx, engine, x, w, xt, "f32", stream).astype(np.float64)
        if m > 48 and group % 64 == 0 and xt == "f32" and stream is None:
            assert np.isnan(got[~np.isfinite(want)]).all()  # the 8-bit GEMM scales f32 rows by their largest value
        else:
            assert np.array_equal(np.isnan(got), np.isnan(want))
            assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
        ok = np.isfinite(want).all(1)
        if ok.any():
            ref, tol = truth(x[ok], w, False) if m > 48 else tight(x[ok], w, False)
            if m > 48:  # (the fp16 term of truth() past 16 rows)
                tol = tol + 2.0 ** -10 * np.abs(x[ok].astype(np.float64)) @ np.abs(W).T
            check(got[ok], ref, tol, f"beside {m}x{n}x{k} {xt}")


@pytest.mark.parametrize("m", [1, 2, 6, 16, 40])
@pytest.mark.parametrize("sign", [-1, 1])
def test_mlp_of_a_saturated_gate(ctx, engine, m, sign):
    """A gate past fp16's range: silu of a large negative one is 0, of a large positive one infinite in fp16."""
    g = np.random.default_rng(m)
    H, I = 256, 64
    one = np.ones((I, H // 64), np.float32)
    gate = (np.full((I, H), 8, np.uint8), sign * 50 * one, None, 64)
    up = (np.full((I, H), 8, np.uint8), 1e-3 * one, None, 64)
    down = weight(g, H, I, 64)
    X = UnifiedTensor.new(ctx, np.ones((m, H)), dtype=DType.FP16)
    Y = UnifiedTensor.empty(ctx, [m, H], DType.FP32)
    h = engine.mlp_swiglu(ctx, X, *[QuantizedTensor.affine4(ctx, *w) for w in (gate, up, down)], Y)
    h = h.to_vec().ravel()[:m * I].astype(np.float64)
    assert np.all(h == (np.inf if sign > 0 else 0.0))
    if sign < 0:
        assert np.all(Y.to_vec() == 0)
