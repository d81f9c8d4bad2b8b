"""4-bit Linears whose group size neither divides a kernel's batch of 256 k nor is
a multiple of it: each element meets the scale and bias of its own group.
Tolerances as in test_gpu_linear4.py, without its fp16 term: every row here
goes 16 at a time with exact codes, or is a whole number."""
import numpy as np
import pytest
from test_gpu_linear4 import KIND, acts, check, run, truth, weight

from rusty_amd import DType, QuantizedTensor, UnifiedTensor
from rusty_amd.hiprt import Stream

pytestmark = pytest.mark.gpu

GROUPS = [(40, 960, 96), (24, 1600, 160), (40, 1920, 192), (70, 672, 224), (33, 2560, 320), (24, 3840, 384),
          (300, 1280, 640), (4133, 480, 96), (9, 1056, 1056), (11, 49920, 96), (19, 20480, 160)]


@pytest.mark.parametrize("xt", ["f16", "f32"])
@pytest.mark.parametrize("n,k,group", GROUPS, ids=lambda v: str(v))
def test_whole_numbers(ctx, engine, n, k, group, xt):
    """Scales of 1, 2 and 4 with either sign, biases to 8 and activations of -1, 0 and 1: the kernels' terms,
    s (16 + u) x and (b - 16 s) x, are whole and add to at most 49920 (124 + 72) < 2^24, exact in any order,
    so one element with a neighbour's scale shows.  (Past 48 rows the weights, of at most 68, are exact in fp16 too.)"""
    g = np.random.default_rng(n + k + group)
    u = g.integers(0, 16, (n, k), dtype=np.uint8)
    s = 2.0 ** g.integers(0, 3, (n, k // group)) * g.choice([-1, 1], (n, k // group))
    b = g.integers(-8, 9, s.shape).astype(np.float64)
    qt = QuantizedTensor.affine4(ctx, u, s, b, group)
    at = np.unique(g.integers(0, n, 200))
    W = u[at] * np.repeat(s[at], group, 1) + np.repeat(b[at], group, 1)
    for m in (1, 2, 3, 8, 9, 16, 18, 60):
        x = g.integers(-1, 2, (m, k)).astype(KIND[xt][0])
        got = run(ctx, engine, x, qt, xt, "f32")
        assert np.array_equal(got[:, at], x.astype(np.float64) @ W.T), m
        if m == 60:  # a caller's stream: 16 rows at a time
            got = run(ctx, engine, x, qt, xt, "f32", Stream())
            assert np.array_equal(got[:, at], x.astype(np.float64) @ W.T), "stream"


@pytest.mark.parametrize("xt,yt", [("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("n,k,group", GROUPS[:8], ids=lambda v: str(v))
def test_rows(ctx, engine, n, k, group, xt, yt):
    g = np.random.default_rng(n + k)
    w = weight(g, n, k, group)
    qt = QuantizedTensor.affine4(ctx, *w)
    for m in (3, 8, 9, 16):
        x = acts(g, m, k, xt)
        want, tol = truth(x, w, yt == "f16")
        check(run(ctx, engine, x, qt, xt, yt), want, tol, f"{m}x{n}x{k}/{group} {xt}->{yt}")


@pytest.mark.parametrize("m", [5, 16, 33])
def test_mlp_and_lora(ctx, engine, m):
    """The forms over these Linears: whole numbers through the LoRA Linear (exact), the MLP's h."""
    g = np.random.default_rng(m)
    H, I, group = 480, 288, 96
    gate, up = weight(g, I, H, group), weight(g, I, H, group)
    down = weight(g, H, I, group)
    x = acts(g, m, H, "f16")
    Q = [QuantizedTensor.affine4(ctx, *w) for w in (gate, up, down)]
    X = UnifiedTensor.new(ctx, x, dtype=DType.FP16)
    Y = UnifiedTensor.empty(ctx, [m, H], DType.FP32)
    h = engine.mlp_swiglu(ctx, X, *Q, Y).to_vec().ravel()[:m * I].reshape(m, I)
    parts = [truth(x[i:i + 16], w, True) for i in range(0, m, 16) for w in (gate, up)]
    (a, ta), (b, tb) = ([np.concatenate(p) for p in zip(*parts[i::2])] for i in (0, 1))
    silu = a / (1 + np.exp(-a))
    th = 1.1 * ta * (np.abs(b) + tb) + np.abs(silu) * tb + 2.0 ** -11 * np.abs(silu * b) * 1.01 + 2.0 ** -24
    check(h, silu * b, th, f"h m={m}")
    u, s = g.integers(0, 16, (I, H), dtype=np.uint8), 2.0 ** g.integers(0, 3, (I, H // group))
    qt = QuantizedTensor.affine4(ctx, u, s, None, group)
    A, B = g.integers(-1, 2, (H, 4)).astype(np.float32), g.integers(-1, 2, (4, I)).astype(np.float32)
    xi = g.integers(-1, 2, (m, H)).astype(np.float16)
    Z = UnifiedTensor.empty(ctx, [m, I], DType.FP32)
    T = lambda v, d=DType.FP32: UnifiedTensor.new(ctx, v, dtype=d)  # noqa: E731
    engine.qmatmul_lora(ctx, T(xi, DType.FP16), qt, T(A), T(B), Z)
    x64 = xi.astype(np.float64)
    assert np.array_equal(Z.to_vec(), x64 @ (u * np.repeat(s, group, 1)).T + x64 @ A.astype(np.float64) @ B)
