"""The SwiGLU MLP whose three Linears have different formats, one of them 4-bit, at
sizes whose halves of the workspace start anywhere.

Activations of -1, 0 and 1 and whole weights of at most 8: gate and up are whole numbers below
2048, exact in every kernel and in fp16.  h = silu(g) u is rounded to fp16 once: half a step, 2^-11 of it
(at least 2^-25), and 2^-20 for the exponential and its f32 steps.  y adds I products of h in f32 with
codes that carry an offset d (16 with 4 bits, up to 1152 with 8, gemv_decode.hip) and takes d sum h away again:
partial sums of at most sum |h| (|w| + 2 d), I roundings of them, and one of y.
"""
import itertools

import numpy as np
import pytest

from rusty_amd import DType, QuantizedTensor, UnifiedTensor

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def linear(ctx, g, kind, n, k):
    """(weight, its whole values)"""
    if kind == "i8":
        q = g.integers(-8, 9, (n, k), dtype=np.int8)
        return QuantizedTensor.rowwise(ctx, q, np.ones(n)), q.astype(np.float64)
    group = 32 if kind == "u4" else 16
    u = g.integers(0, 16, (n, k), dtype=np.uint8)
    group = group if k % group == 0 else 2
    s, b = np.ones((n, k // group), np.float32), np.full((n, k // group), -8, np.float32)
    make = QuantizedTensor.affine4 if kind == "u4" else QuantizedTensor.affine
    return make(ctx, u, s, b, group), u - 8.0


@pytest.mark.parametrize("xt", [DType.FP16, DType.FP32], ids=["f16", "f32"])
@pytest.mark.parametrize("m", [1, 2, 5, 16, 17, 51])
@pytest.mark.parametrize("H,I", [(64, 50), (128, 96), (96, 34)])
def test_mlp(ctx, engine, H, I, m, xt):
    for kinds in itertools.product(("u4", "u8", "i8"), repeat=3):
        if "u4" not in kinds:
            continue
        g = np.random.default_rng(m + H)
        (gate, G), (up, P), (down, D) = (linear(ctx, g, k, *s) for k, s in zip(kinds, ((I, H), (I, H), (H, I))))
        x = g.integers(-1, 2, (m, H)).astype(np.float64)
        X = UnifiedTensor.new(ctx, x, dtype=xt)
        Y = UnifiedTensor.empty(ctx, [m, H], DType.FP32)
        h = engine.mlp_swiglu(ctx, X, gate, up, down, Y).to_vec().ravel()[:m * I].reshape(m, I).astype(np.float64)
        a, b = x @ G.T, x @ P.T
        assert np.abs(a).max() < 2048 and np.abs(b).max() < 2048
        want = a / (1 + np.exp(-a)) * b
        assert np.all(np.abs(h - want) <= (2.0 ** -11 + 2.0 ** -20) * np.abs(want) + 2.0 ** -25), kinds
        y, d = h @ D.T, 16 if kinds[2] == "u4" else 1152
        assert np.all(np.abs(Y.to_vec() - y) <= I * U * (np.abs(h) @ (np.abs(D) + 2 * d).T) + U * np.abs(y)), kinds
