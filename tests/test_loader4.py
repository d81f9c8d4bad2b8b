"""4-bit MLX affine safetensors (rusty_amd/loader.py): the packing on the host,
and a checkpoint's Linear through upload_quantized on the device."""
import numpy as np
import pytest

from rusty_amd.loader import LoaderError, QuantizationConfig, WeightsContext, save_safetensors

Q4 = QuantizationConfig(64, 4, "affine")


def write(path, n=6, k=128, group=64, seed=0, sdt="F16"):
    g = np.random.default_rng(seed)
    u = g.integers(0, 16, (n, k), dtype=np.uint32)
    words = np.zeros((n, k // 8), np.uint32)
    for j in range(8):  # element 8 i + j in bits 4 j .. 4 j + 3 of word i
        words |= u[:, j::8] << np.uint32(4 * j)
    s = g.uniform(0.001, 0.02, (n, k // group)).astype(np.float16)
    b = (-7.5 * s).astype(np.float16)
    if sdt == "BF16":
        enc = lambda a: (a.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)  # noqa: E731
        dec = lambda a: (enc(a).astype(np.uint32) << 16).view(np.float32)  # noqa: E731
    else:
        enc = dec = lambda a: a  # noqa: E731
    save_safetensors(path, {"w.weight": ("U32", words), "w.scales": (sdt, enc(s)), "w.biases": (sdt, enc(b))})
    return u.astype(np.uint8), dec(s).astype(np.float32), dec(b).astype(np.float32)


@pytest.mark.parametrize("sdt", ["F16", "BF16"])
def test_packing(tmp_path, sdt):
    u, s, b = write(tmp_path / "m.safetensors", sdt=sdt)
    wc = WeightsContext()
    wc.load_file(tmp_path / "m.safetensors")
    codes, got_s, got_b = wc._quantized4_host("w", Q4)
    assert codes.shape == (6, 64)
    assert np.array_equal(codes & 15, u[:, 0::2]) and np.array_equal(codes >> 4, u[:, 1::2])
    assert np.array_equal(got_s, s) and np.array_equal(got_b, b)


def test_errors(tmp_path):
    write(tmp_path / "m.safetensors")
    wc = WeightsContext()
    wc.load_file(tmp_path / "m.safetensors")
    with pytest.raises(LoaderError, match="not a multiple"):
        wc._quantized4_host("w", QuantizationConfig(48, 4, "affine"))
    with pytest.raises(LoaderError, match="expected 24"):
        wc._quantized4_host("w", QuantizationConfig(32, 4, "affine"))
    with pytest.raises(LoaderError, match="expected 4-bit"):
        wc._quantized4_host("w", QuantizationConfig(64, 8, "affine"))
    with pytest.raises(LoaderError, match="Weight not found"):
        wc._quantized4_host("x", Q4)


@pytest.mark.gpu
def test_upload_and_multiply(ctx, engine, tmp_path):
    from rusty_amd import DType, UnifiedTensor, _lib

    u, s, b = write(tmp_path / "m.safetensors", n=40, k=256, seed=3)
    wc = WeightsContext()
    wc.load_file(tmp_path / "m.safetensors")
    w = wc.upload_quantized("w", ctx, Q4)
    assert (w.n_out, w.k_in, w.format, w.group) == (40, 256, _lib.RQ_Q_AFFINE_U4, 64)
    W = u * np.repeat(s, 64, 1).astype(np.float64) + np.repeat(b, 64, 1)
    dense = wc.upload_dequantized("w", ctx, Q4).to_vec()
    # one rounding of the product, one of the sum
    assert np.all(np.abs(dense - W) <= 2.0 ** -23 * (np.abs(W) + np.abs(np.repeat(b, 64, 1))))
    x = np.random.default_rng(1).standard_normal((3, 256)).astype(np.float32)
    Y = UnifiedTensor.empty(ctx, [3, 40])
    engine.qmatmul(ctx, UnifiedTensor.new(ctx, x), w, Y)
    # f32 sums of 256 terms of at most |x| (|s| 47 + |b|), two fp16 terms of x (2^-21)
    size = np.abs(x) @ (np.repeat(s, 64, 1) * (u + 32.0) + np.abs(np.repeat(b, 64, 1))).T
    assert np.all(np.abs(Y.to_vec() - x.astype(np.float64) @ W.T) <= (72 * 2.0 ** -24 + 2.0 ** -21) * size)
