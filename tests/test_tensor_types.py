"""The element type that UnifiedTensor.new takes for an array without one named
(host side only: the device calls are recorded, none is made)."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest

from rusty_amd import DType, UnifiedTensor, engine


@pytest.fixture
def copies(monkeypatch):
    """What reaches the device, as bytes."""
    seen = []

    def call(name, *args):
        if name == "rq_memcpy_h2d":
            seen.append(ctypes.string_at(args[2], args[3]))

    monkeypatch.setattr(engine, "call", call)
    return seen


CTX = SimpleNamespace(handle=None)


@pytest.mark.parametrize("np_t", [np.float32, np.float16, np.int8, np.uint8, np.uint32])
def test_kept(copies, np_t):
    a = np.arange(6).astype(np_t).reshape(2, 3)
    t = UnifiedTensor.new(CTX, a)
    assert t.dtype.np == a.dtype and t.shape == (2, 3) and copies == [a.tobytes()]


@pytest.mark.parametrize("np_t", [np.float64, np.int32, np.int64, np.uint64, np.int16, np.bool_])
def test_widened_to_f32(copies, np_t):
    """Every other type is a list of numbers: FP32, whatever element types buffers may have by name."""
    a = np.array([0, 1, 1, 0], dtype=np_t)
    assert UnifiedTensor.new(CTX, a).dtype is DType.FP32 and copies == [a.astype(np.float32).tobytes()]
    assert UnifiedTensor.new(CTX, a.tolist()).dtype is DType.FP32


@pytest.mark.parametrize("kind", list(DType))
def test_named(copies, kind):
    a = np.array([3, 0, 7])
    t = UnifiedTensor.new(CTX, a, dtype=kind)
    assert t.dtype is kind and t.nbytes == 3 * kind.itemsize and copies == [a.astype(kind.np).tobytes()]
