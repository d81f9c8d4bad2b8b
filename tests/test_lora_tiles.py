"""Which products add their rows' adapters in their own tiles: by the set's rank and number of adapters, too."""
import ctypes

import pytest

from rusty_amd import _lib


def tile(m, n, k, rank, adapters, affine=False):
    f = _lib.lib().rusty_gemm_lora_tile
    f.argtypes, f.restype = [ctypes.c_int] + [ctypes.c_int64] * 3 + [ctypes.c_int] + [ctypes.c_int64] * 2, ctypes.c_int
    return f(int(affine), m, n, k, 256, rank, adapters)


def test_few_turns_of_the_adapters():
    assert [tile(2048, 4096, 4096, r, 4) for r in (4, 16, 64, 128)] == [128256] * 4
    assert tile(1024, 4096, 4096, 16, 4) == 128128 and tile(2048, 4096, 4096, 16, 64) == 128256


def test_many_turns_of_the_adapters():
    """Ranks and adapters that the tiles would take one after another for longer than a pass of their own."""
    assert [tile(2048, 2560, 2048, 256, a) for a in (4, 16, 64, 10 ** 9)] == [-1] * 4
    assert [tile(2048, 4096, 4096, r, 64) for r in (64, 128, 256)] == [-1] * 3
    assert [tile(1024, 4096, 4096, r, 64) for r in (16, 64, 256)] == [-1] * 3


@pytest.mark.parametrize("affine", [False, True])
def test_more_never_brings_the_tiles_back(affine):
    for m, n, k in ((2048, 4096, 4096), (300, 11008, 4096), (5000, 1024, 512), (1100, 5640, 192), (128, 65536, 64)):
        for set_of in (lambda i: (i, 4), lambda i: (32, i)):
            chosen = [tile(m, n, k, *set_of(i), affine) > 0 for i in (1, 2, 4, 8, 16, 32, 64, 128, 256)]
            assert chosen == sorted(chosen, reverse=True)
