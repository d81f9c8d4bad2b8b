"""Sizes at the ends of the attention entry points' ranges (host arithmetic, no device)."""
import ctypes

from test_attn_args import SHAPE, attn, tree

from rusty_amd import _lib


def test_positions_round_up_below_2_31():
    """The kernels count a cache's positions in tiles with 32 bits: capacities that would wrap are refused."""
    most = 0x7fffffff - 1024
    fn = _lib.lib().rq_attn_tree_workspace
    a = attn(1, 1)
    for cap in (most + 1, 0x7fffffff):
        assert tree(a, n_seqs=1, capacity=cap, strides=(0, 0, 64)) == SHAPE
        assert fn(ctypes.byref(a), 1, 1, 1, cap) == 0
    assert tree(a, n_seqs=1, capacity=most, strides=(0, 0, 64)) == 0 and fn(ctypes.byref(a), 1, 1, 1, most) > 0
