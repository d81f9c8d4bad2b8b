"""rq_llama_verify that fails on its way, at each step at which a launch or a copy
may: the sequence is as it was, for the decode steps, further passes and the read-outs."""
import ctypes

import numpy as np
import pytest
from test_gpu_verify import DRAFT_CFGS, TINY, _greedy

from rusty_amd import RqError, _lib
from rusty_amd.llama import LlamaRunner, synth_weights

pytestmark = pytest.mark.gpu

STEPS = {"upload": 1, "last token": 2, "pass": 3, "copy back": 4, "commit": 5}


@pytest.fixture
def fail_at():
    fn = _lib.lib().rusty_verify_fail_at
    fn.argtypes, fn.restype = [ctypes.c_int], None
    yield fn
    fn(0)


@pytest.mark.parametrize("step", list(STEPS))
@pytest.mark.parametrize("cfg", DRAFT_CFGS, ids=["gqa2_hd64", "mqa_hd128"])
def test_sequence_stays(ctx, fail_at, cfg, step):
    w = synth_weights(cfg, seed=7)
    prompt = np.random.default_rng(2).integers(0, cfg.vocab, 21)
    want = _greedy(ctx, cfg, w, prompt, 24)
    r = LlamaRunner(ctx, cfg, w)
    r.prefill(prompt)
    n, logits = 22, r.logits()

    def fails():
        # a tree whose right path is not in order, so that cache rows would move
        right = [int(t) for t in want[n:n + 3]]
        tokens = [(right[0] + 1) % cfg.vocab, right[0], (right[1] + 1) % cfg.vocab, right[1], right[2]]
        fail_at(STEPS[step])
        with pytest.raises(RqError, match="RQ_ERR_HIP"):
            r.verify(tokens, [-1, -1, 1, 1, 3])
        fail_at(0)
        np.testing.assert_array_equal(r.tokens(), want[:n])
        np.testing.assert_array_equal(r.logits(), logits)

    fails()
    r.decode(4)  # the steps continue from the same token and position
    n, logits = n + 4, r.logits()
    np.testing.assert_array_equal(r.tokens(), want[:n])
    fails()
    assert r.verify(want[n:n + 3], [-1, 0, 1]) == 3
    n += 4
    r.decode(2)
    np.testing.assert_array_equal(r.tokens(), want[:n + 2])
    r.close()


def test_first_call_fails(ctx, fail_at):
    """An error of the first call, which allocates."""
    w = synth_weights(TINY, seed=8)
    prompt = np.random.default_rng(5).integers(0, TINY.vocab, 9)
    want = _greedy(ctx, TINY, w, prompt, 8)
    for step in STEPS.values():
        r = LlamaRunner(ctx, TINY, w)
        r.prefill(prompt)
        fail_at(step)
        with pytest.raises(RqError):
            r.verify(want[10:12], [-1, 0])
        fail_at(0)
        assert r.verify(want[10:12], [-1, 0]) == 2
        np.testing.assert_array_equal(r.tokens(), want[:13])
        r.close()
