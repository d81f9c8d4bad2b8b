"""rq_llama_verify: drafted trees through the Llama runner in one pass, against its
own decode steps (the tokens) and the float64 oracle (the logits, to 1e-2 of
their largest as for the decode steps: fp16 activations and cache)."""
import numpy as np
import pytest

from oracle import llama as ol
from rusty_amd import RqError
from rusty_amd.llama import LlamaConfig, LlamaRunner, synth_weights

pytestmark = pytest.mark.gpu

TINY = LlamaConfig(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, intermediate=512, vocab=1000,
                   max_seq=96)

DRAFT_CFGS = [TINY, LlamaConfig(n_layers=2, hidden=512, n_heads=4, n_kv_heads=1, head_dim=128, intermediate=384,
                                vocab=777, max_seq=200)]


def _greedy(ctx, cfg, w, prompt, steps):
    r = LlamaRunner(ctx, cfg, w)
    r.prefill(prompt)
    r.decode(steps)
    toks = r.tokens()
    r.close()
    return toks


@pytest.mark.parametrize("cfg", DRAFT_CFGS, ids=["gqa2_hd64", "mqa_hd128"])
@pytest.mark.parametrize("group", [0, 64])
def test_verify_follows_the_greedy_path(ctx, cfg, group):
    """Trees that hold the greedy continuation among wrong drafts: as many
    drafts are followed as they hold, the sequence is the decode steps', and
    the cache serves the steps after it."""
    w = synth_weights(cfg, seed=5, affine_group=group)
    prompt = np.random.default_rng(21).integers(0, cfg.vocab, 33)
    want = _greedy(ctx, cfg, w, prompt, 40)
    wrong = lambda t, k=1: int((t + k) % cfg.vocab)  # noqa: E731
    r = LlamaRunner(ctx, cfg, w)
    r.prefill(prompt)
    n = 34  # tokens of the sequence (one of them not cached yet)
    nxt = lambda i: int(want[n + i])  # noqa: E731
    # no drafts: one decode step
    assert r.verify([], []) == 0
    n += 1
    # a chain, all right
    assert r.verify([nxt(0), nxt(1), nxt(2)], [-1, 0, 1]) == 3
    n += 4
    # a tree in breadth-first order: wrong siblings, the right path 1 -> 3 -> 6
    t = [wrong(nxt(0)), nxt(0), wrong(nxt(1)), nxt(1), wrong(nxt(2)), wrong(nxt(2), 2), nxt(2), wrong(nxt(3))]
    assert r.verify(t, [-1, -1, 1, 1, 0, 3, 3, 6]) == 3
    n += 4
    # nothing right; a right token under a wrong one does not count
    assert r.verify([wrong(nxt(0)), nxt(1), wrong(nxt(0), 2)], [-1, 0, -1]) == 0
    n += 1
    # two equal drafts: the first one's children are followed
    assert r.verify([nxt(0), nxt(0), wrong(nxt(1)), nxt(1)], [-1, -1, 0, 1]) == 1
    n += 2
    # 17 rows and more take the prefill products
    t, p = [nxt(0)], [-1]
    for i in range(1, 20):
        t.append(nxt(1) if i == 15 else wrong(nxt(1), i))
        p.append(0)
    assert r.verify(t, p) == 2
    n += 3
    r.decode(5)
    n += 5
    got = r.tokens()
    assert got.shape == (n,)
    np.testing.assert_array_equal(got, want[:n])
    r.close()


def test_verify_logits_and_capacity(ctx):
    """The last followed row's logits match the oracle's; a pass may fill the
    cache to its end and no further, and refused calls change nothing."""
    cfg = TINY
    w = synth_weights(cfg, seed=9)
    prompt = np.random.default_rng(3).integers(0, cfg.vocab, 50)
    want = _greedy(ctx, cfg, w, prompt, 46)
    r = LlamaRunner(ctx, cfg, w)
    with pytest.raises(RqError, match="no sequence"):
        r.verify([1], [-1])
    r.prefill(prompt)
    for bad, match in ((([cfg.vocab], [-1]), "vocabulary"), (([-1], [-1]), "vocabulary"), (([1], [0]), "no earlier"),
                       (([1, 2], [-1, 1]), "no earlier"), (([1], [-2]), "no earlier"),
                       (([1] * 64, list(range(-1, 63))), "outside 0..63"), (([1] * 46, [-1] * 46), "exceed")):
        with pytest.raises(RqError, match=match):
            r.verify(*bad)
    with pytest.raises(ValueError):
        r.verify([1, 2], [-1])
    np.testing.assert_array_equal(r.tokens(), want[:51])
    logits, n = [r.logits()], 51
    for k in (3, 0, 7, 20):
        a = r.verify(want[n:n + k], list(range(-1, k - 1)))
        assert a == k
        n += k + 1
        logits.append(r.logits())
    # 84 + ... positions are cached; fill the rest with one chain
    left = cfg.max_seq - (n - 1)
    assert r.verify(want[n:n + left - 1], list(range(-1, left - 2))) == left - 1
    np.testing.assert_array_equal(r.tokens(), want)
    with pytest.raises(RqError, match="RQ_ERR_SHAPE"):
        r.verify([], [])
    ref = ol.forward(cfg, w, want[:n - 1], first=49)
    for i, lg in zip([0, 4, 5, 13, 34], logits):
        scale = np.abs(ref[i]).max()
        assert np.abs(lg - ref[i]).max() <= 1e-2 * scale
    # a new prompt starts over
    r.prefill(prompt)
    assert r.verify([int(want[51])], [-1]) == 1
    r.close()


def test_verify_on_another_stream(ctx):
    from rusty_amd.hiprt import Stream

    cfg = TINY
    w = synth_weights(cfg, seed=13)
    prompt = np.random.default_rng(4).integers(0, cfg.vocab, 20)
    want = _greedy(ctx, cfg, w, prompt, 12)
    r = LlamaRunner(ctx, cfg, w)
    s = Stream()
    r.prefill(prompt, stream=s.h)
    assert r.verify(want[21:25], [-1, 0, 1, 2], stream=s.h) == 4
    r.decode(3, stream=s.h)
    np.testing.assert_array_equal(r.tokens(stream=s.h), want[:29])
    r.close()
