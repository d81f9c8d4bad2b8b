"""A batch of requests as a serving program runs it: prompts packed through one
attention layer into a paged cache, then decode steps of one token per request, each
request with its adapter (or none).  Every stage is checked against 64 bits on what the
stage before it left, with the tolerances of that operator's own tests; the decode
step is then captured and replayed."""
import numpy as np
import pytest

from rusty_amd import DType, LoraSet, PagedCache, QuantizedTensor, Rope, UnifiedTensor
from rusty_amd._lib import call
from rusty_amd.hiprt import Graph, Stream
from test_gpu_attn import check as check_attn
from test_gpu_attn import packed_truth
from test_gpu_loras import adapters, truth as loras_truth
from test_gpu_paged import truth as paged_truth
from test_gpu_rope import check, turned

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, PAGE = 256, 8, 2, 64, 16
QKV = (HEADS + 2 * KV) * DIM
PROMPTS = [37, 1, 16, 90, 5]
IDS = [0, 2, -1, 1, 0]  # each request's adapter
STEPS = 4


class Layer:
    def __init__(self, ctx, engine, seed):
        g = np.random.default_rng(seed)
        self.ctx, self.engine = ctx, engine
        self.T = lambda a, d=None: UnifiedTensor.new(ctx, a, dtype=d)  # noqa: E731
        self.weights = {}
        for name, (n, k) in {"qkv": (QKV, HIDDEN), "o": (HIDDEN, HEADS * DIM)}.items():
            codes, s = g.integers(-127, 128, (n, k)).astype(np.int8), (g.random(n) * 0.002).astype(np.float32)
            a, b = adapters(g, 3, 8, k, n, "f16")
            self.weights[name] = (QuantizedTensor.rowwise(ctx, codes, s), codes * s.astype(np.float64)[:, None], a, b,
                                  LoraSet(self.T(a), self.T(b), self.T(np.array([1.0, 2.0, 0.5], np.float32))))
        self.rope = Rope(ctx, DIM, scaling="ramp", factor=4.0, trained=2048.0)
        self.freqs, self.magnitude = Rope.frequencies_of(DIM, scaling="ramp", factor=4.0, trained=2048.0)
        need = [-(-(p + STEPS) // PAGE) for p in PROMPTS]
        self.table = np.full((len(PROMPTS), max(need)), -1, np.int32)
        places, first = g.permutation(sum(need) + 2), 0
        for s, n in enumerate(need):
            self.table[s, :n] = places[first:first + n]
            first += n
        shape = (sum(need) + 2, KV, PAGE, DIM)
        self.K, self.V = (self.T(np.full(shape, np.nan, np.float16)) for _ in range(2))
        self.cache = PagedCache(self.K, self.V, self.T(self.table, DType.I32))

    def linear(self, name, x, ids, out, work, stream=None):
        self.engine.qmatmul_loras(self.ctx, x, self.weights[name][0], self.weights[name][4], ids, out, workspace=work, stream=stream)

    def work(self, name, x, out):
        return self.engine.qmatmul_loras_workspace(self.ctx, x, self.weights[name][0], self.weights[name][4], out)

    def check_linear(self, name, x, ids, got, what):
        _, w, a, b, _ = self.weights[name]
        check(got, *loras_truth(x, w, a, b, [1.0, 2.0, 0.5], ids, [8] * 3, "f16", False), what)

    def rows(self, buf):
        """q, k, v within the fused product's rows, as views."""
        n, size = buf.shape[0], 2
        view = lambda first, heads: UnifiedTensor(self.ctx, buf.ptr + first * DIM * size, (n, heads, DIM), DType.FP16, owner=False)  # noqa: E731
        return view(0, HEADS), view(HEADS, KV), view(HEADS + KV, KV)

    def cached(self, s, n):
        """Keys and values of sequence s, [kv, n, dim]."""
        out = []
        for pool in (self.K.to_vec(), self.V.to_vec()):
            rows = np.concatenate([pool[p] for p in self.table[s] if p >= 0], 1)
            out.append(rows[:, :n])
        return out


def split(qkv):
    r = qkv.reshape(-1, HEADS + 2 * KV, DIM)
    return r[:, :HEADS], r[:, HEADS:HEADS + KV], r[:, HEADS + KV:]


def test_prompts_then_decode_steps(ctx, engine):
    L = Layer(ctx, engine, 1)
    T = L.T
    g = np.random.default_rng(2)
    starts = np.concatenate([[0], np.cumsum(PROMPTS)]).astype(np.int32)
    total = int(starts[-1])
    row_ids = np.repeat(IDS, PROMPTS).astype(np.int32)
    positions = np.concatenate([np.arange(p) for p in PROMPTS]).astype(np.int32)
    # prompts: qkv -> rotary and cache -> causal attention -> o
    x = g.standard_normal((total, HIDDEN)).astype(np.float16)
    X, I, S, P = T(x), T(row_ids, DType.I32), T(starts, DType.I32), T(positions, DType.I32)
    qkv, q = T(np.zeros((total, QKV), np.float16)), T(np.zeros((total, HEADS, DIM), np.float16))
    L.linear("qkv", X, I, qkv, L.work("qkv", X, qkv))
    L.check_linear("qkv", x, row_ids, qkv.to_vec(), "prompts: qkv")
    vq, vk, vv = L.rows(qkv)
    engine.rope_append(ctx, vq, vk, vv, L.rope, P, L.cache, q, starts=S, q_row=QKV, k_row=QKV, v_row=QKV)
    hq, hk, hv = split(qkv.to_vec())
    check(q.to_vec(), *turned(hq, positions, L.freqs, L.magnitude, DIM, "half"), "prompts: q")
    wk, tk = turned(hk, positions, L.freqs, L.magnitude, DIM, "half")
    keys = np.zeros((total, KV, DIM), np.float16)
    for s, (a, b) in enumerate(zip(starts[:-1], starts[1:])):
        k, v = L.cached(s, b - a)
        keys[a:b] = k.transpose(1, 0, 2)
        check(keys[a:b], wk[a:b], tk[a:b], f"prompts: keys of {s}")
        assert np.array_equal(v.transpose(1, 0, 2), hv[a:b])
    K, att = T(keys), T(np.zeros((total, HEADS, DIM), np.float16))
    engine.attn_packed(ctx, q, K, vv, S, att, v_row=QKV)
    check_attn(att.to_vec(), *packed_truth(q.to_vec(), keys, hv, starts, 1 / 8, True), "prompts: attention")
    out = T(np.zeros((total, HIDDEN), np.float16))
    A = att.reshaped((total, HEADS * DIM))
    L.linear("o", A, I, out, L.work("o", A, out))
    L.check_linear("o", A.to_vec(), row_ids, out.to_vec(), "prompts: o")

    # decode: one token per request, eager; then the same steps captured, from a copy of the cache
    n = len(PROMPTS)
    ids = np.array(IDS, np.int32)
    saved = L.K.to_vec(), L.V.to_vec()
    xs = [g.standard_normal((n, HIDDEN)).astype(np.float16) for _ in range(STEPS)]
    X, I = T(xs[0]), T(ids, DType.I32)
    P, N = T(np.zeros(n, np.int32), DType.I32), T(np.zeros(n, np.int32), DType.I32)
    qkv, q, att = (T(np.zeros(sh, np.float16)) for sh in ((n, QKV), (n, HEADS, DIM), (n, HEADS, DIM)))
    out = T(np.zeros((n, HIDDEN), np.float16))
    A = att.reshaped((n, HEADS * DIM))
    vq, vk, vv = L.rows(qkv)
    works = [(L.work("qkv", X, qkv), engine.attn_paged_workspace(ctx, q, L.cache), L.work("o", A, out)) for _ in range(2)]

    def step(work, stream=None):
        L.linear("qkv", X, I, qkv, work[0], stream)
        engine.rope_append(ctx, vq, vk, vv, L.rope, P, L.cache, q, q_row=QKV, k_row=QKV, v_row=QKV, stream=stream)
        engine.attn_paged(ctx, q, L.cache, N, att, workspace=work[1], stream=stream)
        L.linear("o", A, I, out, work[2], stream)

    def put(t, a):
        call("rq_memcpy_h2d", ctx.handle, t.ptr, a.ctypes.data, a.nbytes, None)

    def at(i):
        put(X, xs[i])
        put(P, np.array([p + i for p in PROMPTS], np.int32))
        put(N, np.array([p + i + 1 for p in PROMPTS], np.int32))
        ctx.sync()

    eager = []
    for i in range(STEPS):
        at(i)
        step(works[0])
        positions = np.array([p + i for p in PROMPTS])
        L.check_linear("qkv", xs[i], ids, qkv.to_vec(), f"step {i}: qkv")
        hq, hk, hv = split(qkv.to_vec())
        check(q.to_vec(), *turned(hq, positions, L.freqs, L.magnitude, DIM, "half"), f"step {i}: q")
        wk, tk = turned(hk, positions, L.freqs, L.magnitude, DIM, "half")
        rows = [L.cached(s, p + i + 1) for s, p in enumerate(PROMPTS)]
        for s, (k, v) in enumerate(rows):
            check(k[:, -1], wk[s], tk[s], f"step {i}: key of {s}")
            assert np.array_equal(v[:, -1], hv[s])
        check_attn(att.to_vec(), *paged_truth(q.to_vec(), rows, 1 / 8, True), f"step {i}: attention")
        L.check_linear("o", A.to_vec(), ids, out.to_vec(), f"step {i}: o")
        eager.append(out.to_vec())

    stream = Stream()
    graph = Graph(stream.h, lambda: step(works[1], stream.h))
    put(L.K, saved[0])
    put(L.V, saved[1])
    for i in range(STEPS):
        at(i)
        graph.launch()
        stream.synchronize()
        rows = [L.cached(s, p + i + 1) for s, p in enumerate(PROMPTS)]
        check_attn(att.to_vec(), *paged_truth(q.to_vec(), rows, 1 / 8, True), f"replay {i}: attention")
        assert np.array_equal(out.to_vec(), eager[i]), f"replay {i}"
        step(works[0])  # eager work between the replays: the step again, with the same result
        assert np.array_equal(out.to_vec(), eager[i]), f"eager after replay {i}"
