"""An attention layer with 4-bit Linears as a server runs it: two prompts
through the fused q/k/v product, rq_attn_packed on its rows and the output
product, their keys and values into a cache, then a drafted tree for each
through the same products and rq_attn_tree.  Every stage is checked against
64 bits from what the device handed to it, with that stage's tolerance."""
import numpy as np
import pytest
from test_gpu_attn import attend, tree_masks
from test_gpu_attn import check as check_attn
from test_gpu_linear4 import check, truth, weight

from rusty_amd import DType, QuantizedTensor, UnifiedTensor

pytestmark = pytest.mark.gpu

KIND = {"f16": (np.float16, DType.FP16), "f32": (np.float32, DType.FP32)}


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (6, 1, 128)])
def test_prompts_then_trees(ctx, engine, heads, kv, dim, dtype):
    f16, (np_t, kind) = dtype == "f16", KIND[dtype]
    g = np.random.default_rng(dim + heads)
    hidden, wide, scale = heads * dim, (heads + 2 * kv) * dim, dim ** -0.5
    wqkv, wo = weight(g, wide, hidden, 64), weight(g, hidden, hidden, 32)
    qkv4, o4 = QuantizedTensor.affine4(ctx, *wqkv), QuantizedTensor.affine4(ctx, *wo)
    T = lambda a, d=kind: UnifiedTensor.new(ctx, a, dtype=d)  # noqa: E731

    def product(x, w, q4, n, what):
        y = UnifiedTensor.empty(ctx, [x.shape[0], n], kind)
        engine.qmatmul(ctx, T(x), q4, y)
        got = y.to_vec()
        check(got, *truth(x, w, f16), what)
        return y, got.astype(np_t)

    def split(a):
        a = a.reshape(len(a), heads + 2 * kv, dim)
        return a[:, :heads], a[:, heads:heads + kv], a[:, heads + kv:]

    # prompts
    lengths, nodes, cap = [70, 9], [6, 13], 96
    starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    x = g.standard_normal((starts[-1], hidden)).astype(np_t)
    y, rows = product(x, wqkv, qkv4, wide, "q/k/v of prompts")
    q, k, v = split(rows)
    fused = [UnifiedTensor(ctx, y.ptr + at * dim * kind.itemsize, [len(x), h, dim], kind, owner=False)
             for h, at in ((heads, 0), (kv, heads), (kv, heads + kv))]
    out = T(np.zeros((len(x), heads, dim)))
    engine.attn_packed(ctx, *fused, T(starts, DType.I32), out, q_row=wide, k_row=wide, v_row=wide)
    got = out.to_vec()
    for s, n in enumerate(lengths):
        a = slice(starts[s], starts[s] + n)
        for h in range(heads):
            j = h // (heads // kv)
            check_attn(got[a, h], *attend(q[a, h], k[a, j], v[a, j], np.tril(np.ones((n, n), bool)), scale, f16),
                       f"prompt {s} head {h}")
    product(got.reshape(len(x), hidden).astype(np_t), wo, o4, hidden, "output of prompts")
    # their keys and values, with stale ones behind
    kc, vc = (g.standard_normal((2, kv, cap, dim)).astype(np_t) for _ in range(2))
    for s, n in enumerate(lengths):
        kc[s, :, :n], vc[s, :, :n] = (a[starts[s]:starts[s] + n].transpose(1, 0, 2) for a in (k, v))

    # drafted trees
    first = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    mask = tree_masks(g, nodes)
    x = g.standard_normal((first[-1], hidden)).astype(np_t)
    _, rows = product(x, wqkv, qkv4, wide, "q/k/v of trees")
    q, k, v = split(rows)
    for s, n in enumerate(nodes):
        a = slice(first[s], first[s] + n)
        kc[s, :, lengths[s]:lengths[s] + n], vc[s, :, lengths[s]:lengths[s] + n] = (z[a].transpose(1, 0, 2) for z in (k, v))
    out = T(np.zeros((len(x), heads, dim)))
    engine.attn_tree(ctx, T(q), T(kc), T(vc), T(first, DType.I32), T(np.array(lengths, np.int32), DType.I32),
                     T(mask, DType.U64), out, max(nodes))
    got = out.to_vec()
    for s, n in enumerate(nodes):
        end = lengths[s] + n
        keep = np.ones((n, end), bool)
        for i in range(n):
            keep[i, lengths[s]:] = [int(mask[first[s] + i]) >> j & 1 for j in range(n)]
        for h in range(heads):
            j = h // (heads // kv)
            check_attn(got[first[s]:first[s] + n, h],
                       *attend(q[first[s]:first[s] + n, h], kc[s, j, :end], vc[s, j, :end], keep, scale, f16),
                       f"tree {s} head {h}")
    product(got.reshape(len(x), hidden).astype(np_t), wo, o4, hidden, "output of trees")
