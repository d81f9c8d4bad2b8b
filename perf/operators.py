"""Operators of a serving program: 4-bit Linears, attention of drafted trees over
a KV cache, causal attention of packed prompts.

``linear4``  Y[m, n] = X[m, k] . W[n, k]^T, W = u * s + b with 4-bit codes u
             (two per byte, the even element in the low nibble) and an f32
             scale and bias per ``group`` elements of a row.
``tree``     for each sequence, a few drafted tokens attend to the ``length``
             cached positions before them and to the drafted tokens (cached
             right behind) that their mask names: themselves and their ancestors.
``packed``   prompts one after another in one buffer, each token attending to
             itself and the tokens before it in its own prompt.

Query head h reads key/value head h / (heads / kv_heads).  Values: weights of
standard deviation 0.02 around zero (the usual Llama init), normal
activations, queries, keys and values.
"""
from __future__ import annotations

import math
import random

import torch

own = False

W_STD = 0.02
CODE_STD = 4.61  # of codes uniform in 0..15
_TORCH = {"f16": torch.float16, "f32": torch.float32}
_SIZE = {"f16": 2, "f32": 4}
_shared = {}


# ---- the cases -----------------------------------------------------------------


def listed():
    return [
        # One token through one Linear of a 7B-shape block: the smallest product
        # of a decoding program, latency and launch included.
        _linear("linear4_one_token", 1, 4096, 4096, 64, "f16", "f16"),
        # One token's logits: the 1.1B shape's lm_head, f32 out.
        _linear("linear4_head", 1, 32000, 2048, 64, "f16", "f32"),
        # Eight drafted tokens (or sequences) through a 7B-shape gate or up product.
        _linear("linear4_batch", 8, 11008, 4096, 64, "f16", "f16"),
        # A ragged batch in f32 through the down product, finer groups.
        _linear("linear4_ragged_f32", 13, 4096, 11008, 32, "f32", "f32"),
        # One sequence, one token, the 1.1B shape at the end of its 512-token
        # prompt: plain decoding, the smallest attention call.
        _tree("tree_one_token", [512], [1], 640, 32, 4, 64, "f16"),
        # Eight chats, trees of up to 16 nodes, 1.1B heads.
        _tree("tree_chats", [611, 1290, 37, 2047, 945, 1600, 333, 1811], [16, 11, 16, 7, 16, 16, 1, 13], 2176, 32, 4, 64,
              "f16"),
        # A long document at the runner's cache limit, a tree of 64, heads of 128.
        _tree("tree_long", [32701], [64], 32768, 32, 8, 128, "f16"),
        # The same pass in the reference's type, a few sequences.
        _tree("tree_f32", [700, 1501, 64, 1023], [13, 8, 13, 5], 1536, 32, 4, 64, "f32"),
        # A handful of very short prompts (one of a single token).
        _packed("packed_short", [37, 1, 12, 5, 64], 32, 4, 64, "f16", False),
        # A batch of chat prompts of every length, read in place from the fused
        # q/k/v product's rows.
        _packed("packed_chats", [611, 129, 37, 1047, 945, 1, 333, 780, 208], 32, 4, 64, "f16", True),
        # One long document with heads of 128.
        _packed("packed_long", [8192], 32, 8, 128, "f16", False),
        # Prompts in the reference's type.
        _packed("packed_f32", [417, 1000, 83], 32, 4, 64, "f32", False),
    ]


def _linear(name, m, n, k, group, x, y):
    return {"name": name, "op": "linear4", "m": m, "n": n, "k": k, "group": group, "x": x, "y": y}


def _text(values):
    return ",".join(str(v) for v in values)


def _tree(name, lengths, nodes, capacity, heads, kv, dim, dtype):
    return {"name": name, "op": "tree", "lengths": _text(lengths), "nodes": _text(nodes), "capacity": capacity,
            "heads": heads, "kv": kv, "dim": dim, "dtype": dtype}


def _packed(name, lengths, heads, kv, dim, dtype, fused):
    return {"name": name, "op": "packed", "lengths": _text(lengths), "heads": heads, "kv": kv, "dim": dim,
            "dtype": dtype, "fused": fused}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 4, 64), (32, 8, 128), (32, 32, 64), (16, 16, 128), (12, 4, 64), (8, 1, 128), (14, 2, 64), (40, 8, 128)]


def draw(rng):
    """One more case of the ranges above: 1..16 rows and weights of 256..11008
    a side; trees of 1..64 nodes over 0..32768 cached positions, up to 16
    sequences; up to 24 prompts of 8192 tokens together."""
    op = rng.choices(["linear4", "tree", "packed"], [4, 4, 4])[0]
    if op == "linear4":
        group = rng.choice([32, 64, 64, 128])
        k = max(group, _log(rng, 256, 11008) // group * group)
        n = _log(rng, 256, 11008) // rng.choice([1, 8, 64])
        n = n if n >= 256 else n * 64
        x, y = rng.choice([("f16", "f16"), ("f16", "f16"), ("f32", "f32"), ("f16", "f32")])
        return _nameless(_linear("", _log(rng, 1, 16), min(n, 11008), k, group, x, y))
    heads, kv, dim = rng.choice(HEADS)
    dtype = rng.choice(["f16", "f16", "f16", "f32"])
    if op == "tree":
        count = _log(rng, 1, 16)
        nodes = [rng.choice([1, _log(rng, 1, 64), _log(rng, 4, 24)]) for _ in range(count)]
        most = (16384 if dtype == "f16" else 4096) // count
        lengths = [max(0, _log(rng, 1, most) - 1) for _ in range(count)]
        capacity = max(a + b for a, b in zip(lengths, nodes)) + rng.randrange(0, 65)
        return _nameless(_tree("", lengths, nodes, capacity, heads, kv, dim, dtype))
    total = _log(rng, 16, 6144 if dtype == "f16" else 2048)
    count = min(total, _log(rng, 1, 24))
    cuts = sorted(rng.randrange(0, total + 1) for _ in range(count - 1))
    lengths = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    return _nameless(_packed("", lengths, heads, kv, dim, dtype, rng.random() < 0.5))


def _nameless(case):
    case.pop("name")
    return case


def _ints(text):
    return [int(v) for v in text.split(",")]


def _starts(counts):
    s = [0]
    for c in counts:
        s.append(s[-1] + c)
    return s


# ---- inputs ----------------------------------------------------------------------


def _ancestors(seed, counts):
    """A random tree per sequence as one mask per node: bit j for node j of the
    same sequence that is the node itself or an ancestor of it."""
    r = random.Random(seed * 7919 + 17)
    rows = []
    for c in counts:
        masks = []
        for i in range(c):
            parent = r.randrange(-1 if i == 0 else max(0, i - 4), i) if i else -1
            masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
        rows += masks
    return rows


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    normal = lambda shape, t: torch.randn(shape, generator=g, device="cuda").to(_TORCH[t])  # noqa: E731
    op = case["op"]
    if op == "linear4":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        codes = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        s = (torch.rand((n, k // group), generator=g, device="cuda") + 0.5) * (W_STD / CODE_STD)
        b = -7.5 * s * (0.95 + 0.1 * torch.rand(s.shape, generator=g, device="cuda"))
        return {"codes": codes, "scales": s, "biases": b, "x": normal((m, k), case["x"])}
    heads, kv, dim, t = case["heads"], case["kv"], case["dim"], case["dtype"]
    lengths = _ints(case["lengths"])
    if op == "tree":
        nodes = _ints(case["nodes"])
        masks = _ancestors(int(seed), nodes)
        signed = [v - (1 << 64) if v >> 63 else v for v in masks]
        shape = (len(lengths), kv, case["capacity"], dim)  # stale positions hold other sequences' rows
        return {"q": normal((sum(nodes), heads, dim), t), "k": normal(shape, t), "v": normal(shape, t),
                "starts": torch.tensor(_starts(nodes), dtype=torch.int32, device="cuda"),
                "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                "mask": torch.tensor(signed, dtype=torch.int64, device="cuda")}
    total = sum(lengths)
    out = {"starts": torch.tensor(_starts(lengths), dtype=torch.int32, device="cuda")}
    if case["fused"]:
        out["qkv"] = normal((total, (heads + 2 * kv) * dim), t)
    else:
        out.update(q=normal((total, heads, dim), t), k=normal((total, kv, dim), t), v=normal((total, kv, dim), t))
    return out


def _rows(case, t):
    """q, k, v of a packed case as [tokens, heads, dim] views."""
    if not case["fused"]:
        return t["q"], t["k"], t["v"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    rows = t["qkv"].view(-1, heads + 2 * kv, dim)
    return rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]


def prepare(case, seed):
    t = _inputs(case, seed)
    s = {"case": case, "t": t}
    if case["op"] == "linear4":
        s["out"] = torch.empty((case["m"], case["n"]), dtype=_TORCH[case["y"]], device="cuda")
    else:
        rows = sum(_ints(case["nodes" if case["op"] == "tree" else "lengths"]))
        s["out"] = torch.empty((rows, case["heads"], case["dim"]), dtype=_TORCH[case["dtype"]], device="cuda")
    if own:
        _prepare_own(case, t, s)
    torch.cuda.synchronize()
    return s


def _prepare_own(case, t, s):
    """What a program holds: tensor views, the weight, the workspace."""
    from rusty_amd import ComputeEngine, DType, QuantizedTensor, UnifiedTensor, WgpuContext

    if not _shared:
        _shared["ctx"] = WgpuContext(0)
        _shared["eng"] = ComputeEngine(_shared["ctx"])
    ctx, eng = _shared["ctx"], _shared["eng"]
    kinds = {torch.float16: DType.FP16, torch.float32: DType.FP32, torch.uint8: DType.U8, torch.int32: DType.I32,
             torch.int64: DType.U64}
    view = lambda x, shape=None: UnifiedTensor(ctx, x.data_ptr(), shape or x.shape, kinds[x.dtype], owner=False)  # noqa: E731
    s["out_v"] = view(s["out"])
    if case["op"] == "linear4":
        s["w"] = QuantizedTensor.from_affine4(view(t["codes"]), view(t["scales"]), view(t["biases"]), case["group"])
        s["x"] = view(t["x"])
    elif case["op"] == "tree":
        s["v"] = {n: view(t[n]) for n in ("q", "k", "v", "starts", "lengths", "mask")}
        nodes = _ints(case["nodes"])
        s["most"] = max(nodes)
        s["work"] = eng.attn_tree_workspace(ctx, s["v"]["q"], s["v"]["k"], s["most"])
    else:
        q, k, v = _rows(case, t)
        s["v"] = {"q": view(q), "k": view(k), "v": view(v), "starts": view(t["starts"])}
        s["row"] = t["qkv"].shape[1] if case["fused"] else None


# ---- one pass ----------------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        ctx, eng, v = _shared["ctx"], _shared["eng"], state.get("v")
        if case["op"] == "linear4":
            eng.qmatmul(ctx, state["x"], state["w"], state["out_v"])
        elif case["op"] == "tree":
            eng.attn_tree(ctx, v["q"], v["k"], v["v"], v["starts"], v["lengths"], v["mask"], state["out_v"],
                          state["most"], workspace=state["work"])
        else:
            row = state["row"]
            eng.attn_packed(ctx, v["q"], v["k"], v["v"], v["starts"], state["out_v"], q_row=row, k_row=row, v_row=row)
        return state["out"]
    return {"linear4": _plain_linear, "tree": _plain_tree, "packed": _plain_packed}[case["op"]](case, state["t"], state["out"])


def _plain_linear(case, t, out):
    n, k, group = case["n"], case["k"], case["group"]
    u = torch.stack((t["codes"] & 15, t["codes"] >> 4), 2).view(n, k // group, group).float()
    w = (u * t["scales"][:, :, None] + t["biases"][:, :, None]).view(n, k)
    out.copy_(t["x"].float() @ w.T)
    return out


def _attend(q, k, v, keep):
    """q [kv, rows, dim] over k, v [kv, keys, dim]; keep [1 or kv, rows, keys].
    A row that keeps no key gives zeros."""
    s = torch.matmul(q, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(q.shape[2]))
    s = torch.where(keep, s, torch.full_like(s, -math.inf))
    top = s.amax(2, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(2, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)


def _grouped(q, kv):
    """[rows, heads, dim] -> f32 [kv, heads per kv * rows, dim]"""
    rows, heads, dim = q.shape
    return q.float().view(rows, kv, heads // kv, dim).permute(1, 2, 0, 3).reshape(kv, -1, dim)


def _ungrouped(o, rows, heads):
    kv, _, dim = o.shape
    return o.view(kv, heads // kv, rows, dim).permute(2, 0, 1, 3).reshape(rows, heads, dim)


def _plain_tree(case, t, out):
    heads, kv = case["heads"], case["kv"]
    lengths, nodes = _ints(case["lengths"]), _ints(case["nodes"])
    first = 0
    for i, (length, n) in enumerate(zip(lengths, nodes)):
        rows = slice(first, first + n)
        bits = torch.arange(n, device="cuda")
        tree = (t["mask"][rows, None] >> bits & 1) == 1
        keep = torch.cat((torch.ones((n, length), dtype=torch.bool, device="cuda"), tree), 1)
        k, v = t["k"][i, :, :length + n].float(), t["v"][i, :, :length + n].float()
        o = _attend(_grouped(t["q"][rows], kv), k, v, keep.repeat(heads // kv, 1)[None])
        out[rows] = _ungrouped(o, n, heads).to(out.dtype)
        first += n
    return out


def _plain_packed(case, t, out):
    heads, kv = case["heads"], case["kv"]
    q, k, v = _rows(case, t)
    first = 0
    for n in _ints(case["lengths"]):
        at = torch.arange(n, device="cuda")
        # a long prompt takes one key/value head and 2048 queries at a time
        for g in ([slice(j, j + 1) for j in range(kv)] if n > 1024 else [slice(0, kv)]):
            kg = k[first:first + n, g].float().transpose(0, 1).contiguous()
            vg = v[first:first + n, g].float().transpose(0, 1).contiguous()
            per, count = heads // kv, kg.shape[0]
            for lo in range(0, n, 2048):
                hi = min(n, lo + 2048)
                qg = _grouped(q[first + lo:first + hi, g.start * per:g.start * per + count * per], count)
                keep = (at[None, :hi] <= at[lo:hi, None]).repeat(per, 1)[None]
                o = _attend(qg, kg[:, :hi], vg[:, :hi], keep)
                out[first + lo:first + hi, g.start * per:g.start * per + count * per] = \
                    _ungrouped(o, hi - lo, count * per).to(out.dtype)
        first += n
    return out


# ---- what a pass cannot do without -----------------------------------------------------


def work(case):
    if case["op"] == "linear4":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k // 2 + 8 * n * (k // case["group"]) + m * k * _SIZE[case["x"]] + m * n * _SIZE[case["y"]],
                "flops": 2 * m * n * k}
    heads, kv, dim, size = case["heads"], case["kv"], case["dim"], _SIZE[case["dtype"]]
    lengths = _ints(case["lengths"])
    if case["op"] == "tree":
        nodes = _ints(case["nodes"])
        keys = sum(a + b for a, b in zip(lengths, nodes))
        masks = _ancestors(0, nodes)
        pairs = sum(a * b for a, b in zip(lengths, nodes)) + sum(bin(m).count("1") for m in masks)
        return {"bytes": 2 * keys * kv * dim * size + sum(nodes) * (2 * heads * dim * size + 8) + 8 * len(nodes) + 4,
                "flops": 4 * heads * dim * pairs}
    total = sum(lengths)
    return {"bytes": total * dim * size * (2 * heads + 2 * kv) + 4 * len(lengths) + 4,
            "flops": 4 * heads * dim * sum(n * (n + 1) // 2 for n in lengths)}


# ---- the true result, in 64 bits ---------------------------------------------------------


def exact(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "linear4":
        c = t["codes"].to(torch.int32)
        y = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
        for half in (0, 1):  # even elements in the low nibbles, odd ones in the high
            u = (c // (16 if half else 1)) % 16
            g = (torch.arange(u.shape[1], device="cuda") * 2 + half) // case["group"]
            w = u.double() * t["scales"].double()[:, g] + t["biases"].double()[:, g]
            y += t["x"][:, half::2].double() @ w.T.contiguous()
        return y
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    counts = _ints(case["nodes"] if case["op"] == "tree" else case["lengths"])
    out = torch.zeros((sum(counts), heads, dim), dtype=torch.float64, device="cuda")
    masks = _ancestors(int(seed), counts) if case["op"] == "tree" else None
    first = 0
    for i, n in enumerate(counts):
        for h in range(heads if n else 0):
            j = h * kv // heads
            if masks is not None:
                length = _ints(case["lengths"])[i]
                k, v = t["k"][i, j, :length + n].double(), t["v"][i, j, :length + n].double()
                allowed = torch.tensor([[m >> b & 1 for b in range(n)] for m in masks[first:first + n]], device="cuda")
                hidden = torch.cat((torch.zeros((n, length), device="cuda"), 1 - allowed), 1).bool()
                q = t["q"][first:first + n, h]
            else:
                qa, ka, va = _rows(case, t)
                q, k, v = qa[first:first + n, h], ka[first:first + n, j].double(), va[first:first + n, j].double()
                hidden = torch.ones((n, n), device="cuda").triu(1).bool()
            s = (q.double() @ k.T.contiguous()) / math.sqrt(dim)
            out[first:first + n, h] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v
        first += n
    return out
