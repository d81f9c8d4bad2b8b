"""Operators of a program that serves many requests at once: rotary positions
(and the keys' and values' way into a paged cache), attention of one new token
per sequence over that cache, a quantized Linear with an adapter per token.

``rope``    each head's first ``rot`` elements turned in pairs by the angle
            position * frequency: out_a = x_a cos - x_b sin, out_b = x_b cos +
            x_a sin, times a magnitude.  Pairs are (i, i + rot / 2), layout
            ``half``, or (2 i, 2 i + 1), ``interleaved``.  The frequencies are
            theta^(-2 i / rot), scaled for contexts longer than the trained
            one (see ``_frequencies``).  ``backward``: the gradient of x from
            that of out, the turn the other way.
``append``  q and k turned so, q into a buffer of its own, k and v into the
            pages of their sequence: position p lies in page table[s][p / page]
            at p % page.
``paged``   for each sequence, one token attends to the ``length`` positions
            cached for it (its own among them).
``loras``   Y = X . W^T + scale_i (X . A_i^T) . B_i, i the adapter of the row
            (none where it is negative), W quantized.

Query head h reads key/value head h / (heads / kv_heads).  Values: weights of
standard deviation 0.02 around zero (the usual Llama init), adapters of the
size that training leaves them at, normal activations, queries, keys, values.
"""
from __future__ import annotations

import math
import random

import torch

own = False

W_STD = 0.02
_TORCH = {"f16": torch.float16, "f32": torch.float32}
_SIZE = {"f16": 2, "f32": 4}
_BYTES = {"rowwise8": 1.0, "affine8": 1.0, "affine4": 0.5}  # a weight's code
_shared = {}


# ---- the cases -----------------------------------------------------------------


def listed():
    return [
        # One token's query heads, the 1.1B shape: the smallest call, all latency.
        _rope("rope_one_token", 1, 32, 64, 64, "half", "none", 512, "f16", False),
        # The gradient of a training batch's queries, pairs side by side, half of each head turned.
        _rope("rope_gradient", 8192, 32, 128, 64, "interleaved", "none", 2048, "f16", True),
        # A piece of a long document in the reference's type, far positions, frequencies by ramp.
        _rope("rope_far_f32", 1537, 14, 64, 64, "half", "ramp", 120000, "f32", False),
        # A decode step of 64 chats, read from the rows of the fused q/k/v product.
        _append("append_step", [1] * 64, 2047, 32, 4, 64, 64, "half", "none", 16, "heads", "f16", True),
        # Nine chat prompts of every length on their way into the cache, frequencies by bands.
        _append("append_prompts", [611, 129, 37, 1047, 945, 1, 333, 780, 208], 300, 32, 8, 128, 128, "half", "bands", 16,
                "heads", "f16", True),
        # One sequence of the 1.1B shape: plain decoding, the smallest attention call.
        _paged("paged_one", [513], 32, 4, 64, 16, "heads", "f16"),
        # 48 chats of every length, the 1.1B shape.
        _paged("paged_chats", _lengths(48, 37, 2047, 11), 32, 4, 64, 16, "heads", "f16"),
        # A few long documents at the runner's cache limit beside short questions, heads of 128.
        _paged("paged_long", [32701, 212, 20011, 33, 9000, 30001], 32, 8, 128, 64, "positions", "f16"),
        # The reference's type, every query head with keys of its own.
        _paged("paged_f32", [700, 1501, 64, 3001, 1023, 1, 410], 16, 16, 128, 32, "heads", "f32"),
        # One request, one token through a 7B-shape block's Linear.
        _loras("loras_one_token", [1], 1, 4096, 4096, 16, "rowwise8", "f16", "f16", "f16", False),
        # A decode step of 16 requests over 11 adapters (some have none), up or gate product, 4-bit weights.
        _loras("loras_batch", [1] * 16, 11, 11008, 4096, 16, "affine4", "f16", "f16", "f16", True),
        # Prompts of six requests packed, adapters of rank 32.
        _loras("loras_prompts", [611, 129, 37, 1047, 23, 201], 5, 4096, 4096, 32, "rowwise8", "f16", "f16", "f16", False),
    ]


def _lengths(count, lo, hi, seed):
    r = random.Random(seed)
    return [_log(r, lo, hi) for _ in range(count)]


def _text(values):
    return ",".join(str(v) for v in values)


def _rope(name, tokens, heads, dim, rot, layout, scaling, far, dtype, backward):
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "dim": dim, "rot": rot, "layout": layout,
            "scaling": scaling, "far": far, "dtype": dtype, "backward": backward}


def _append(name, lengths, before, heads, kv, dim, rot, layout, scaling, page, order, dtype, fused):
    """``before``: each sequence has up to so many positions already."""
    return {"name": name, "op": "append", "lengths": _text(lengths), "before": before, "heads": heads, "kv": kv,
            "dim": dim, "rot": rot, "layout": layout, "scaling": scaling, "page": page, "order": order, "dtype": dtype,
            "fused": fused}


def _paged(name, lengths, heads, kv, dim, page, order, dtype):
    return {"name": name, "op": "paged", "lengths": _text(lengths), "heads": heads, "kv": kv, "dim": dim, "page": page,
            "order": order, "dtype": dtype}


def _loras(name, lengths, adapters, n, k, rank, weight, x, y, adapter, some):
    """``lengths``: rows one after another of one request; ``some``: a request may have no adapter."""
    return {"name": name, "op": "loras", "lengths": _text(lengths), "adapters": adapters, "n": n, "k": k, "rank": rank,
            "weight": weight, "x": x, "y": y, "adapter": adapter, "some": some}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cut(rng, total, count):
    cuts = sorted(rng.randrange(0, total + 1) for _ in range(count - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


HEADS = [(32, 4, 64), (32, 8, 128), (32, 32, 64), (16, 16, 128), (12, 4, 64), (8, 1, 128), (14, 2, 64), (40, 8, 128)]
SCALINGS = ["none", "none", "linear", "stretch", "bands", "ramp"]


def draw(rng):
    """One more case of the ranges above: 1..8192 rows of positions up to
    131072, heads of 32..256; 1..64 sequences in pages of 8..256 positions, up
    to 65536 cached ones together; 1..2048 rows over 1..64 adapters of rank
    4..128, weights of 256..11008 a side."""
    op = rng.choices(["rope", "append", "paged", "loras"], [3, 2, 4, 4])[0]
    dtype = rng.choice(["f16", "f16", "f16", "f32"])
    layout, scaling = rng.choice(["half", "interleaved"]), rng.choice(SCALINGS)
    heads, kv, dim = rng.choice(HEADS)
    page, order = rng.choice([8, 16, 16, 32, 64, 128, 256]), rng.choice(["heads", "heads", "positions"])
    if op == "rope":
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        heads = _log(rng, 1, 40)
        rot = dim if rng.random() < 0.6 else rng.randrange(1, dim // 2 + 1) * 2
        tokens = min(_log(rng, 1, 8192), (1 << 24) // (heads * dim))
        return _nameless(_rope("", tokens, heads, dim, rot, layout, scaling, _log(rng, 64, 131072), dtype, rng.random() < 0.4))
    if op == "append":
        count = _log(rng, 1, 64)
        lengths = [1] * count if rng.random() < 0.4 else _cut(rng, max(count, _log(rng, 16, 4096)), count)
        rot = dim if rng.random() < 0.6 else rng.randrange(1, dim // 2 + 1) * 2
        return _nameless(_append("", lengths, min(_log(rng, 1, 2048), 32768 // count), heads, kv, dim, rot, layout, scaling,
                                 page, order, dtype, rng.random() < 0.5))
    if op == "paged":
        count = _log(rng, 1, 64)
        most = (1 << 28) // (2 * kv * dim * _SIZE[dtype])  # cached positions together: 256 MiB of keys and values
        top = max(1, min(32768, most // count))
        lengths = [_log(rng, 1, top) - (rng.random() < 0.1) for _ in range(count)]
        return _nameless(_paged("", lengths, heads, kv, dim, page, order, dtype))
    weight = rng.choice(["rowwise8", "rowwise8", "affine8", "affine4"])
    k = max(64, _log(rng, 256, 11008) // 64 * 64)
    n = max(256, _log(rng, 256, 11008) // rng.choice([1, 8, 64]) * rng.choice([1, 8, 64]))
    n = min(n, 11008)
    adapters, rank = _log(rng, 1, 64), min(128, _log(rng, 4, 160))
    if rng.random() < 0.5:
        lengths = [1] * _log(rng, 1, 64)
        x, y, a = rng.choice([("f16", "f16", "f16"), ("f16", "f16", "f32"), ("f32", "f32", "f32"), ("f16", "f32", "f16")])
        if len(lengths) > 16:
            x, y = "f16", "f16"
    else:
        total = min(_log(rng, 17, 2048), (1 << 35) // (n * k))
        lengths = _cut(rng, total, min(total, _log(rng, 1, 12)))
        x, y, a = "f16", "f16", rng.choice(["f16", "f16", "f32"])
    return _nameless(_loras("", lengths, adapters, n, k, rank, weight, x, y, a, rng.random() < 0.5))


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


# ---- rotary frequencies ------------------------------------------------------------

# Eight times a trained context of 8192 positions.
THETA, FACTOR, TRAINED = 10000.0, 8.0, 8192
BANDS = (1.0, 4.0)    # trained context / wavelength: stretched fully below the first, not at all above the second
RAMP = (1.0, 32.0)    # turns within the trained context, likewise


def _frequencies(rot, scaling):
    """(frequency of each pair, magnitude), in 64 bits."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = THETA ** (-2 * i / rot)
    if scaling == "linear":  # positions interpolated
        return f / FACTOR, 1.0
    if scaling == "stretch":  # the base grows so that the slowest pair is interpolated
        return (THETA * FACTOR ** (rot / (rot - 2) if rot > 2 else 1.0)) ** (-2 * i / rot), 1.0
    if scaling == "bands":  # slow pairs interpolated, fast ones kept, between them by wavelength
        kept = ((TRAINED * f / (2 * math.pi) - BANDS[0]) / (BANDS[1] - BANDS[0])).clamp(0, 1)
        return f * (kept + (1 - kept) / FACTOR), 1.0
    if scaling == "ramp":  # the same by the pair's index, and scores sharpened
        at = lambda turns: rot * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(THETA))  # noqa: E731
        lo, hi = max(math.floor(at(RAMP[1])), 0), min(math.ceil(at(RAMP[0])), rot - 1)
        slow = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * (1 - slow + slow / FACTOR), 0.1 * math.log(FACTOR) + 1
    return f, 1.0


# ---- inputs ----------------------------------------------------------------------


def _page_table(case, counts, g, room=None):
    """Pages of each sequence: a random choice of the pool's, none (-1) past its end.  ``room``: positions that the
    pool is made for, per sequence, where that is more."""
    need = [-(-c // case["page"]) for c in counts]
    most = [-(-c // case["page"]) for c in room or counts]
    width, total = max(max(most), 1), sum(most) + 5
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    first = 0
    for s, n in enumerate(need):
        table[s, :n] = order[first:first + n]
        first += n
    shape = (total, case["kv"], case["page"], case["dim"])
    return table, shape if case["order"] == "heads" else (shape[0], shape[2], shape[1], shape[3])


def _before(case, seed):
    """Positions that each sequence of an append has already."""
    r = random.Random(seed * 7919 + 17)
    return [r.randrange(0, case["before"] + 1) for _ in _ints(case["lengths"])]


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    normal = lambda shape, t: torch.randn(shape, generator=g, device="cuda", dtype=_TORCH[t])  # noqa: E731
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    op = case["op"]
    if op == "rope":
        x = normal((case["tokens"], case["heads"], case["dim"]), case["dtype"])
        at = torch.randint(0, case["far"], (case["tokens"],), generator=g, device="cuda", dtype=torch.int32)
        return {"x": x, "positions": at}
    if op == "append":
        heads, kv, dim, t = case["heads"], case["kv"], case["dim"], case["dtype"]
        counts, before = _ints(case["lengths"]), _before(case, int(seed))
        table, shape = _page_table(case, [a + b for a, b in zip(counts, before)], g, [c + case["before"] for c in counts])
        out = {"table": table, "k_pages": normal(shape, t), "v_pages": normal(shape, t), "starts": whole(_starts(counts)),
               "positions": whole([b + i for b, c in zip(before, counts) for i in range(c)])}
        total = sum(counts)
        if case["fused"]:
            out["qkv"] = normal((total, (heads + 2 * kv) * dim), t)
        else:
            out.update(q=normal((total, heads, dim), t), k=normal((total, kv, dim), t), v=normal((total, kv, dim), t))
        return out
    if op == "paged":
        counts, t = _ints(case["lengths"]), case["dtype"]
        table, shape = _page_table(case, counts, g)
        return {"table": table, "k_pages": normal(shape, t), "v_pages": normal(shape, t), "lengths": whole(counts),
                "q": normal((len(counts), case["heads"], case["dim"]), t)}
    n, k, rank, count = case["n"], case["k"], case["rank"], case["adapters"]
    rows = _ints(case["lengths"])
    r = random.Random(int(seed) * 7919 + 5)
    ids = [r.randrange(-1 if case["some"] else 0, count) for _ in rows]
    out = {"x": normal((sum(rows), k), case["x"]), "ids": whole([i for i, c in zip(ids, rows) for _ in range(c)]),
           "a": (torch.randn((count, rank, k), generator=g, device="cuda") * k ** -0.5).to(_TORCH[case["adapter"]]),
           "b": (torch.randn((count, rank, n), generator=g, device="cuda") * 0.02).to(_TORCH[case["adapter"]]),
           "factors": torch.rand((count,), generator=g, device="cuda") * 1.5 + 0.5}
    if case["weight"] == "rowwise8":
        out["codes"] = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
        out["scales"] = (torch.rand((n,), generator=g, device="cuda") + 0.5) * (W_STD / 73)
        return out
    half = case["weight"] == "affine4"
    out["codes"] = torch.randint(0, 256, (n, k // 2 if half else k), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.rand((n, k // 64), generator=g, device="cuda") + 0.5) * (W_STD / (4.61 if half else 74))
    out["scales"], out["biases"] = s, -(7.5 if half else 127.5) * s * (0.95 + 0.1 * torch.rand(s.shape, generator=g, device="cuda"))
    return out


def _rows(case, t):
    """q, k, v of an append as [tokens, heads, dim] views."""
    if not case["fused"]:
        return t["q"], t["k"], t["v"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    rows = t["qkv"].view(-1, heads + 2 * kv, dim)
    return rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]


def prepare(case, seed):
    t = _inputs(case, seed)
    s = {"case": case, "t": t}
    op = case["op"]
    empty = lambda shape, t: torch.empty(shape, dtype=_TORCH[t], device="cuda")  # noqa: E731
    if op == "rope":
        s["out"] = torch.empty_like(t["x"])
    elif op == "append":
        s["out"] = empty((t["positions"].numel(), case["heads"], case["dim"]), case["dtype"])
    elif op == "paged":
        s["out"] = torch.empty_like(t["q"])
    else:
        s["out"] = empty((t["x"].shape[0], case["n"]), case["y"])
    if op in ("rope", "append"):
        f, s["magnitude"] = _frequencies(case["rot"], case["scaling"])
        s["frequencies"] = f.cuda()
    if own:
        _prepare_own(case, t, s)
    torch.cuda.synchronize()
    return s


def _prepare_own(case, t, s):
    """What a program holds: tensor views, the rotary plan, the cache, the weight and its adapters, a workspace."""
    from rusty_amd import ComputeEngine, DType, LoraSet, PagedCache, QuantizedTensor, Rope, UnifiedTensor, WgpuContext

    if not _shared:
        _shared["ctx"] = WgpuContext(0)
        _shared["eng"] = ComputeEngine(_shared["ctx"])
    ctx, eng = _shared["ctx"], _shared["eng"]
    kinds = {torch.float16: DType.FP16, torch.float32: DType.FP32, torch.uint8: DType.U8, torch.int8: DType.I8,
             torch.int32: DType.I32}
    view = lambda x: UnifiedTensor(ctx, x.data_ptr(), x.shape, kinds[x.dtype], owner=False)  # noqa: E731
    op = case["op"]
    s["out_v"] = view(s["out"])
    if op in ("rope", "append"):
        low, high = BANDS if case["scaling"] == "bands" else RAMP
        s["rope"] = Rope(ctx, case["dim"], rot_dim=case["rot"], layout=case["layout"], theta=THETA, scaling=case["scaling"],
                         factor=FACTOR, trained=TRAINED, low=low, high=high)
        s["positions"] = view(t["positions"])
    if op in ("append", "paged"):
        s["cache"] = PagedCache(view(t["k_pages"]), view(t["v_pages"]), view(t["table"]), order=case["order"])
    if op == "rope":
        s["x"] = view(t["x"])
    elif op == "append":
        s["qkv"] = [view(x) for x in _rows(case, t)]
        s["row"] = t["qkv"].shape[1] if case["fused"] else None
        s["starts"] = view(t["starts"])
    elif op == "paged":
        s["q"], s["lengths"] = view(t["q"]), view(t["lengths"])
        s["work"] = eng.attn_paged_workspace(ctx, s["q"], s["cache"])
    else:
        if case["weight"] == "rowwise8":
            s["w"] = QuantizedTensor.from_rowwise(view(t["codes"]), view(t["scales"]))
        elif case["weight"] == "affine8":
            s["w"] = QuantizedTensor.from_affine(view(t["codes"]), view(t["scales"]), view(t["biases"]), 64)
            s["w"].prepare(ctx)
        else:
            s["w"] = QuantizedTensor.from_affine4(view(t["codes"]), view(t["scales"]), view(t["biases"]), 64)
        s["set"] = LoraSet(view(t["a"]), view(t["b"]), view(t["factors"]))
        s["x"], s["ids"] = view(t["x"]), view(t["ids"])
        s["work"] = eng.qmatmul_loras_workspace(ctx, s["x"], s["w"], s["set"], s["out_v"])


# ---- one pass ----------------------------------------------------------------------


def run(state):
    case = state["case"]
    op, t = case["op"], state["t"]
    if own:
        ctx, eng = _shared["ctx"], _shared["eng"]
        if op == "rope":
            eng.rope(ctx, state["x"], state["rope"], state["positions"], state["out_v"], backward=case["backward"])
        elif op == "append":
            (q, k, v), row = state["qkv"], state["row"]
            eng.rope_append(ctx, q, k, v, state["rope"], state["positions"], state["cache"], state["out_v"],
                            starts=state["starts"], q_row=row, k_row=row, v_row=row)
        elif op == "paged":
            eng.attn_paged(ctx, state["q"], state["cache"], state["lengths"], state["out_v"], workspace=state["work"])
        else:
            eng.qmatmul_loras(ctx, state["x"], state["w"], state["set"], state["ids"], state["out_v"],
                              workspace=state["work"])
    elif op == "rope":
        state["out"].copy_(_turned(t["x"], t["positions"], state, case, case["backward"]))
    elif op == "append":
        _plain_append(case, t, state)
    elif op == "paged":
        _plain_paged(case, t, state["out"])
    else:
        _plain_loras(case, t, state["out"])
    if op == "append":
        return {"q": state["out"], "k_pages": t["k_pages"], "v_pages": t["v_pages"]}
    return state["out"]


def _turned(x, positions, state, case, backward=False):
    """x [tokens, heads, dim] in 32 bits with its pairs turned; the angles in 64."""
    rot = case["rot"]
    angle = positions.double()[:, None] * state["frequencies"]
    c = (angle.cos() * state["magnitude"]).float()[:, None]
    s = (angle.sin() * state["magnitude"]).float()[:, None]
    if backward:
        s = -s
    x = x.float()
    y = x.clone()
    if case["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    return y


def _plain_append(case, t, state):
    q, k, v = _rows(case, t)
    state["out"].copy_(_turned(q, t["positions"], state, case))
    counts = torch.tensor(_ints(case["lengths"]), device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts, output_size=k.shape[0])
    at = t["positions"].long()
    page, within = t["table"].long()[seq, at // case["page"]], at % case["page"]
    heads_first = case["order"] == "heads"
    for pool, rows in (("k_pages", _turned(k, t["positions"], state, case)), ("v_pages", v)):
        p = t[pool] if not heads_first else t[pool].transpose(1, 2)
        p[page, within] = rows.to(p.dtype)


def _cached(case, t, s, n):
    """Keys and values of sequence s, [kv, n, dim] each."""
    pages = t["table"][s, :-(-n // case["page"])].long()
    for pool in ("k_pages", "v_pages"):
        x = t[pool][pages]
        x = x.transpose(1, 2) if case["order"] == "heads" else x
        yield x.reshape(-1, case["kv"], case["dim"])[:n].transpose(0, 1)


def _plain_paged(case, t, out):
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    for s, n in enumerate(_ints(case["lengths"])):
        if n == 0:
            out[s] = 0
            continue
        k, v = (x.float().contiguous() for x in _cached(case, t, s, n))
        q = t["q"][s].float().view(kv, heads // kv, dim)
        score = torch.matmul(q, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(dim))
        p = torch.exp(score - score.amax(2, keepdim=True))
        out[s] = (torch.matmul(p, v) / p.sum(2, keepdim=True)).view(heads, dim).to(out.dtype)


def _weight(case, t):
    n, k = case["n"], case["k"]
    if case["weight"] == "rowwise8":
        return t["codes"].float() * t["scales"][:, None]
    u = t["codes"]
    if case["weight"] == "affine4":
        u = torch.stack((u & 15, u >> 4), 2)
    return (u.reshape(n, k // 64, 64).float() * t["scales"][:, :, None] + t["biases"][:, :, None]).view(n, k)


def _plain_loras(case, t, out):
    x = t["x"].float()
    y = x @ _weight(case, t).T
    for i in range(case["adapters"]):
        mine = (t["ids"] == i).float()[:, None]
        y += ((x * mine) @ t["a"][i].float().T) @ t["b"][i].float() * t["factors"][i]
    out.copy_(y)


# ---- what a pass cannot do without -----------------------------------------------------


def work(case):
    op = case["op"]
    if op == "rope":
        values = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * values * _SIZE[case["dtype"]] + 4 * case["tokens"] + 4 * case["rot"],
                "flops": 3 * values * case["rot"] // case["dim"]}
    if op == "append":
        heads, kv, dim, counts = case["heads"], case["kv"], case["dim"], _ints(case["lengths"])
        total = sum(counts)
        pages = sum(-(-c // case["page"]) for c in counts)
        return {"bytes": 2 * total * (heads + 2 * kv) * dim * _SIZE[case["dtype"]] + 4 * (total + pages + len(counts) + 1)
                + 4 * case["rot"], "flops": 3 * total * (heads + kv) * case["rot"]}
    if op == "paged":
        heads, kv, dim, size, counts = case["heads"], case["kv"], case["dim"], _SIZE[case["dtype"]], _ints(case["lengths"])
        keys = sum(counts)
        pages = sum(-(-c // case["page"]) for c in counts)
        return {"bytes": 2 * keys * kv * dim * size + 2 * len(counts) * heads * dim * size + 4 * (pages + len(counts)),
                "flops": 4 * keys * heads * dim}
    n, k, rank, rows = case["n"], case["k"], case["rank"], _ints(case["lengths"])
    m, used = sum(rows), min(case["adapters"], len(rows))
    groups = 4 * n if case["weight"] == "rowwise8" else 8 * n * (k // 64)
    return {"bytes": int(n * k * _BYTES[case["weight"]]) + groups + m * k * _SIZE[case["x"]] + m * n * _SIZE[case["y"]]
            + used * rank * (n + k) * _SIZE[case["adapter"]] + 4 * (m + used),
            "flops": 2 * m * n * k + 2 * m * rank * (n + k)}


# ---- the true result, in 64 bits ---------------------------------------------------------


def _turned_exact(x, positions, case, sign=1.0):
    """Complex numbers times exp(i angle)."""
    rot = case["rot"]
    f, magnitude = _frequencies(rot, case["scaling"])
    turn = torch.polar(torch.full_like(f, magnitude).cuda().expand(len(positions), -1).contiguous(),
                       sign * torch.outer(positions.double(), f.cuda()))[:, None]
    x = x.double()
    y = x.clone()
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if case["layout"] == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    t = _inputs(case, seed)
    op = case["op"]
    if op == "rope":
        return _turned_exact(t["x"], t["positions"], case, -1.0 if case["backward"] else 1.0)
    if op == "append":
        q, k, v = _rows(case, t)
        pools = {"k_pages": t["k_pages"].double(), "v_pages": t["v_pages"].double()}
        table, positions, token = t["table"].tolist(), t["positions"].tolist(), 0
        turned = {"k_pages": _turned_exact(k, t["positions"], case), "v_pages": v.double()}
        for s, c in enumerate(_ints(case["lengths"])):
            while c > 0:  # as far as the page goes
                p, o = divmod(positions[token], case["page"])
                m = min(c, case["page"] - o)
                for name, pool in pools.items():
                    rows = turned[name][token:token + m]
                    if case["order"] == "heads":
                        pool[table[s][p], :, o:o + m] = rows.transpose(0, 1)
                    else:
                        pool[table[s][p], o:o + m] = rows
                token, c = token + m, c - m
        return {"q": _turned_exact(q, t["positions"], case), **pools}
    if op == "paged":
        heads, kv = case["heads"], case["kv"]
        out = torch.zeros((len(t["lengths"]), heads, case["dim"]), dtype=torch.float64, device="cuda")
        for s, n in enumerate(_ints(case["lengths"])):
            if n == 0:
                continue
            k, v = _cached(case, t, s, n)
            for h in range(heads):
                j = h * kv // heads
                score = (k[j].double() * t["q"][s, h].double()).sum(1) / math.sqrt(case["dim"])
                out[s, h] = (torch.softmax(score, 0)[:, None] * v[j].double()).sum(0)
        return out
    n, k = case["n"], case["k"]
    if case["weight"] == "rowwise8":
        w = t["codes"].double() * t["scales"].double()[:, None]
    else:
        c = t["codes"].to(torch.int32)
        u = torch.empty((n, k), dtype=torch.float64, device="cuda")
        if case["weight"] == "affine4":
            u[:, 0::2], u[:, 1::2] = (c % 16).double(), (c // 16).double()
        else:
            u[:] = c.double()
        group = torch.arange(k, device="cuda") // 64
        w = u * t["scales"].double()[:, group] + t["biases"].double()[:, group]
    x = t["x"].double()
    y = x @ w.T.contiguous()
    first = 0
    for c in _ints(case["lengths"]):
        i = int(t["ids"][first]) if c else -1
        if i >= 0:
            rows = slice(first, first + c)
            y[rows] += t["factors"][i].double() * ((x[rows] @ t["a"][i].double().T.contiguous()) @ t["b"][i].double())
        first += c
    return y
