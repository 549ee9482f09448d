"""Measured cases of the streaming operators: rotary positions over several axes, the append to a paged
key/value cache, attention of a chunk of new tokens over that cache, and attention with a sliding window
and sinks over contiguous keys.

Each case is one call as a streaming program makes it. `run` computes it with elementary torch operations in
32 bits (angles in 64), or, where `own` is true, with this package's operators; `exact` gives the definition
in 64 bits. Head dim 128 throughout, as everywhere in the package.
"""
import math
import random

import numpy as np
import torch

own = False

DIM = 128
SCALE = DIM ** -0.5
LOG2E = 1.4426950408889634
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}

# The head dims that turn with each axis. "video": frame, row and column, each with its own frequencies,
# dims (2i, 2i + 1) in pairs. "video-wide": a narrow frame axis and a small base. "text-image": one
# frequency scale over the head, its pairs (i, i + 64) shared out to the axes. "line": one axis.
AXES = {
    "video": {"sections": (44, 42, 42), "theta": 10000.0, "paired": True, "shared": False},
    "video-wide": {"sections": (16, 56, 56), "theta": 256.0, "paired": True, "shared": False},
    "text-image": {"sections": (32, 48, 48), "theta": 1000000.0, "paired": False, "shared": True},
    "line": {"sections": (128,), "theta": 500000.0, "paired": False, "shared": True},
}


def listed():
    return [
        # One new token a sequence, behind a long text and image context: the latency of a decoding step.
        {"name": "rotary-token", "op": "rotary", "axes": "text-image", "batch": 2, "heads": 40, "kv_heads": 8, "tokens": 1,
         "far": 1000000, "dtype": "bf16", "inverse": False, "projected": True},
        # Queries and keys of a whole 720p layer, as the projections leave them ([B, N, H, 128]).
        {"name": "rotary-layer", "op": "rotary", "axes": "video", "batch": 1, "heads": 12, "kv_heads": 12, "tokens": 75600,
         "far": 0, "dtype": "bf16", "inverse": False, "projected": True},
        # The gradient of three frames' queries and keys: the turn back.
        {"name": "rotary-gradient", "op": "rotary", "axes": "video-wide", "batch": 2, "heads": 40, "kv_heads": 40, "tokens": 10799,
         "far": 77, "dtype": "fp16", "inverse": True, "projected": False},
        # A decoding step of 64 sequences writes its keys and values into pages of 64.
        {"name": "append-token", "op": "append", "axes": "line", "seqs": 64, "longest": 1, "held": 400, "heads": 32, "kv_heads": 8,
         "page": 64, "dtype": "bf16", "spread": 1},
        # Three 720p frames join a stream's cache.
        {"name": "append-frames", "op": "append", "axes": "video", "seqs": 1, "longest": 10800, "held": 3600, "heads": 12,
         "kv_heads": 12, "page": 128, "dtype": "bf16", "spread": 2},
        # A decoding step of a batch with shared heads and ragged contexts.
        {"name": "chunk-token", "op": "chunk", "seqs": 48, "longest": 1, "held": 16000, "heads": 32, "kv_heads": 8, "page": 64,
         "window": 0, "sinks": 0, "block": 1, "dtype": "bf16", "spread": 3},
        # One token against one very long cache of small pages: little to share out over the SMs but the keys.
        {"name": "chunk-token-long", "op": "chunk", "seqs": 1, "longest": 1, "held": 131001, "heads": 12, "kv_heads": 12, "page": 16,
         "window": 0, "sinks": 0, "block": 1, "dtype": "bf16", "spread": 4},
        # Prompt chunks and single tokens in one batch.
        {"name": "chunk-ragged", "op": "chunk", "seqs": 9, "longest": 701, "held": 7300, "heads": 16, "kv_heads": 4, "page": 16,
         "window": 0, "sinks": 0, "block": 1, "dtype": "fp16", "spread": 5},
        # A new 720p frame against the stream so far: full attention within the frame and to all before it.
        {"name": "chunk-frame", "op": "chunk", "seqs": 1, "longest": 3600, "held": 72000, "heads": 12, "kv_heads": 12, "page": 128,
         "window": 0, "sinks": 0, "block": 3600, "dtype": "bf16", "spread": 6},
        # One token of each of four streams against a rolling window and the first tokens.
        {"name": "window-token", "op": "window", "batch": 4, "heads": 40, "kv_heads": 8, "tokens": 1, "keys": 8191, "window": 4096,
         "sinks": 4, "block": 1, "dtype": "bf16"},
        # A causal pass over a text with a narrow window.
        {"name": "window-text", "op": "window", "batch": 1, "heads": 16, "kv_heads": 4, "tokens": 8191, "keys": 8191,
         "window": 1024, "sinks": 4, "block": 1, "dtype": "fp16"},
        # Five 720p frames, each against itself, the frame before it and the first tokens.
        {"name": "window-frames", "op": "window", "batch": 1, "heads": 12, "kv_heads": 12, "tokens": 18000, "keys": 18000,
         "window": 7200, "sinks": 256, "block": 3600, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_heads(rng):
    kv = rng.choice((1, 2, 4, 5, 8, 12))
    return kv * rng.choice((1, 1, 2, 4, 5, 8)), kv


def _draw_one(rng):
    op = rng.choice(("rotary", "append", "chunk", "chunk", "window", "window"))
    heads, kv = _draw_heads(rng)
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "rotary":
        return {"op": op, "axes": rng.choice(tuple(AXES)), "batch": rng.choice((1, 1, 2, 3)), "heads": heads, "kv_heads": kv,
                "tokens": _log(rng, 1, 75600), "far": rng.choice((0, 13, 4099, 1000003)), "dtype": rng.choice((dtype, "fp32")),
                "inverse": rng.random() < 0.4, "projected": rng.random() < 0.5}
    if op == "append":
        return {"op": op, "axes": rng.choice(tuple(AXES)), "seqs": rng.choice((1, 2, 7, 33, 64)), "longest": _log(rng, 1, 4096),
                "held": _log(rng, 1, 4000), "heads": heads, "kv_heads": kv, "page": rng.choice((16, 32, 64, 128, 256)),
                "dtype": dtype, "spread": rng.randrange(1 << 20)}
    if op == "chunk":
        longest = rng.choice((1, 1, 2, 5, _log(rng, 1, 3600), _log(rng, 1, 3600)))
        windowed = rng.random() < 0.4
        return {"op": op, "seqs": rng.choice((1, 2, 7, 24, 61)), "longest": longest, "held": _log(rng, 1, 100000), "heads": heads,
                "kv_heads": kv, "page": rng.choice((16, 32, 64, 128, 256)), "window": _log(rng, 1, 5000) if windowed else 0,
                "sinks": rng.choice((0, 4, 131)) if windowed else 0, "block": rng.choice((1, 1, 1, 37, 256)), "dtype": dtype,
                "spread": rng.randrange(1 << 20)}
    keys = _log(rng, 1, 20000)
    tokens = rng.choice((1, min(keys, 3), keys, keys, max(1, keys // 3)))
    return {"op": op, "batch": rng.choice((1, 1, 2, 3)), "heads": heads, "kv_heads": kv, "tokens": tokens, "keys": keys,
            "window": rng.choice((0, _log(rng, 1, 8000), _log(rng, 1, 8000))), "sinks": rng.choice((0, 1, 4, 200)),
            "block": rng.choice((1, 1, 1, 53, 1024)), "dtype": dtype}


def _plain_bytes(case):
    """Of the scores, or of the cache and the rows, as the plain form holds them."""
    if case["op"] == "chunk":
        return 4 * case["seqs"] * (case["longest"] + case["held"]) * (case["heads"] * case["longest"] + 2 * DIM * case["kv_heads"])
    if case["op"] == "window":
        return 4 * case["batch"] * case["heads"] * case["tokens"] * case["keys"]
    if case["op"] == "append":
        return 8 * case["seqs"] * (case["longest"] + case["held"]) * DIM * (case["heads"] + 2 * case["kv_heads"])
    return 8 * case["batch"] * case["tokens"] * DIM * (case["heads"] + case["kv_heads"])


def draw(rng):
    """A case that costs no more than the largest listed one of its operator."""
    most = {op: max(_plain_bytes(c) for c in listed() if c["op"] == op) for op in ("rotary", "append", "chunk", "window")}
    while True:
        case = _draw_one(rng)
        if _plain_bytes(case) <= most[case["op"]] / 2:
            return case


# ---- sizes that follow from a case ------------------------------------------------------------------


def _chunks(case):
    """(chunk lengths, cached lengths after the chunk) of a ragged batch: one sequence has both in full."""
    rng = random.Random(case["spread"])
    new = [case["longest"]] + [rng.randint(1, case["longest"]) for _ in range(case["seqs"] - 1)]
    held = [case["held"]] + [rng.randint(0, case["held"]) for _ in range(case["seqs"] - 1)]
    return new, [a + b for a, b in zip(new, held)]


def _visible(first, tokens, keys, window, sinks, block):
    """(pairs that attend, keys that any query sees) of queries at first, first + 1, ... over `keys` keys."""
    end = ((first + np.arange(tokens, dtype=np.int64)) // block + 1) * block
    low = np.maximum(end - window, 0) if window else np.zeros_like(end)
    end = np.clip(end, 0, keys)
    low = np.minimum(low, end)
    head = np.minimum(np.minimum(sinks if window else 0, end), low)
    pairs = int((end - low + head).sum())
    seen = int(end.max() - low.min() + min(head.max(), low.min())) if tokens else 0
    return pairs, seen


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "rotary":
        rows = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"])
        axes = len(AXES[case["axes"]]["sections"])
        return {"bytes": 2 * rows * DIM * e + case["tokens"] * axes * 4, "flops": rows * DIM * 3}
    if case["op"] == "append":
        new, _ = _chunks(case)
        rows = sum(new) * (case["heads"] + 2 * case["kv_heads"])
        return {"bytes": 2 * rows * DIM * e + sum(new) * 4 * len(AXES[case["axes"]]["sections"]),
                "flops": sum(new) * (case["heads"] + case["kv_heads"]) * DIM * 3}
    if case["op"] == "chunk":
        new, held = _chunks(case)
        seen = [_visible(n - m, m, n, case["window"], case["sinks"], case["block"]) for m, n in zip(new, held)]
        pairs, keys, rows = sum(p for p, _ in seen), sum(k for _, k in seen), sum(new) * case["heads"]
    else:
        pairs, keys = _visible(case["keys"] - case["tokens"], case["tokens"], case["keys"], case["window"], case["sinks"],
                               case["block"])
        pairs, keys, rows = pairs * case["batch"], keys * case["batch"], case["batch"] * case["tokens"] * case["heads"]
    return {"bytes": rows * (2 * DIM * e + 4) + 2 * keys * case["kv_heads"] * DIM * e, "flops": 4 * DIM * pairs * case["heads"]}


# ---- inputs ------------------------------------------------------------------------------------------


def _positions(case, tokens, gen, device):
    """int32 [tokens, axes]: the (frame, row, column) of a token of 45 x 80 frames, or one or three text positions."""
    axes = len(AXES[case["axes"]]["sections"])
    n = torch.arange(tokens, device=device)
    far = case.get("far", 11)
    if axes == 3:
        p = torch.stack((n // 3600 + far, n // 80 % 45, n % 80), -1)
    else:
        p = (n + far)[:, None]
    return (p + torch.randint(0, 3, (1, axes), generator=gen, device=device)).to(torch.int32)


def prepare(case, seed):
    device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=device).manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device, dtype=torch.float32 if dtype == torch.float32 else dtype)

    state = {"case": case}
    if case["op"] == "rotary":
        for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
            if case["projected"]:
                state[name] = normal(case["batch"], case["tokens"], heads, DIM).transpose(1, 2)
            else:
                state[name] = normal(case["batch"], heads, case["tokens"], DIM)
        state["positions"] = _positions(case, case["tokens"], gen, device)
        return state
    if case["op"] == "window":
        state["q"] = normal(case["batch"], case["heads"], case["tokens"], DIM)
        state["k"] = normal(case["batch"], case["kv_heads"], case["keys"], DIM)
        state["v"] = normal(case["batch"], case["kv_heads"], case["keys"], DIM)
        return state
    new, held = _chunks(case)
    tokens, page = sum(new), case["page"]
    width = -(-max(held) // page)
    used = [-(-n // page) for n in held]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=gen, device=device).to(torch.int32)
    place = np.full((case["seqs"], width), -1, dtype=np.int64)
    at = 0
    for s, n in enumerate(used):
        place[s, :n] = np.arange(at, at + n)
        at += n
    place = torch.from_numpy(place).to(device)
    state["table"] = torch.where(place >= 0, order[place.clamp(min=0)], torch.zeros_like(order[:1])).contiguous()
    state["starts"] = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device=device)
    state["lengths"] = torch.tensor(held, dtype=torch.int32, device=device)
    state["keys"] = normal(pages, case["kv_heads"], page, DIM)
    state["values"] = normal(pages, case["kv_heads"], page, DIM)
    state["q"] = normal(tokens, case["heads"], DIM)
    if case["op"] == "append":
        state["k"] = normal(tokens, case["kv_heads"], DIM)
        state["v"] = normal(tokens, case["kv_heads"], DIM)
        state["positions"] = _positions(case, tokens, gen, device)
    return state


# ---- the operators, plain --------------------------------------------------------------------------------


def _angles(positions, axes):
    """float64 [..., 64]: the angle of each pair of head dims."""
    parts, done = [], 0
    for a, dims in enumerate(axes["sections"]):
        i = torch.arange(dims // 2, dtype=torch.float64, device=positions.device)
        power = (i + done) * 2 / DIM if axes["shared"] else i * 2 / dims
        parts.append(positions[..., a:a + 1].double() * axes["theta"] ** -power)
        done += dims // 2
    return torch.cat(parts, -1)


def _turn(x, angles, axes, inverse, kind=torch.float32):
    """x [..., 128] turned by angles [..., 64], in `kind`."""
    cos, sin = angles.cos().to(kind), angles.sin().to(kind)
    if inverse:
        sin = -sin
    x = x.to(kind)
    if axes["paired"]:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    a, b = x[..., :DIM // 2], x[..., DIM // 2:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _mask(first, tokens, keys, window, sinks, block, lengths):
    """bool [B, tokens, keys] of queries at first[b], first[b] + 1, ... over lengths[b] of the keys."""
    end = (torch.div(first[:, None] + torch.arange(tokens, device=first.device), block, rounding_mode="floor") + 1) * block
    j = torch.arange(keys, device=first.device)
    seen = (j < end[..., None]) & (j < lengths[:, None, None])
    if window:
        seen &= (j >= end[..., None] - window) | (j < sinks)
    return seen


def _attend(q, k, v, seen, dtype):
    """q [B, Hk, G, N, 128] float, k and v [B, Hk, K, 128] float, seen [B, N, K] -> outputs in `dtype`, base-2 lse."""
    s = torch.matmul(q * SCALE, k[:, :, None].transpose(-1, -2))
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s, v[:, :, None]) / total.masked_fill(total == 0, 1.0)
    return o.to(dtype), ((top + total.log()) * LOG2E)[..., 0]


def _window_plain(state):
    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    b, h, n, _ = q.shape
    lengths = torch.full((b,), k.shape[2], device=q.device)
    seen = _mask(lengths - n, n, k.shape[2], case["window"], case["sinks"], case["block"], lengths)
    o, lse = _attend(q.float().unflatten(1, (k.shape[1], -1)), k.float(), v.float(), seen, q.dtype)
    return o.flatten(1, 2), lse.flatten(1, 2)


def _chunk_plain(state):
    case, q, starts, lengths = state["case"], state["q"], state["starts"].long(), state["lengths"].long()
    kv, longest = case["kv_heads"], case["longest"]
    k, v = (state[x][state["table"].long()].transpose(1, 2).flatten(2, 3).float() for x in ("keys", "values"))
    new = starts[1:] - starts[:-1]
    rows = (starts[:-1, None] + torch.arange(longest, device=q.device)).clamp(max=q.shape[0] - 1)
    padded = q[rows].float().permute(0, 2, 1, 3).unflatten(1, (kv, -1))
    seen = _mask(lengths - new, longest, k.shape[2], case["window"], case["sinks"], case["block"], lengths)
    o, lse = _attend(padded, k, v, seen, q.dtype)
    t = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(starts, t, right=True) - 1
    at = t - starts[seq]
    return o.flatten(1, 2).transpose(1, 2)[seq, at], lse.flatten(1, 2).transpose(1, 2)[seq, at]


def _append_plain(state):
    axes = AXES[state["case"]["axes"]]
    starts, lengths, page = state["starts"].long(), state["lengths"].long(), state["case"]["page"]
    angles = _angles(state["positions"], axes)[:, None]
    q, k = (_turn(state[x], angles, axes, False).to(state[x].dtype) for x in ("q", "k"))
    t = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(starts, t, right=True) - 1
    at = lengths[seq] - starts[seq + 1] + t
    where = state["table"].long()[seq, at // page]
    state["keys"][where, :, at % page] = k
    state["values"][where, :, at % page] = state["v"]
    return q, state["keys"], state["values"]


def _rotary_plain(state):
    axes = AXES[state["case"]["axes"]]
    angles = _angles(state["positions"], axes)
    return tuple(_turn(state[x], angles, axes, state["case"]["inverse"]).to(state[x].dtype) for x in ("q", "k"))


# ---- the operators, as a user calls them -------------------------------------------------------------------


def _own(state):
    from ab_attention_b200 import KVCache, RotaryAxes, append_kv, apply_rotary, chunk_attention, window_attention

    case = state["case"]
    if case["op"] == "rotary":
        return apply_rotary(state["q"], state["k"], state["positions"], RotaryAxes(**AXES[case["axes"]]), inverse=case["inverse"])
    if case["op"] == "window":
        return window_attention(state["q"], state["k"], state["v"], window=case["window"] or None, sinks=case["sinks"],
                                block=case["block"], return_lse=True)
    cache = KVCache(state["keys"], state["values"])
    if case["op"] == "append":
        q = append_kv(cache, state["k"], state["v"], state["table"], state["starts"], state["lengths"],
                      positions=state["positions"], axes=RotaryAxes(**AXES[case["axes"]]), q=state["q"])
        return q, cache.keys, cache.values
    return chunk_attention(state["q"], cache, state["table"], state["starts"], state["lengths"], longest=case["longest"],
                           window=case["window"] or None, sinks=case["sinks"], block=case["block"], return_lse=True)


def run(state):
    if own:
        return _own(state)
    return {"rotary": _rotary_plain, "append": _append_plain, "chunk": _chunk_plain, "window": _window_plain}[state["case"]["op"]](state)


# ---- the definition in 64 bits -------------------------------------------------------------------------------


def _exact_turn(x, positions, name, inverse):
    """Each pair as a complex number times exp(i * angle)."""
    axes = AXES[name]
    turns = []
    for a, dims in enumerate(axes["sections"]):
        before = sum(axes["sections"][:a]) // 2
        for i in range(dims // 2):
            power = 2 * (before + i) / DIM if axes["shared"] else 2 * i / dims
            turns.append(positions[:, a].double() / axes["theta"] ** power)
    turn = torch.stack(turns, 1)
    turn = torch.polar(torch.ones_like(turn), -turn if inverse else turn)
    x = x.double()
    if axes["paired"]:
        return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
    z = torch.complex(x[..., :64].contiguous(), x[..., 64:].contiguous()) * turn
    return torch.cat((z.real, z.imag), -1)


def _exact_rows(q, k, v, first, window, sinks, block):
    """q [N, H, 128] at first, first + 1, ... over k and v [K, Hk, 128], a head and some rows at a time."""
    n, heads, _ = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(n, heads, DIM, dtype=torch.float64, device=q.device)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64, device=q.device)
    j = torch.arange(k.shape[0], device=q.device)
    some = max(1, (1 << 28) // max(1, k.shape[0]))
    for h in range(heads):
        kh, vh = k[:, h // group].double(), v[:, h // group].double()
        for a in range(0, n, some):
            p = first + torch.arange(a, min(n, a + some), device=q.device)
            end = (p // block + 1) * block
            hidden = j[None] >= end[:, None]
            if window:
                hidden |= (j[None] < (end - window)[:, None]) & (j[None] >= sinks)
            s = (q[a:a + some, h].double() @ kh.T / math.sqrt(DIM)).masked_fill(hidden, -math.inf)
            l = torch.logsumexp(s, -1)
            w = torch.exp(s - torch.where(l == -math.inf, 0.0, l)[:, None])
            out[a:a + some, h] = w @ vh
            lse[a:a + some, h] = l / math.log(2.0)
    return out, lse


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        return tuple(_exact_turn(state[x], state["positions"], case["axes"], case["inverse"]) for x in ("q", "k"))
    rules = {x: case[x] for x in ("window", "sinks", "block")} if case["op"] in ("chunk", "window") else {}
    if case["op"] == "window":
        both = [_exact_rows(*(state[x][b].transpose(0, 1) for x in ("q", "k", "v")), case["keys"] - case["tokens"], **rules)
                for b in range(case["batch"])]
        return torch.stack([o.transpose(0, 1) for o, _ in both]), torch.stack([l.T for _, l in both])
    new, held = _chunks(case)
    page, at = case["page"], 0
    if case["op"] == "append":
        q, k = (_exact_turn(state[x].transpose(0, 1), state["positions"], case["axes"], False).transpose(0, 1) for x in ("q", "k"))
        keys, values = state["keys"].double(), state["values"].double()
        for s, (m, n) in enumerate(zip(new, held)):
            for p in range((n - m) // page, (n - 1) // page + 1):
                low, high = max(n - m, p * page), min(n, (p + 1) * page)
                rows = slice(at + low - (n - m), at + high - (n - m))
                to = int(state["table"][s, p])
                keys[to, :, low - p * page:high - p * page] = k[rows].transpose(0, 1)
                values[to, :, low - p * page:high - p * page] = state["v"][rows].transpose(0, 1).double()
            at += m
        return q, keys, values
    outs, lses = [], []
    for s, (m, n) in enumerate(zip(new, held)):
        pages = state["table"][s, :-(-n // page)].long()
        k, v = (state[x][pages].transpose(1, 2).flatten(0, 1)[:n] for x in ("keys", "values"))
        o, l = _exact_rows(state["q"][at:at + m], k, v, n - m, **rules)
        outs.append(o)
        lses.append(l)
        at += m
    return torch.cat(outs), torch.cat(lses)
