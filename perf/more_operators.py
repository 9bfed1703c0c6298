"""Calls of the operators that keep a long request's memory bounded, for measuring their performance.

A batch is held as the attention operators hold one: rows of all sequences one after another, offsets, and a paged cache
behind a block table.  `write` rotates a step's queries and keys by their positions and puts keys and values into their
slots, `rotate` does the same to the rows of a training step, with the gradients.  `weights` sums, for each key of the
cache, the softmax weights that a step's rows gave it; `evict` says which keys a request of too many keeps and where they
go, `move` moves them.  `state` carries a recurrent layer's state over the sequences (`scan` with its backward pass).

`run` computes them from elementary torch operations, or where `own` is true by the library's calls.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# Scores of the plain form that one call may hold (requests x heads x new rows x longest), in values.
MOST_SCORES = 1 << 30
MOST_ROTATED = 1 << 27  # items of a rotation
MOST_CACHE = 1 << 28    # items of a cache's keys
MOST_SCAN = 1 << 27     # items of a recurrence


def listed():
    return [
        # One decoding step of a small batch in buffers of a fixed capacity, at far positions.  Latency.
        {"name": "write_decode_64", "op": "write", "type": "bf16", "tokens": 64, "padding": 8, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "page": 16, "far": 131_000, "scale": 1.0, "factor": 1.0},
        # A step of prompts, half of each head rotated, pairs side by side, frequencies stretched for long contexts.
        {"name": "write_prompt_32k", "op": "write", "type": "f16", "tokens": 32_749, "padding": 0, "heads": 16,
         "kv_heads": 4, "dim": 128, "rotary": 64, "interleaved": True, "page": 64, "far": 32_749, "scale": 4.0,
         "factor": 1.14},
        # A training step's rotations and their gradients, in the fused projection's rows.
        {"name": "rotate_train_11k", "op": "rotate", "type": "bf16", "tokens": 11_059, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "far": 4096, "scale": 1.0, "factor": 1.0},
        # A decoding step of a large batch adds its weights to the keys' sums.
        {"name": "weights_decode_256", "op": "weights", "type": "bf16", "requests": 256, "low": 200, "high": 4000,
         "new_low": 1, "new_high": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "decay": 0.98, "mix": 1},
        # The last 32 rows of three long prompts vote on all of their keys.
        {"name": "weights_window_3", "op": "weights", "type": "f16", "requests": 3, "low": 9000, "high": 60_000,
         "new_low": 32, "new_high": 32, "heads": 16, "kv_heads": 4, "dim": 128, "page": 64, "decay": 1.0, "mix": 2},
        # A few keys too many in each request of a batch that is held at 1,024.  Latency.
        {"name": "evict_held_256", "op": "evict", "requests": 256, "low": 1025, "high": 1040, "keep": 1024, "share": 1.0,
         "first": 4, "recent": 64, "page": 16, "mix": 3},
        # Long prompts cut to a quarter.
        {"name": "evict_prompts_16", "op": "evict", "requests": 16, "low": 2000, "high": 131_000, "keep": 131_000,
         "share": 0.25, "first": 4, "recent": 256, "page": 64, "mix": 4},
        # The rows of such a batch: up to 16 a request.
        {"name": "move_held_256", "op": "move", "type": "f16", "requests": 256, "low": 1025, "high": 1040, "keep": 1024,
         "share": 1.0, "kv_heads": 8, "dim": 128, "page": 16, "mix": 5},
        # The rows of long prompts that are cut.
        {"name": "move_prompts_16", "op": "move", "type": "bf16", "requests": 16, "low": 3000, "high": 40_000,
         "keep": 40_000, "share": 0.25, "kv_heads": 8, "dim": 128, "page": 64, "mix": 6},
        # A decoding step: one token for each request's state.  Latency.
        {"name": "state_step_256", "op": "state", "type": "bf16", "sequences": 256, "low": 1, "high": 1, "channels": 4096,
         "mix": 7},
        # Fine-tuning on short examples, in 32 bits, of a width that no vector divides.
        {"name": "scan_short_f32", "op": "scan", "type": "f32", "sequences": 7, "low": 60, "high": 517, "channels": 770,
         "mix": 8},
        # A training step over long documents.
        {"name": "scan_long_bf16", "op": "scan", "type": "bf16", "sequences": 6, "low": 700, "high": 16_384,
         "channels": 4096, "mix": 9},
    ]


def _size(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["write", "rotate", "weights", "weights", "evict", "move", "state", "scan", "scan"])
    mix = rng.randrange(1 << 20)
    if op in ("state", "scan"):
        channels = rng.choice([_size(rng, 16, 8192), 64 * _size(rng, 1, 96), 4096, 2048, 1000])
        high = _size(rng, 1, 32_768) if rng.random() < 0.8 else 1
        sequences = _size(rng, 1, max(1, min(512, MOST_SCAN // 2 // (high * channels))))
        high = min(high, MOST_SCAN // 2 // channels)
        return {"op": op, "type": rng.choice(["bf16", "bf16", "f16", "f32"]), "sequences": sequences,
                "low": max(1, high // rng.choice([1, 2, 8, 40])), "high": high, "channels": channels, "mix": mix}
    page = rng.choice([8, 16, 16, 24, 32, 64, 128, 256])
    if op == "evict":
        high = _size(rng, 40, 131_000)
        requests = _size(rng, 1, max(1, min(512, 1_600_000 // high)))
        return {"op": op, "requests": requests, "low": max(1, high // rng.choice([1, 3, 20])), "high": high,
                "keep": _size(rng, 1, high), "share": rng.choice([1.0, 0.9, 0.5, 0.25, 0.1]),
                "first": rng.choice([0, 1, 4, 37]), "recent": _size(rng, 1, 1000), "page": page, "mix": mix}
    dim = rng.choice([64, 128, 128, 128, 32, 80, 96, 112, 120])
    group = rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    heads = group * kv_heads
    kind = rng.choice(["bf16", "bf16", "f16"])
    if op == "move":
        high = _size(rng, 40, 40_000)
        requests = _size(rng, 1, max(1, min(512, MOST_CACHE // (high * kv_heads * dim))))
        return {"op": op, "type": kind, "requests": requests, "low": max(1, high // rng.choice([1, 3, 20])), "high": high,
                "keep": _size(rng, 1, high), "share": rng.choice([1.0, 0.9, 0.5, 0.25, 0.1]), "kv_heads": kv_heads,
                "dim": dim, "page": page, "mix": mix}
    if op == "weights":
        new_high = rng.choice([1, 1, 1, 4, 32, 100])
        high = _size(rng, max(16, new_high), 60_000)
        most = min(MOST_CACHE // 2 // (high * kv_heads * dim), MOST_SCORES // (high * heads * new_high))
        if most < 1:
            high, most = max(16, new_high), 64
        requests = _size(rng, 1, max(1, min(512, most)))
        return {"op": op, "type": kind, "requests": requests, "low": max(new_high, high // rng.choice([1, 3, 20])),
                "high": high, "new_low": rng.choice([1, new_high]), "new_high": new_high, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "page": page, "decay": rng.choice([1.0, 0.9]), "mix": mix}
    rotary = rng.choice([dim, dim, dim // 2, 2 * rng.randrange(1, dim // 2 + 1)])
    tokens = _size(rng, 1, MOST_ROTATED // 3 // ((heads + 2 * kv_heads) * dim))
    case = {"op": op, "type": kind, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "interleaved": rng.random() < 0.4, "far": _size(rng, tokens, 1_048_576) if tokens < 1_048_576
            else tokens, "scale": rng.choice([1.0, 1.0, 4.0, 32.0]), "factor": rng.choice([1.0, 1.0, 1.2])}
    return case | {"page": page, "padding": rng.choice([0, 0, 1, 37])} if op == "write" else case


# ---- inputs ----------------------------------------------------------------------------------------
def _lengths(count, low, high, mix):
    """Lengths spread over their logarithm, the longest of them `high`.  The case alone decides them."""
    rng = random.Random(mix)
    return [high] + [_size(rng, low, high) for _ in range(count - 1)]


def _shuffled(values, seed):
    values = list(values)
    random.Random(seed).shuffle(values)
    return values


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _offsets(lengths):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return _ints(total)


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _rows(g, dtype, rows, heads, dim, gain=1.0, outliers=False):
    """Normal rows; `outliers`: one channel in 32 of four times the width, as learned keys have them."""
    x = _normal(g, rows, heads, dim)
    if outliers:
        x[..., 5::32] *= 4.0
    return (x * gain).to(dtype)


def _frequencies(case):
    """Radians a position, of each pair: powers of 10,000, stretched by `scale`."""
    half = case["rotary"] // 2
    i = torch.arange(half, dtype=torch.float64)
    return (10000.0 ** (-i / half) / case["scale"]).cuda()


def _spans(g, case, tokens):
    """Positions up to `far`, and requests: each row of few another request's, otherwise runs of 1,000 consecutive ones."""
    run = 1 if tokens <= 512 else max(1, min(1000, case["far"] // 2))
    starts = torch.randint(0, max(1, case["far"] - run), (-(-tokens // run),), device="cuda", generator=g)
    t = torch.arange(tokens, device="cuda")
    return (starts[t // run] + t % run).to(torch.int32), (t // run).to(torch.int32)


def _prepare_write(case, seed):
    g, dtype, page = _generator(seed), DTYPE[case["type"]], case["page"]
    real, total = case["tokens"], case["tokens"] + case["padding"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    pages = -(-real // page) + 32
    order = torch.randperm(pages, device="cuda", generator=g)
    t = torch.arange(total, device="cuda")
    slots = order[(t // page).clamp_max(pages - 1)] * page + t % page
    positions, requests = _spans(g, case, total)
    # Requests that had keys evicted: their positions are ahead of their lengths.
    shifts = torch.randint(0, 1000, (total,), device="cuda", generator=g).to(torch.int32)
    shifts[::2] = 0
    slots[real:], requests[real:], positions[real:] = -1, -1, 0
    fused = _rows(g, dtype, total, h + 2 * hk, d)
    cache = lambda: torch.zeros(pages, page, hk, d, dtype=dtype, device="cuda")
    return {"q": fused[:, :h], "key": fused[:, h:h + hk], "value": fused[:, h + hk:], "positions": positions,
            "requests": requests, "shifts": shifts, "frequencies": _frequencies(case), "slots": slots,
            "q_out": torch.zeros(total, h, d, dtype=dtype, device="cuda"), "key_cache": cache(), "value_cache": cache(),
            "slot_positions": torch.full((pages, page), -1, dtype=torch.int32, device="cuda")}


def _prepare_rotate(case, seed):
    g, dtype, tokens = _generator(seed), DTYPE[case["type"]], case["tokens"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    fused, back = _rows(g, dtype, tokens, h + 2 * hk, d), torch.zeros(tokens, h + 2 * hk, d, dtype=dtype, device="cuda")
    like = lambda n: torch.empty(tokens, n, d, dtype=dtype, device="cuda")
    return {"q": fused[:, :h], "key": fused[:, h:h + hk], "positions": _spans(g, case, tokens)[0],
            "frequencies": _frequencies(case), "q_out": like(h), "k_out": like(hk), "dq_out": _rows(g, dtype, tokens, h, d),
            "dk_out": _rows(g, dtype, tokens, hk, d), "dq": back[:, :h], "dk": back[:, h:h + hk]}


def _tables(g, lengths, page):
    """A block table over pages in any order, and how many there are."""
    used = [-(-n // page) for n in lengths]
    width, pages = max(used), sum(used) + 7
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    have = _ints(used, torch.int64)[:, None]
    column = torch.arange(width, device="cuda")[None, :]
    filled = column < have
    table[filled] = order[(have.cumsum(0) - have + column)[filled]]
    return table, pages


def _paged_lengths(case):
    kv = _lengths(case["requests"], case["low"], case["high"], case["mix"])
    new = _lengths(case["requests"], case["new_low"], case["new_high"], case["mix"] + 1)
    return list(zip(kv, new))


def _skewed(g, *shape):
    """Sums of weights as caches gather them: a few large, most of them small, some equal to others."""
    return (torch.exp(1.5 * _normal(g, *shape)) * 64).round() / 64


def _prepare_weights(case, seed):
    g, dtype, page = _generator(seed), DTYPE[case["type"]], case["page"]
    both = _shuffled(_paged_lengths(case), seed)
    kv, new = [a for a, _ in both], [b for _, b in both]
    h, hk, d, t = case["heads"], case["kv_heads"], case["dim"], sum(new)
    table, pages = _tables(g, kv, page)
    s = {"q": _rows(g, dtype, t, h, d, 1.5), "table": table, "q_offsets": _offsets(new), "kv": _ints(kv),
         "known": _ints([a - b for a, b in both]), "longest": max(kv), "new_longest": max(new),
         "key_cache": _rows(g, dtype, pages * page, hk, d, outliers=True).view(pages, page, hk, d),
         "before": _skewed(g, pages, page), "after": torch.zeros(pages, page, device="cuda")}
    # The log-sums that the step's attention gave, rounded from 64 bits.
    s["lse"] = torch.full((h, t), -math.inf, device="cuda")
    at = 0
    for r, (m, n) in enumerate(both):
        keys = s["key_cache"][table[r, :-(-m // page)].long()].flatten(0, 1)[:m]
        late = torch.arange(m, device="cuda") > torch.arange(n, device="cuda")[:, None] + (m - n)
        for head in range(hk):
            rows = s["q"][at:at + n, head * (h // hk):(head + 1) * (h // hk)].transpose(0, 1).float()
            scores = (rows.reshape(-1, d) @ keys[:, head].float().t()).view(-1, n, m) * d ** -0.5
            s["lse"][head * (h // hk):(head + 1) * (h // hk), at:at + n] = \
                torch.logsumexp(scores.masked_fill_(late, -math.inf), -1)
        at += n
    return s


def _kept(case, n):
    return max(1, min(n, case["keep"], math.ceil(n * case["share"])))


def _prepare_evict(case, seed):
    g, page = _generator(seed), case["page"]
    lengths = _shuffled(_lengths(case["requests"], case["low"], case["high"], case["mix"]), seed)
    table, pages = _tables(g, lengths, page)
    keep = [_kept(case, n) for n in lengths]
    gone = [random.Random(seed + i).choice([0, 0, 977]) for i in range(len(lengths))]
    # Positions of the keys: in order but for a twentieth, which earlier evictions have moved.
    positions = torch.full((pages, page), -1, dtype=torch.int32, device="cuda")
    for r, n in enumerate(lengths):
        p = torch.arange(n, device="cuda") + gone[r]
        some = torch.randperm(n, device="cuda", generator=g)[:n // 20]
        p[some] = p[some.sort().values]
        at = torch.arange(n, device="cuda")
        positions[table[r, at // page].long(), at % page] = p.to(torch.int32)
    width = max(1, max(min(k, n - k) for k, n in zip(keep, lengths)))
    count = len(lengths)
    return {"table": table, "kv": _ints(lengths), "keep": _ints(keep), "shifts": _ints(gone), "positions": positions,
            "weights": _skewed(g, pages, page), "longest": max(lengths),
            "move_from": torch.empty(count, width, dtype=torch.int64, device="cuda"),
            "move_to": torch.empty(count, width, dtype=torch.int64, device="cuda"),
            "kept": torch.empty(count, dtype=torch.int32, device="cuda"),
            "shifts_out": torch.empty(count, dtype=torch.int32, device="cuda"),
            "released": torch.full((pages,), -1, dtype=torch.int32, device="cuda"),
            "counts": torch.empty(2, dtype=torch.int32, device="cuda")}


def _prepare_move(case, seed):
    g, dtype, page = _generator(seed), DTYPE[case["type"]], case["page"]
    hk, d = case["kv_heads"], case["dim"]
    lengths = _shuffled(_lengths(case["requests"], case["low"], case["high"], case["mix"]), seed)
    table, pages = _tables(g, lengths, page)
    keep = [_kept(case, n) for n in lengths]
    width = max(1, max(min(k, n - k) for k, n in zip(keep, lengths)))
    moves = [torch.full((len(lengths), width), -1, dtype=torch.int64, device="cuda") for _ in range(2)]
    for r, (n, k) in enumerate(zip(lengths, keep)):
        held = torch.zeros(n, dtype=torch.bool, device="cuda")
        held[torch.randperm(n, device="cuda", generator=g)[:k]] = True
        for where, index in zip(moves, (held[k:].nonzero()[:, 0] + k, (~held[:k]).nonzero()[:, 0])):
            where[r, :index.numel()] = table[r, index // page].long() * page + index % page
    cache = lambda: _rows(g, dtype, pages * page, hk, d).view(pages, page, hk, d)
    return {"move_from": moves[0], "move_to": moves[1], "key_cache": cache(), "value_cache": cache(),
            "weights": _skewed(g, pages, page),
            "positions": torch.randint(0, 1 << 20, (pages, page), device="cuda", generator=g).to(torch.int32)}


def _prepare_scan(case, seed):
    g, dtype, channels = _generator(seed), DTYPE[case["type"]], case["channels"]
    lengths = _shuffled(_lengths(case["sequences"], case["low"], case["high"], case["mix"]), seed)
    tokens, count = sum(lengths), case["sequences"]
    # Channels that remember for two tokens to a thousand, each token's gate a little shorter or longer.
    span = torch.exp(-math.log(2000.0) * torch.rand(channels, device="cuda", generator=g))
    s = {"x": _normal(g, tokens, channels).to(dtype), "offsets": _offsets(lengths),
         "log_decay": (-0.5 * span * torch.exp(0.4 * _normal(g, tokens, channels))).to(dtype),
         "initial": _normal(g, count, channels), "final": torch.empty(count, channels, device="cuda"),
         "out": torch.empty(tokens, channels, dtype=dtype, device="cuda")}
    if case["op"] == "scan":
        s |= {"dout": _normal(g, tokens, channels).to(dtype), "dfinal": _normal(g, count, channels),
              "dx": torch.empty_like(s["x"]), "dlog_decay": torch.empty_like(s["x"]),
              "dinitial": torch.empty(count, channels, device="cuda")}
    return s


def prepare(case, seed):
    make = {"write": _prepare_write, "rotate": _prepare_rotate, "weights": _prepare_weights, "evict": _prepare_evict,
            "move": _prepare_move, "state": _prepare_scan, "scan": _prepare_scan}
    state = {"case": dict(case)} | make[case["op"]](case, seed)
    torch.cuda.synchronize()
    return state


# ---- the plain forms -------------------------------------------------------------------------------
def _turned(x, positions, s, sign):
    """Rows [T, H, D] turned by their positions' angles, which 32 bits do not hold at far positions."""
    case, half = s["case"], s["case"]["rotary"] // 2
    angle = positions.double()[:, None] * s["frequencies"]
    c, n = (case["factor"] * angle.cos()).float()[:, None], (sign * case["factor"] * angle.sin()).float()[:, None]
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else \
        (slice(0, half), slice(half, 2 * half))
    y = x.float()
    a, b = y[..., first].clone(), y[..., second].clone()
    y = y.clone()
    y[..., first], y[..., second] = a * c - b * n, a * n + b * c
    return y.to(x.dtype)


def _write(s):
    real = s["requests"] >= 0
    positions = (s["positions"] + s["shifts"][s["requests"].clamp_min(0).long()])[real]
    s["q_out"][real] = _turned(s["q"][real], positions, s, 1.0)
    keep = (s["slots"] >= 0)[real]
    at = s["slots"][real][keep]
    s["key_cache"].flatten(0, 1)[at] = _turned(s["key"][real], positions, s, 1.0)[keep]
    s["value_cache"].flatten(0, 1)[at] = s["value"][real][keep]
    s["slot_positions"].flatten()[at] = positions[keep]
    return {k: s[k] for k in ("q_out", "key_cache", "value_cache", "slot_positions")}


def _rotate(s):
    p = s["positions"]
    return {"q_out": _turned(s["q"], p, s, 1.0), "k_out": _turned(s["key"], p, s, 1.0),
            "dq": _turned(s["dq_out"], p, s, -1.0), "dk": _turned(s["dk_out"], p, s, -1.0)}


def _weights(s):
    case, page, table, rows = s["case"], s["case"]["page"], s["table"].long(), s["q"].shape[0]
    h, hk, d, n, m = case["heads"], case["kv_heads"], case["dim"], s["new_longest"], s["longest"]
    j, i = torch.arange(m, device="cuda"), torch.arange(n, device="cuda")
    held = table[:, j // page].clamp_min(0)
    at = s["q_offsets"][:-1, None].long() + i
    real = at < s["q_offsets"][1:, None]
    at = at.clamp_max(rows - 1)
    q = s["q"][at].float().view(-1, n, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(-1, hk, h // hk * n, d)
    lse = s["lse"].t()[at].view(-1, n, hk, h // hk).permute(0, 2, 3, 1)
    new, kv = s["q_offsets"].diff().long()[:, None, None], s["kv"].long()[:, None, None]
    visible = (j <= i[:, None] + kv - new) & (j < kv) & real[:, :, None]
    total = torch.zeros(table.shape[0], m, device="cuda")
    for head in range(hk):
        k = s["key_cache"][held, j % page, head].float()
        scores = torch.matmul(q[:, head], k.transpose(-1, -2)).mul_(d ** -0.5).view(-1, h // hk, n, m)
        scores.sub_(lse[:, head][..., None]).exp_().masked_fill_(~visible[:, None], 0.0)
        total += scores.sum((1, 2))
    known = j < s["known"][:, None]
    before = s["before"][held, j % page]
    total += torch.where(known, before * case["decay"], 0.0)
    mine = j < s["kv"][:, None]
    s["after"][held[mine], (j % page).expand(held.shape)[mine]] = total[mine]
    return {"after": s["after"]}


def _evict(s):
    case, page, table = s["case"], s["case"]["page"], s["table"].long()
    n, keep = s["kv"].long()[:, None], s["keep"].long()[:, None]
    j = torch.arange(s["longest"], device="cuda")[None, :]
    held = table[:, j[0] // page].clamp_min(0)
    weight, position = s["weights"][held, j % page], s["positions"][held, j % page]
    safe = (position < case["first"]) | (position >= s["shifts"][:, None] + n - case["recent"])
    weight = torch.where(safe, math.inf, weight).masked_fill(j >= n, -math.inf)
    order = weight.argsort(dim=1, descending=True, stable=True)
    rank = torch.empty_like(order).scatter_(1, order, j.expand(order.shape).contiguous())
    keep = torch.minimum(n, keep)
    stays = (rank < keep) & (j < n)
    slot = held * page + j % page
    out = {}
    for name, chosen in (("move_from", stays & (j >= keep)), ("move_to", ~stays & (j < keep))):
        where = torch.full((table.shape[0], s["move_from"].shape[1] + 1), -1, dtype=torch.int64, device="cuda")
        at = torch.where(chosen, chosen.cumsum(1) - 1, s["move_from"].shape[1])
        out[name] = where.scatter_(1, at, slot)[:, :-1].contiguous()
    # Pages that no kept key is in, in the requests' order.
    n, keep = n[:, 0], keep[:, 0]
    column = torch.arange(table.shape[1], device="cuda")[None, :]
    free = (column >= ((keep + page - 1) // page)[:, None]) & (column < ((n + page - 1) // page)[:, None])
    pages = s["table"][free]
    released = torch.full_like(s["released"], -1)
    released[:pages.numel()] = pages
    counts = torch.stack([free.sum(), keep.sum()]).int()
    return out | {"kept": keep.int(), "shifts": (s["shifts"] + n - keep).int(), "released": released, "counts": counts}


def _move(s):
    real = s["move_from"] >= 0
    source, target = s["move_from"][real], s["move_to"][real]
    for name in ("key_cache", "value_cache", "weights", "positions"):
        rows = s[name].flatten(0, 1)
        rows[target] = rows[source]
    return {k: s[k] for k in ("key_cache", "value_cache", "weights", "positions")}


def _scanned(decay, x):
    """y[t] = decay[t] y[t - 1] + x[t] along the first axis, by doubling; both are used up."""
    step = 1
    while step < x.shape[0]:
        x[step:] += decay[step:] * x[:-step].clone()
        decay[step:] *= decay[:-step].clone()
        step *= 2
    return x


def _scan(s):
    # In 64 bits: a channel that remembers thousands of tokens adds up as many roundings.
    dtype, starts, ends = s["x"].dtype, s["offsets"][:-1].long(), s["offsets"][1:].long() - 1
    decay, x = s["log_decay"].double().exp(), s["x"].double()
    cut = decay.clone()
    x[starts] += decay[starts] * s["initial"]
    cut[starts] = 0.0
    h = _scanned(cut, x)
    out = {"out": h.to(dtype), "final": h[ends].float()}
    if s["case"]["op"] == "state":
        return out
    # Backwards in time: g[t] = dout[t] + decay[t + 1] g[t + 1].
    g = s["dout"].double()
    g[ends] += s["dfinal"]
    cut = torch.zeros_like(decay)
    cut[:-1] = decay[1:]
    cut[ends] = 0.0
    g = _scanned(cut.flip(0), g.flip(0)).flip(0)
    before = torch.zeros_like(h)
    before[1:] = h[:-1]
    before[starts] = s["initial"].double()
    return out | {"dx": g.to(dtype), "dlog_decay": (g * decay * before).to(dtype),
                  "dinitial": (g * decay)[starts].float()}


# ---- the library's calls ---------------------------------------------------------------------------
def _library():
    here = os.path.abspath("luisacompute-parallelprimitive_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import lcpp_hip
    return lcpp_hip


def _workspace(s, nbytes):
    """Temporary storage, which a program keeps between its calls."""
    if "temp" not in s:
        s["temp"] = torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda")
    return s["temp"]


def _own(s):
    hip, case = _library(), s["case"]
    op = case["op"]
    if op == "write":
        hip.paged_write_rotary(case["type"], s["q"], s["key"], s["value"], s["positions"], s["frequencies"], s["slots"],
                               s["q_out"], s["key_cache"], s["value_cache"], slot_positions=s["slot_positions"],
                               requests=s["requests"], shifts=s["shifts"], interleaved=case["interleaved"],
                               factor=case["factor"])
        return {k: s[k] for k in ("q_out", "key_cache", "value_cache", "slot_positions")}
    if op == "rotate":
        hip.rotary(case["type"], s["q"], s["key"], s["positions"], s["frequencies"], s["q_out"], s["k_out"],
                   interleaved=case["interleaved"], factor=case["factor"])
        hip.rotary(case["type"], s["dq_out"], s["dk_out"], s["positions"], s["frequencies"], s["dq"], s["dk"],
                   interleaved=case["interleaved"], factor=case["factor"], inverse=True)
        return {k: s[k] for k in ("q_out", "k_out", "dq", "dk")}
    if op == "weights":
        temp = _workspace(s, hip.attention_paged_weights_temp_bytes(case["requests"], s["q"].shape[0], s["longest"],
                                                                    case["heads"], case["kv_heads"], case["dim"]))
        hip.attention_paged_weights(case["type"], s["q"], s["key_cache"], s["table"], s["q_offsets"], s["kv"], s["lse"],
                                    s["after"], weights_in=s["before"], known_lengths=s["known"], decay=case["decay"],
                                    max_kv_length=s["longest"], temp=temp)
        return {"after": s["after"]}
    if op == "evict":
        hip.page_release(s["kv"], s["keep"], case["page"], s["table"], s["kept"], s["released"], s["counts"],
                         shifts=s["shifts"], shifts_out=s["shifts_out"])
        temp = _workspace(s, hip.evict_plan_temp_bytes(case["requests"], s["longest"]))
        hip.evict_plan(s["weights"], s["positions"], s["table"], s["kv"], s["kept"], s["move_from"], s["move_to"],
                       first=case["first"], recent=case["recent"], shifts=s["shifts"], max_kv_length=s["longest"],
                       temp=temp)
        return {k: s[k] for k in ("move_from", "move_to", "kept", "released", "counts")} | {"shifts": s["shifts_out"]}
    if op == "move":
        hip.paged_move(case["type"], s["move_from"], s["move_to"], s["key_cache"], s["value_cache"], weights=s["weights"],
                       positions=s["positions"])
        return {k: s[k] for k in ("key_cache", "value_cache", "weights", "positions")}
    sizes = (case["sequences"], s["x"].shape[0], case["channels"])
    temp = _workspace(s, hip.recurrence_temp_bytes(*sizes))
    hip.recurrence(case["type"], s["x"], s["log_decay"], s["offsets"], s["out"], initial=s["initial"], final=s["final"],
                   temp=temp)
    if op == "state":
        return {k: s[k] for k in ("out", "final")}
    hip.recurrence_backward(case["type"], s["log_decay"], s["out"], s["dout"], s["offsets"], s["dx"], s["dlog_decay"],
                            initial=s["initial"], dfinal=s["dfinal"], dinitial=s["dinitial"], temp=temp)
    return {k: s[k] for k in ("out", "final", "dx", "dlog_decay", "dinitial")}


def run(state):
    if own:
        return _own(state)
    return {"write": _write, "rotate": _rotate, "weights": _weights, "evict": _evict, "move": _move, "state": _scan,
            "scan": _scan}[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    op = case["op"]
    if op in ("write", "rotate"):
        t, d = case["tokens"], case["dim"]
        if op == "write":
            return {"bytes": t * (4 * (case["heads"] + 2 * case["kv_heads"]) * d + 24),
                    "flops": 3 * t * (case["heads"] + case["kv_heads"]) * case["rotary"]}
        return {"bytes": 2 * t * (4 * (case["heads"] + case["kv_heads"]) * d + 4),
                "flops": 6 * t * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    if op == "weights":
        both = _paged_lengths(case)
        rows, keys = sum(n for _, n in both), sum(m for m, _ in both)
        pairs = sum(n * m for m, n in both) - sum(n * (n - 1) // 2 for _, n in both)
        h, d = case["heads"], case["dim"]
        return {"bytes": rows * h * (2 * d + 4) + keys * (2 * case["kv_heads"] * d + 8), "flops": 2 * d * h * pairs}
    if op in ("evict", "move"):
        # A key that stays is past the end with the chance of any key to be: K (n - K) / n moves of n keys to K.
        lengths = _lengths(case["requests"], case["low"], case["high"], case["mix"])
        moves = sum(_kept(case, n) * (n - _kept(case, n)) / n for n in lengths)
        if op == "evict":
            cells = sum(-(-n // case["page"]) for n in lengths)
            return {"bytes": int(8 * sum(lengths) + 4 * cells + 16 * moves), "flops": 0}
        return {"bytes": int(moves * (16 + 16 + 8 * case["kv_heads"] * case["dim"])), "flops": 0}
    tokens = sum(_lengths(case["sequences"], case["low"], case["high"], case["mix"]))
    c, size, states = case["channels"], 4 if case["type"] == "f32" else 2, case["sequences"] * case["channels"]
    if op == "state":
        return {"bytes": 3 * size * tokens * c + 8 * states, "flops": 2 * tokens * c}
    return {"bytes": 8 * size * tokens * c + 20 * states, "flops": 6 * tokens * c}


# ---- in 64 bits ------------------------------------------------------------------------------------
def _exact_turn(x, angle, factor, interleaved):
    """Each pair as a complex number, times the number at the angle."""
    half = angle.shape[1]
    y = x.double().clone()
    spin = torch.polar(torch.full_like(angle, factor), angle)[:, None]
    if interleaved:
        z = torch.view_as_complex(y[..., :2 * half].reshape(*y.shape[:2], half, 2).contiguous()) * spin
        y[..., :2 * half] = torch.view_as_real(z).flatten(2)
    else:
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * spin
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


def _exact_write(case, s):
    real = (s["requests"] >= 0).nonzero()[:, 0]
    positions = s["positions"][real].long() + s["shifts"][s["requests"][real].long()].long()
    angle = positions.double()[:, None] * s["frequencies"]
    q, keys = s["q_out"].double(), s["key_cache"].double()
    q[real] = _exact_turn(s["q"][real], angle, case["factor"], case["interleaved"])
    there = s["slots"][real] >= 0
    slots = s["slots"][real][there]
    turned = _exact_turn(s["key"][real], angle, case["factor"], case["interleaved"])
    keys.view(-1, *keys.shape[2:])[slots] = turned[there]
    return {"q_out": q, "key_cache": keys, "value_cache": None, "slot_positions": None}


def _exact_rotate(case, s):
    angle = s["positions"].double()[:, None] * s["frequencies"]
    turn = lambda x, a: _exact_turn(x, a, case["factor"], case["interleaved"])
    return {"q_out": turn(s["q"], angle), "k_out": turn(s["key"], angle), "dq": turn(s["dq_out"], -angle),
            "dk": turn(s["dk_out"], -angle)}


def _exact_weights(case, s):
    page, group, scale = case["page"], case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["dim"])
    after = s["after"].double()
    at, lengths, known = s["q_offsets"].tolist(), s["kv"].tolist(), s["known"].tolist()
    for r, m in enumerate(lengths):
        n = at[r + 1] - at[r]
        used = s["table"][r, :-(-m // page)].long()
        total = torch.zeros(m, dtype=torch.float64, device="cuda")
        visible = torch.ones(n, m, dtype=torch.bool, device="cuda").tril(m - n)
        for h in range(case["heads"]):
            k = s["key_cache"][used, :, h // group].flatten(0, 1)[:m].double()
            w = torch.exp(s["q"][at[r]:at[r + 1], h].double() @ k.t() * scale - s["lse"][h, at[r]:at[r + 1], None].double())
            total += torch.where(visible, w, 0.0).sum(0)
        total[:known[r]] += case["decay"] * s["before"][used].flatten()[:known[r]].double()
        whole = after[used].flatten()
        whole[:m] = total
        after[used] = whole.view(-1, page)
    return {"after": after}


def _exact_scan(case, s):
    """Token by token, all sequences that have one at a time."""
    at = s["offsets"].tolist()
    lengths = [b - a for a, b in zip(at, at[1:])]
    order = sorted(range(len(lengths)), key=lambda b: -lengths[b])
    starts = _ints([at[b] for b in order], torch.int64)
    counts, left = [], len(order)
    for t in range(max(lengths)):
        while lengths[order[left - 1]] <= t:
            left -= 1
        counts.append(left)
    h, out = s["initial"][order].double(), torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
    decay = s["log_decay"].double().exp_()
    for t, n in enumerate(counts):
        rows = starts[:n] + t
        h[:n] = decay[rows] * h[:n] + s["x"][rows].double()
        out[rows] = h[:n]
    final = torch.empty_like(h)
    final[order] = h
    if case["op"] == "state":
        return {"out": out, "final": final}
    dx, dlog = torch.empty_like(out), torch.empty_like(out)
    c, initial = s["dfinal"][order].double(), s["initial"][order].double()
    for t in range(len(counts) - 1, -1, -1):
        n = counts[t]
        rows = starts[:n] + t
        g = s["dout"][rows].double() + c[:n]
        dx[rows] = g
        c[:n] = decay[rows] * g
        dlog[rows] = c[:n] * (out[rows - 1] if t else initial[:n])
    dinitial = torch.empty_like(c)
    dinitial[order] = c
    return {"out": out, "final": final, "dx": dx, "dlog_decay": dlog, "dinitial": dinitial}


def exact(case, seed):
    if case["op"] in ("evict", "move"):
        return None  # whole numbers and copies: equal, or wrong
    if case["op"] == "weights" and case["requests"] * case["heads"] > 16_384:
        return None
    make = {"write": _exact_write, "rotate": _exact_rotate, "weights": _exact_weights, "state": _exact_scan,
            "scan": _exact_scan}
    return make[case["op"]](case, prepare(case, seed))
