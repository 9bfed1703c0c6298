"""Calls of the attention operators over ragged batches that their performance is measured by.

A batch is held as the library's segmented calls hold one: rows of all sequences one after another, and offsets.  A
request goes through the operators in this order: `plan` lays a step out (offsets, positions, pages taken from a free
list, a slot of the cache for every new token), `write` puts the step's keys and values into their slots, `prompt` is
causal attention over the packed rows (`train` with its backward pass), and `paged` is attention of a few new tokens,
one or a tree of drafted ones, over the pages.

`run` computes them from elementary torch operations in 32 bits, or where `own` is true by the library's calls.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}
# Scores of the plain form that one call may hold (sequences x heads x longest x longest), in values.
MOST_SCORES = 16 * 16384 * 16384


def listed():
    return [
        # One decoding step of a small batch: a scan of 64 lengths and 64 slots.  Latency.
        {"name": "plan_decode_64", "op": "plan", "requests": 64, "cached_low": 17, "cached_high": 4000, "new_low": 1,
         "new_high": 1, "page": 16, "capacity": 64, "mix": 1},
        # A step that mixes decoding with prompts of up to 2,000 tokens, in buffers of a fixed capacity.
        {"name": "plan_mixed_4096", "op": "plan", "requests": 4096, "cached_low": 1, "cached_high": 8000, "new_low": 1,
         "new_high": 2000, "page": 16, "capacity": 1_200_000, "mix": 2},
        # The keys and values of one decoding step.
        {"name": "write_decode_256", "op": "write", "type": "bf16", "tokens": 256, "kv_heads": 8, "dim": 128, "page": 16,
         "spare": 512},
        # The keys and values of a batch of prompts, 128 MiB each.
        {"name": "write_prompt_65k", "op": "write", "type": "f16", "tokens": 65_521, "kv_heads": 8, "dim": 128,
         "page": 64, "spare": 64},
        # A handful of short prompts, 1 to 200 tokens, on a small model.  Latency.
        {"name": "prompt_short_d64", "op": "prompt", "type": "bf16", "sequences": 7, "low": 1, "high": 200, "prefix": 0,
         "heads": 8, "kv_heads": 2, "dim": 64, "mix": 3},
        # A batch of prompts of ordinary and uneven lengths, packed.
        {"name": "prompt_ragged_f16", "op": "prompt", "type": "f16", "sequences": 16, "low": 60, "high": 2500,
         "prefix": 0, "heads": 32, "kv_heads": 8, "dim": 128, "mix": 4},
        # One long document.
        {"name": "prompt_16k", "op": "prompt", "type": "bf16", "sequences": 1, "low": 16384, "high": 16384, "prefix": 0,
         "heads": 16, "kv_heads": 4, "dim": 128, "mix": 5},
        # Fine-tuning on short examples, with a head size and lengths that no tile divides.
        {"name": "train_short_d80", "op": "train", "type": "f16", "sequences": 5, "low": 100, "high": 517, "prefix": 0,
         "heads": 12, "kv_heads": 12, "dim": 80, "mix": 6},
        # A training step over rows of about 8,000 tokens with documents packed in them.
        {"name": "train_packed_bf16", "op": "train", "type": "bf16", "sequences": 6, "low": 700, "high": 4096,
         "prefix": 0, "heads": 32, "kv_heads": 8, "dim": 128, "mix": 7},
        # Decoding of a large batch, contexts from 200 to 4,000 tokens.
        {"name": "paged_decode_256", "op": "paged", "type": "bf16", "requests": 256, "low": 200, "high": 4000,
         "new_low": 1, "new_high": 1, "tree": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "mix": 8},
        # Decoding of one request with a very long context.
        {"name": "paged_decode_131k", "op": "paged", "type": "f16", "requests": 1, "low": 131_000, "high": 131_000,
         "new_low": 1, "new_high": 1, "tree": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "mix": 9},
        # Trees of 5 to 48 drafted tokens over contexts of up to 8,000.
        {"name": "paged_tree_24", "op": "paged", "type": "bf16", "requests": 24, "low": 500, "high": 8000, "new_low": 5,
         "new_high": 48, "tree": True, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "mix": 10},
    ]


def _size(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["plan", "write", "prompt", "prompt", "train", "train", "paged", "paged", "paged"])
    mix = rng.randrange(1 << 20)
    if op == "plan":
        requests = _size(rng, 1, 8192)
        new_high = rng.choice([1, 1, 8, 64, 2000])
        cached = _size(rng, 1, 16000)
        low = 1 if rng.random() < 0.8 else 0
        case = {"op": op, "requests": requests, "cached_low": rng.choice([0, 1]), "cached_high": cached, "new_low": low,
                "new_high": new_high, "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 128, 256]), "mix": mix}
        if case["page"] < 8:
            case["cached_high"] = min(cached, 1000)
        total = sum(_lengths(requests, low, new_high, mix + 1))
        case["capacity"] = total + rng.choice([0, 0, 1, 37, 1000])
        return case
    dim = rng.choice([64, 128, 128, 128, 32, 80, 96, 112, 120])
    group = rng.choice([1, 1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    heads = group * kv_heads
    kind = rng.choice(["bf16", "bf16", "f16"])
    if op == "write":
        return {"op": op, "type": kind, "tokens": _size(rng, 1, 65_521), "kv_heads": kv_heads, "dim": dim,
                "page": rng.choice([1, 8, 16, 16, 24, 32, 64, 128, 256]), "spare": _size(rng, 1, 256)}
    if op == "paged":
        tree = rng.random() < 0.5
        new_high = _size(rng, 2, 64) if tree else rng.choice([1, 1, 1, 4, 100])
        new_low = rng.choice([1, new_high])
        high = _size(rng, max(16, new_high), 131_000)
        # At most a quarter of a GiB of keys, as many values, and as many scores as the plain form may hold.
        most = min((1 << 27) // (high * kv_heads * dim), MOST_SCORES // (8 * high * heads * new_high))
        requests = _size(rng, 1, max(1, min(512, most)))
        return {"op": op, "type": kind, "requests": requests, "low": max(new_high, high // rng.choice([1, 3, 20])),
                "high": high, "new_low": new_low, "new_high": new_high, "tree": tree, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "page": rng.choice([8, 16, 16, 24, 32, 64, 128, 256]), "mix": mix}
    high = _size(rng, 1 if op == "prompt" else 24, 8192)
    # As many sequences as the plain form's scores, and the largest listed case's products, allow.
    share = 2 if op == "prompt" else 6
    most = MOST_SCORES // (share * heads * (high + 500) * (high + 500))
    while most < 1 and heads > kv_heads:
        heads = kv_heads
        most = MOST_SCORES // (share * heads * (high + 500) * (high + 500))
    high = high if most else 2048
    sequences = _size(rng, 1, max(1, min(64, most, 32_768 // high)))
    return {"op": op, "type": kind, "sequences": sequences, "low": max(1, high // rng.choice([1, 2, 8, 40])),
            "high": high, "prefix": rng.choice([0, 0, 0, rng.randrange(1, 500), -rng.randrange(1, 9) if high > 16 else 0]),
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "mix": mix}


# ---- inputs ----------------------------------------------------------------------------------------
def _lengths(count, low, high, mix):
    """Lengths spread over their logarithm, the longest of them `high`.  The case alone decides them."""
    rng = random.Random(mix)
    if low < 1:  # some of them none
        return [high] + [_size(rng, 1, high) if rng.random() < 0.8 else 0 for _ in range(count - 1)]
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


def _rows(g, dtype, rows, heads, dim, gain=1.0, outliers=False):
    """Normal rows; `outliers`: one channel in 32 of four times the width, as learned keys have them."""
    x = torch.randn(rows, heads, dim, device="cuda", generator=g)
    if outliers:
        x[..., 5::32] *= 4.0
    return (x * gain).to(dtype)


def _cells(lengths, page):
    return [-(-n // page) for n in lengths]


def _prepare_plan(case, seed):
    count, page = case["requests"], case["page"]
    cached = _lengths(count, case["cached_low"], case["cached_high"], case["mix"])
    new = _lengths(count, case["new_low"], case["new_high"], case["mix"] + 1)
    cached, new = _shuffled(cached, seed), _shuffled(new, seed + 1)
    held, used = _cells(cached, page), _cells([c + n for c, n in zip(cached, new)], page)
    width = -(-(case["cached_high"] + case["new_high"]) // page)
    needed = sum(used) - sum(held)
    pages = torch.randperm(sum(used) + 64, device="cuda", generator=_generator(seed)).to(torch.int32)
    table = torch.full((count, width), -1, dtype=torch.int32, device="cuda")
    column = torch.arange(width, device="cuda")[None, :]
    have = _ints(held, torch.int64)[:, None]
    first = have.cumsum(0) - have
    old = column < have
    table[old] = pages[(first + column)[old]]
    # A free list a little longer than the step needs.
    free = pages[sum(held):sum(held) + needed + 32].contiguous()
    t = case["capacity"]
    empty = lambda n, dtype=torch.int32: torch.empty(n, dtype=dtype, device="cuda")
    return {"cached": _ints(cached), "new": _ints(new), "free": free, "table": table, "offsets": empty(count + 1),
            "kv": empty(count), "request": empty(t), "position": empty(t), "slot": empty(t, torch.int64),
            "counts": empty(2)}


def _prepare_write(case, seed):
    g, dtype, tokens, page = _generator(seed), DTYPE[case["type"]], case["tokens"], case["page"]
    pages = -(-tokens // page) + case["spare"]
    # Slots of the step's tokens: runs inside pages in any order; one token in 50 has none.
    order = torch.randperm(pages, device="cuda", generator=g)
    t = torch.arange(tokens, device="cuda")
    slots = order[t // page] * page + t % page
    slots[torch.rand(tokens, device="cuda", generator=g) < 0.02] = -1
    cache = lambda: torch.zeros(pages, page, case["kv_heads"], case["dim"], dtype=dtype, device="cuda")
    return {"key": _rows(g, dtype, tokens, case["kv_heads"], case["dim"], outliers=True),
            "value": _rows(g, dtype, tokens, case["kv_heads"], case["dim"]), "slots": slots, "key_cache": cache(),
            "value_cache": cache()}


def _prepare_packed(case, seed):
    g, dtype = _generator(seed), DTYPE[case["type"]]
    lengths = _shuffled(_lengths(case["sequences"], case["low"], case["high"], case["mix"]), seed)
    keys = [max(0, n + case["prefix"]) for n in lengths]
    tq, tk, h, hk, d = sum(lengths), sum(keys), case["heads"], case["kv_heads"], case["dim"]
    s = {"q": _rows(g, dtype, tq, h, d, 1.5), "k": _rows(g, dtype, tk, hk, d, outliers=True),
         "v": _rows(g, dtype, tk, hk, d), "q_offsets": _offsets(lengths), "k_offsets": _offsets(keys),
         "q_longest": max(lengths), "k_longest": max(1, max(keys)), "out": torch.empty(tq, h, d, dtype=dtype, device="cuda"),
         "lse": torch.empty(h, tq, device="cuda")}
    if case["op"] == "train":
        s["dout"] = _rows(g, dtype, tq, h, d)
        s |= {"dq": torch.empty_like(s["q"]), "dk": torch.empty_like(s["k"]), "dv": torch.empty_like(s["v"])}
    return s


def _paged_lengths(case):
    kv = _lengths(case["requests"], case["low"], case["high"], case["mix"])
    new = _lengths(case["requests"], case["new_low"], case["new_high"], case["mix"] + 1)
    return list(zip(kv, new))


def _prepare_paged(case, seed):
    g, dtype, page = _generator(seed), DTYPE[case["type"]], case["page"]
    both = _shuffled(_paged_lengths(case), seed)
    kv, new = [a for a, _ in both], [b for _, b in both]
    h, hk, d, count = case["heads"], case["kv_heads"], case["dim"], case["requests"]
    used = _cells(kv, page)
    width, pages = max(used), sum(used) + 7
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((count, width), -1, dtype=torch.int32, device="cuda")
    column = torch.arange(width, device="cuda")[None, :]
    have = _ints(used, torch.int64)[:, None]
    filled = column < have
    table[filled] = order[(have.cumsum(0) - have + column)[filled]]
    t = sum(new)
    s = {"q": _rows(g, dtype, t, h, d, 1.5), "table": table, "q_offsets": _offsets(new), "kv": _ints(kv),
         "key_cache": _rows(g, dtype, pages * page, hk, d, outliers=True).view(pages, page, hk, d),
         "value_cache": _rows(g, dtype, pages * page, hk, d).view(pages, page, hk, d), "longest": max(kv),
         "new_longest": max(new), "out": torch.empty(t, h, d, dtype=dtype, device="cuda"),
         "lse": torch.empty(h, t, device="cuda"), "tree": None}
    if case["tree"]:
        # Every drafted token hangs below an earlier one of its request, or below the context.
        rng, words = random.Random(seed + 2), []
        for n in new:
            mask = []
            for i in range(n):
                parent = rng.randrange(-1, i)
                mask.append((mask[parent] if parent >= 0 else 0) | 1 << i)
            words += mask
        s["tree"] = _ints([w - (1 << 64) if w >> 63 else w for w in words], torch.int64)
    return s


def prepare(case, seed):
    make = {"plan": _prepare_plan, "write": _prepare_write, "prompt": _prepare_packed, "train": _prepare_packed,
            "paged": _prepare_paged}
    state = {"case": dict(case)} | make[case["op"]](case, seed)
    torch.cuda.synchronize()
    return state


# ---- the plain forms -------------------------------------------------------------------------------
def _plan(s):
    page, table, free = s["case"]["page"], s["table"], s["free"]
    cached, new = s["cached"].long().clamp_min(0), s["new"].long().clamp_min(0)
    count, width = table.shape
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), new.cumsum(0)])
    kv = cached + new
    have = ((cached + page - 1) // page).clamp_max(width)
    need = ((kv + page - 1) // page).clamp_max(width) - have
    ends = need.cumsum(0)
    column = torch.arange(width, device="cuda")[None, :]
    index = column - have[:, None] + (ends - need)[:, None]
    fresh = (column >= have[:, None]) & (column < (have + need)[:, None])
    taken = torch.where(index < free.numel(), free[index.clamp(0, free.numel() - 1)], -1)
    table = torch.where(fresh, taken, table)
    t = torch.arange(s["slot"].numel(), device="cuda")
    request = torch.searchsorted(offsets[1:], t, right=True)
    real = request < count
    r = request.clamp_max(count - 1)
    position = cached[r] + t - offsets[r]
    cell = position // page
    held = table[r, cell.clamp(0, width - 1)].long()
    slot = torch.where(real & (cell < width) & (held >= 0), held * page + position % page, -1)
    return {"table": table, "offsets": offsets.int(), "kv": kv.int(), "request": torch.where(real, request, -1).int(),
            "position": torch.where(real, position, 0).int(), "slot": slot,
            "counts": torch.stack([offsets[-1], ends[-1]]).int()}


def _write(s):
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    s["key_cache"].flatten(0, 1)[at] = s["key"][keep]
    s["value_cache"].flatten(0, 1)[at] = s["value"][keep]
    return {"key_cache": s["key_cache"], "value_cache": s["value_cache"]}


def _padded(x, offsets, longest, kv_heads):
    """Rows [T, H, D] as [B, kv_heads, longest * H / kv_heads, D] in 32 bits, zero past each sequence's end."""
    at = offsets[:-1, None].long() + torch.arange(longest, device="cuda")
    real = at < offsets[1:, None]
    if x.shape[0] == 0:
        return torch.zeros(at.shape[0], kv_heads, longest * x.shape[1] // kv_heads, x.shape[2], device="cuda")
    rows = x[at.clamp_max(x.shape[0] - 1)].float() * real[:, :, None, None]
    b, n, h, d = rows.shape
    return rows.view(b, n, kv_heads, h // kv_heads, d).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, d)


def _packed_again(y, offsets, rows, heads):
    """The inverse: [B, kv_heads, group * longest, D] as [T, H, D]."""
    t = torch.arange(rows, device="cuda")
    b = torch.searchsorted(offsets[1:].long(), t, right=True)
    batch, kv_heads, _, d = y.shape
    y = y.view(batch, kv_heads, heads // kv_heads, -1, d)
    return y[b, :, :, t - offsets[b]].reshape(rows, heads, d)


def _softmax(scores, visible):
    """Weights and log-sums of masked scores, in place; rows that see nothing have weights of zero."""
    scores.masked_fill_(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    scores.div_(total.masked_fill(total == 0.0, 1.0))
    return scores, top + total.log()


def _scores(s):
    """Padded operands, softmax weights [B, kv_heads, group * longest, keys] and log-sums of a packed batch."""
    case = s["case"]
    hk, n, m = case["kv_heads"], s["q_longest"], s["k_longest"]
    q = _padded(s["q"], s["q_offsets"], n, hk)
    k, v = _padded(s["k"], s["k_offsets"], m, hk), _padded(s["v"], s["k_offsets"], m, hk)
    i, j = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
    nq, nk = s["q_offsets"].diff()[:, None, None], s["k_offsets"].diff()[:, None, None]
    visible = (j < nk) & (j <= i[:, None] + nk - nq) & (i[:, None] < nq)
    batch, group = q.shape[0], case["heads"] // hk
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(case["dim"] ** -0.5)
    scores, lse = _softmax(scores.view(batch, hk, group, n, m), visible[:, None, None])
    return q, k, v, scores.view(batch, hk, group * n, m), lse.reshape(batch, hk, group * n, 1)


def _prompt(s):
    case, rows = s["case"], s["q"].shape[0]
    _, _, v, weights, lse = _scores(s)
    out = _packed_again(torch.matmul(weights, v), s["q_offsets"], rows, case["heads"])
    lse = _packed_again(lse, s["q_offsets"], rows, case["heads"])
    return {"out": out.to(s["q"].dtype), "lse": lse[:, :, 0].t().contiguous()}


def _train(s):
    case, dtype = s["case"], s["q"].dtype
    q, k, v, weights, _ = _scores(s)
    dout = _padded(s["dout"], s["q_offsets"], s["q_longest"], case["kv_heads"])
    out = torch.matmul(weights, v)
    dv = torch.matmul(weights.transpose(-1, -2), dout)
    inner = torch.matmul(dout, v.transpose(-1, -2))
    inner.sub_((dout * out).sum(-1, keepdim=True)).mul_(weights).mul_(case["dim"] ** -0.5)
    dq, dk = torch.matmul(inner, k), torch.matmul(inner.transpose(-1, -2), q)
    back = lambda y, offsets, like, heads: _packed_again(y, offsets, like.shape[0], heads).to(dtype)
    return {"out": back(out, s["q_offsets"], s["q"], case["heads"]), "dq": back(dq, s["q_offsets"], s["q"], case["heads"]),
            "dk": back(dk, s["k_offsets"], s["k"], case["kv_heads"]),
            "dv": back(dv, s["k_offsets"], s["v"], case["kv_heads"])}


def _paged(s):
    case, page, table, rows = s["case"], s["case"]["page"], s["table"].long(), s["q"].shape[0]
    h, hk, d, n, m = case["heads"], case["kv_heads"], case["dim"], s["new_longest"], s["longest"]
    j = torch.arange(m, device="cuda")
    held = table[:, j // page].clamp_min(0)
    k = s["key_cache"][held, j % page].float().transpose(1, 2)
    v = s["value_cache"][held, j % page].float().transpose(1, 2)
    q = _padded(s["q"], s["q_offsets"], n, hk)
    i = torch.arange(n, device="cuda")
    new, kv = s["q_offsets"].diff().long()[:, None, None], s["kv"].long()[:, None, None]
    drafted = j - (kv - new)
    if s["tree"] is None:
        seen = drafted <= i[:, None]
    else:
        words = s["tree"][(s["q_offsets"][:-1, None].long() + i).clamp_max(rows - 1)][:, :, None]
        seen = (drafted < 0) | (((words >> drafted.clamp(0, 63)) & 1) == 1)
    visible = seen & (j < kv) & (i[:, None] < new)
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5)
    weights, lse = _softmax(scores.view(-1, hk, h // hk, n, m), visible[:, None, None])
    out = torch.matmul(weights.view(-1, hk, h // hk * n, m), v)
    lse = _packed_again(lse.reshape(-1, hk, h // hk * n, 1), s["q_offsets"], rows, h)
    return {"out": _packed_again(out, s["q_offsets"], rows, h).to(s["q"].dtype), "lse": lse[:, :, 0].t().contiguous()}


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
    if op == "plan":
        temp = _workspace(s, hip.page_plan_temp_bytes(case["requests"]))
        hip.page_plan(s["cached"], s["new"], case["page"], s["free"], s["table"], s["offsets"], s["kv"], s["request"],
                      s["position"], s["slot"], s["counts"], temp=temp)
        return {k: s[k] for k in ("table", "offsets", "kv", "request", "position", "slot", "counts")}
    if op == "write":
        hip.paged_write(case["type"], s["key"], s["value"], s["slots"], s["key_cache"], s["value_cache"])
        return {"key_cache": s["key_cache"], "value_cache": s["value_cache"]}
    shape = (case["heads"], case["kv_heads"], case["dim"])
    if op == "paged":
        temp = _workspace(s, hip.attention_paged_temp_bytes(case["requests"], s["q"].shape[0], s["longest"], *shape))
        hip.attention_paged(case["type"], s["q"], s["key_cache"], s["value_cache"], s["table"], s["q_offsets"], s["kv"],
                            s["out"], s["lse"], tree=s["tree"], max_kv_length=s["longest"], temp=temp)
        return {"out": s["out"], "lse": s["lse"]}
    sizes = (case["sequences"], s["q"].shape[0], s["k"].shape[0])
    if op == "prompt":
        temp = _workspace(s, hip.attention_packed_temp_bytes(*sizes, *shape))
        hip.attention_packed(case["type"], s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], s["out"], s["lse"],
                             causal=True, temp=temp)
        return {"out": s["out"], "lse": s["lse"]}
    temp = _workspace(s, max(hip.attention_packed_temp_bytes(*sizes, *shape),
                             hip.attention_packed_backward_temp_bytes(*sizes, *shape)))
    hip.attention_packed(case["type"], s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], s["out"], s["lse"],
                         causal=True, temp=temp)
    hip.attention_packed_backward(case["type"], s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"], s["q_offsets"],
                                  s["k_offsets"], s["dq"], s["dk"], s["dv"], causal=True, temp=temp)
    return {k: s[k] for k in ("out", "dq", "dk", "dv")}


def run(state):
    if own:
        return _own(state)
    return {"plan": _plan, "write": _write, "prompt": _prompt, "train": _train, "paged": _paged}[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "plan":
        count, page = case["requests"], case["page"]
        new = _lengths(count, case["new_low"], case["new_high"], case["mix"] + 1)
        # At the least one new page for every page's worth of new tokens, and the last held page of every request.
        pages = sum(new) // page
        return {"bytes": 20 * count + 8 * pages + 16 * case["capacity"], "flops": 0}
    if op == "write":
        return {"bytes": 8 * case["tokens"] * (1 + case["kv_heads"] * case["dim"]), "flops": 0}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "paged":
        both = _paged_lengths(case)
        rows, keys = sum(n for _, n in both), sum(m for m, _ in both)
        pairs = sum(n * m for m, n in both) - sum(n * (n - 1) // 2 for _, n in both)
        return {"bytes": 4 * rows * h * d + 4 * keys * hk * d + 4 * rows * h, "flops": 4 * d * h * pairs}
    lengths = _lengths(case["sequences"], case["low"], case["high"], case["mix"])
    pairs, rows, keys = 0, sum(lengths), 0
    for n in lengths:
        m = max(0, n + case["prefix"])
        low, high = max(0, m - n + 1), m  # keys that the first and the last row see
        pairs += (low + high) * (high - low + 1) // 2
        keys += m
    if op == "prompt":
        return {"bytes": 4 * rows * h * d + 4 * keys * hk * d + 4 * rows * h, "flops": 4 * d * h * pairs}
    return {"bytes": 8 * rows * h * d + 8 * keys * hk * d, "flops": 14 * d * h * pairs}


# ---- in 64 bits, one sequence and one head at a time -----------------------------------------------
def _exact_head(q, k, v, visible, scale):
    logits = torch.where(visible, q @ k.t() * scale, -math.inf)
    lse = torch.logsumexp(logits, 1)
    weights = torch.where(visible, torch.exp(logits - torch.where(lse == -math.inf, 0.0, lse)[:, None]), 0.0)
    return weights @ v, lse, weights


def _exact_packed(case, s):
    scale, group = 1.0 / math.sqrt(case["dim"]), case["heads"] // case["kv_heads"]
    zero = lambda x: torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    out, dq, dk, dv = zero(s["q"]), zero(s["q"]), zero(s["k"]), zero(s["v"])
    lse = torch.full((case["heads"], s["q"].shape[0]), -math.inf, dtype=torch.float64, device="cuda")
    q_at, k_at = s["q_offsets"].tolist(), s["k_offsets"].tolist()
    for b in range(case["sequences"]):
        rows, keys = slice(q_at[b], q_at[b + 1]), slice(k_at[b], k_at[b + 1])
        n, m = q_at[b + 1] - q_at[b], k_at[b + 1] - k_at[b]
        if n == 0 or m == 0:
            continue
        visible = torch.ones(n, m, dtype=torch.bool, device="cuda").tril(m - n)
        for h in range(case["heads"]):
            q, k, v = s["q"][rows, h].double(), s["k"][keys, h // group].double(), s["v"][keys, h // group].double()
            out[rows, h], lse[h, rows], weights = _exact_head(q, k, v, visible, scale)
            if case["op"] == "train":
                dout = s["dout"][rows, h].double()
                dv[keys, h // group] += weights.t() @ dout
                change = dout @ v.t()
                change = weights * (change - (weights * change).sum(1, keepdim=True))
                dq[rows, h] = scale * (change @ k)
                dk[keys, h // group] += scale * (change.t() @ q)
    return {"out": out, "lse": lse} if case["op"] == "prompt" else {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _exact_paged(case, s):
    scale, group, page = 1.0 / math.sqrt(case["dim"]), case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full((case["heads"], s["q"].shape[0]), -math.inf, dtype=torch.float64, device="cuda")
    at, lengths = s["q_offsets"].tolist(), s["kv"].tolist()
    words = None if s["tree"] is None else [w % (1 << 64) for w in s["tree"].tolist()]
    for r in range(case["requests"]):
        n, m = at[r + 1] - at[r], lengths[r]
        if n == 0 or m == 0:
            continue
        used = s["table"][r, :-(-m // page)].long()
        k = s["key_cache"][used].flatten(0, 1)[:m].double()
        v = s["value_cache"][used].flatten(0, 1)[:m].double()
        if words is None:
            visible = torch.ones(n, m, dtype=torch.bool, device="cuda").tril(m - n)
        else:
            drafted = [[bool(words[at[r] + i] >> b & 1) for b in range(n)] for i in range(n)]
            visible = torch.cat([torch.ones(n, m - n, dtype=torch.bool), torch.tensor(drafted).view(n, n)], 1).cuda()
        rows = slice(at[r], at[r + 1])
        for h in range(case["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            q = s["q"][rows, heads].double().transpose(0, 1).reshape(group * n, -1)
            o, l, _ = _exact_head(q, k[:, h], v[:, h], visible.repeat(group, 1), scale)
            out[rows, heads] = o.view(group, n, -1).transpose(0, 1)
            lse[heads, rows] = l.view(group, n)
    return {"out": out, "lse": lse}


def exact(case, seed):
    if case["op"] in ("plan", "write"):
        return None  # whole numbers and copies: equal, or wrong
    if case["op"] == "paged" and case["requests"] * case["kv_heads"] > 4096:
        return None
    s = prepare(case, seed)
    return _exact_paged(case, s) if case["op"] == "paged" else _exact_packed(case, s)
