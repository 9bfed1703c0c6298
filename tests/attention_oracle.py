"""Plain 64-bit attention over ragged batches (one sequence and one head at a time, on the CPU) with bounds on what 16-bit
kernels with 32-bit sums may be off, and a plain step planner.  Test infrastructure only.

Bounds, element by element, with u the unit roundoff of the 16-bit type (2^-8 for bf16, 2^-11 for f16) and e32 = 2^-23:
the softmax weights are rounded to 16 bits before the product with the values (u), carry the error of a 32-bit
score (dim + 8 roundings of the sum of |q| |k|, as an exponent) and of the exponential and the sum (2^-18, generously),
and the result is rounded once more (u).  Gradients: the same for P and, through dP and delta, for dS, which is rounded
to 16 bits too; delta is taken from the rounded output.  What f16 cannot hold as a normal number is off by up to 2^-25.
"""
import math

import torch

ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -120, torch.float16: 2.0 ** -24}
E32 = 2.0 ** -23


def offsets_of(lengths):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32)


def head(q, k, v, visible, scale, dtype):
    """One head in 64 bits: output, lse, weights, and the bounds of output and weights (relative)."""
    u, dim = ROUNDOFF[dtype], q.shape[1]
    logits = torch.where(visible, q @ k.t() * scale, -math.inf)
    lse = torch.logsumexp(logits, 1) if k.shape[0] else torch.full((q.shape[0],), -math.inf, dtype=torch.float64)
    some = lse > -math.inf
    weights = torch.where(visible, torch.exp(logits - torch.where(some, lse, 0.0)[:, None]), 0.0)
    size = q.abs() @ k.abs().t() * scale
    score_error = torch.where(visible, size, 0.0).amax(1) if k.shape[0] else torch.zeros(q.shape[0], dtype=torch.float64)
    score_error = (dim + 8) * E32 * (score_error + 1.0)  # of a logit, and so of the lse
    relative = 2.0 * score_error + 2.0 ** -18
    out = weights @ v
    bound = u * out.abs() + (u + relative)[:, None] * (weights @ v.abs()) + TINY[dtype] * (1.0 + v.abs().sum(0))
    return out, lse, weights, bound, relative, score_error


def packed(q, k, v, q_offsets, k_offsets, causal, scale, dout=None):
    """Everything of a packed batch, as a dict of (value, bound) pairs."""
    dtype = q.dtype
    u, tiny = ROUNDOFF[dtype], TINY[dtype]
    q, k, v = (x.cpu().double() for x in (q, k, v))
    dout = None if dout is None else dout.cpu().double()
    heads, kv_heads, dim = q.shape[1], k.shape[1], q.shape[2]
    zero = lambda x: (torch.zeros_like(x), torch.zeros_like(x))
    out, dq, dk, dv = zero(q), zero(q), zero(k), zero(v)
    lse = (torch.full((heads, q.shape[0]), -math.inf, dtype=torch.float64), torch.zeros(heads, q.shape[0], dtype=torch.float64))
    at, key_at = q_offsets.tolist(), k_offsets.tolist()
    for b in range(len(at) - 1):
        r, c = slice(at[b], at[b + 1]), slice(key_at[b], key_at[b + 1])
        n, m = at[b + 1] - at[b], key_at[b + 1] - key_at[b]
        if n == 0:
            continue
        visible = torch.ones(n, m, dtype=torch.bool)
        if causal:
            visible = visible.tril(m - n)
        for h in range(heads):
            g = h // (heads // kv_heads)
            qh, kh, vh = q[r, h], k[c, g], v[c, g]
            o, l, p, bound, relative, score_error = head(qh, kh, vh, visible, scale, dtype)
            out[0][r, h], out[1][r, h] = o, bound
            lse[0][h, r] = l
            lse[1][h, r] = 2 * score_error + 8 * E32 * l.abs().nan_to_num(posinf=0.0) + 2.0 ** -18
            if dout is None:
                continue
            do = dout[r, h]
            dp = do @ vh.t()
            delta = (p * dp).sum(1, keepdim=True)
            ds = p * (dp - delta)
            dp_error = (dim + 8) * E32 * (do.abs() @ vh.abs().t())
            delta_error = (do.abs() * (bound + (dim + 8) * E32 * o.abs())).sum(1, keepdim=True)
            p_error = p * relative[:, None]
            ds_error = u * ds.abs() + p * (dp_error + delta_error) + p_error * (dp - delta).abs() + tiny
            ds_error = torch.where(visible, ds_error, 0.0)
            dq[0][r, h] = scale * (ds @ kh)
            dq[1][r, h] = scale * (ds_error @ kh.abs()) * (1 + 2 * u)
            dk[0][c, g] += scale * (ds.t() @ qh)
            dk[1][c, g] += scale * (ds_error.t() @ qh.abs()) * (1 + 2 * u)
            dv[0][c, g] += p.t() @ do
            dv[1][c, g] += ((u * p + p_error + torch.where(visible, tiny, 0.0)).t() @ do.abs()) * (1 + 2 * u)
    for x in (dq, dk, dv):
        x[1].add_(u * x[0].abs() + tiny)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def paged(q, key_cache, value_cache, block_table, q_offsets, kv_lengths, tree, scale):
    dtype = q.dtype
    heads, kv_heads, page, pages = q.shape[1], key_cache.shape[2], key_cache.shape[1], key_cache.shape[0]
    q = q.cpu().double()
    kc, vc = key_cache.cpu().double(), value_cache.cpu().double()
    out = (torch.zeros_like(q), torch.zeros_like(q))
    lse = (torch.full((heads, q.shape[0]), -math.inf, dtype=torch.float64), torch.zeros(heads, q.shape[0], dtype=torch.float64))
    at = q_offsets.tolist()
    for r, length in enumerate(kv_lengths.tolist()):
        rows, n = slice(at[r], at[r + 1]), at[r + 1] - at[r]
        length = min(length, block_table.shape[1] * page)
        if n == 0:
            continue
        position = torch.arange(length)
        held = block_table[r].cpu().long()[position // page]
        there = (held >= 0) & (held < pages)
        held = torch.where(there, held, 0)
        k = torch.where(there[:, None, None], kc[held, position % page], 0.0)
        v = torch.where(there[:, None, None], vc[held, position % page], 0.0)
        visible = torch.zeros(n, length, dtype=torch.bool)
        for i in range(n):
            for j in range(length):
                ahead = j - (length - n)
                if ahead < 0:
                    visible[i, j] = True
                elif tree is None:
                    visible[i, j] = ahead <= i
                else:
                    visible[i, j] = ahead < 64 and bool(int(tree[at[r] + i]) >> ahead & 1)
        visible &= there
        for h in range(heads):
            g = h // (heads // kv_heads)
            clean = lambda x: torch.where(visible.any(0)[:, None], x, 0.0) if length else x
            o, l, _, bound, _, score_error = head(q[rows, h], clean(k[:, g]), clean(v[:, g]), visible, scale, dtype)
            out[0][rows, h], out[1][rows, h] = o, bound
            lse[0][h, rows] = l
            lse[1][h, rows] = 2 * score_error + 8 * E32 * l.abs().nan_to_num(posinf=0.0) + 2.0 ** -18
    return {"out": out, "lse": lse}


def plan(cached, new, page, free, table, capacity):
    """The step planner as a loop; returns what page_plan writes."""
    width = len(table[0]) if table else 0
    table = [list(row) for row in table]
    offsets, kv, tokens, taken = [0], [], [], 0
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        have, need = min(width, -(-c // page)), min(width, -(-(c + n) // page))
        for cell in range(have, need):
            entry = free[taken] if taken < len(free) else -1
            taken += 1
            if len(tokens) + cell * page - c < capacity:
                table[r][cell] = entry
        for position in range(c, c + n):
            cell = position // page
            if len(tokens) < capacity:
                entry = table[r][cell] if cell < width else -1
                tokens.append((r, position, entry * page + position % page if entry >= 0 else -1))
            else:
                tokens.append(None)
        offsets.append(offsets[-1] + n)
        kv.append(c + n)
    total = len(tokens)
    tokens = (tokens + [(-1, 0, -1)] * max(0, capacity - total))[:capacity]
    return {"table": table, "offsets": offsets, "kv": kv, "request": [t[0] for t in tokens],
            "position": [t[1] for t in tokens], "slot": [t[2] for t in tokens], "counts": [total, taken]}


def check(name, got, pair):
    """Element by element within the bound; infinities and NaN in the same places."""
    value, bound = pair
    got = got.detach().cpu().double()
    finite = torch.isfinite(value)
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{name}: NaN elsewhere"
    assert torch.equal(got[~finite].nan_to_num(), value[~finite].nan_to_num()), f"{name}: infinities elsewhere"
    off = (got - value).abs()[finite]
    allowed = bound[finite]
    bad = off > allowed
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / allowed.clamp_min(1e-300)).max()):.2f} of the bound"
