"""Plain 64-bit forms, on the CPU, of the operators that keep a long request's memory bounded (rotary positions, sums of
attention weights, eviction, a gated recurrence), with bounds on what 32-bit kernels may be off.  Test infrastructure only.

u is the unit roundoff of the stored type (2^-8 for bf16, 2^-11 for f16, 2^-24 for f32).
"""
import math

import torch

ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -120, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -126}


# ---- rotary positions ----------------------------------------------------------------------------
def turn(x, positions, frequencies, interleaved, factor=1.0, inverse=False):
    """(value, bound) of rows [T, H, D].  The angle's turns are taken in 64 bits (three roundings, relative 2^-53 each, of
    up to |turns| whole ones), what is left of them in 32 (2^-25 of a half turn); sine and cosine are good to two units of
    2^-24, times the factor, times the item, and the sum: together at most 2^-20 of the pair's absolute sum."""
    half = frequencies.numel()
    x64, angle = x.cpu().double(), positions.cpu().double()[:, None] * frequencies.cpu()[None, :]
    c, s = (factor * angle.cos())[:, None], (factor * (-angle if inverse else angle).sin())[:, None]
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y, bound = x64.clone(), torch.zeros_like(x64)
    a, b = x64[..., first], x64[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    size = abs(factor) * (a.abs() + b.abs()) * (2.0 ** -20 + 2.0 ** -50 * angle.abs()[:, None])
    bound[..., first], bound[..., second] = size, size
    exactly = torch.ones(x.shape[-1], dtype=torch.bool)
    exactly[2 * half:] = False
    bound += (ROUNDOFF[x.dtype] * y.abs() + TINY[x.dtype]) * exactly
    return y, bound


# ---- sums of weights -----------------------------------------------------------------------------
def slots_of(table_row, keys, page, pages):
    """Slots of a request's keys, -1 where the page is not there."""
    out = []
    for j in range(keys):
        cell = table_row[j // page] if j // page < len(table_row) else -1
        out.append(cell * page + j % page if 0 <= cell < pages else -1)
    return out


def weights(q, key_cache, table, q_offsets, kv_lengths, known, lse, before, after, scale, decay, tree=None):
    """(value, bound) of the sums [pages, page].  A score carries (dim + 8) roundings of the sum of |q| |k|, and with the
    log-sum it is off by that much and 2^-22 (|score| + |lse|) + 2^-22; a key's sum adds 2^-24 a term."""
    q, keys, lse64 = q.cpu().double(), key_cache.cpu().double(), lse.cpu().double()
    pages, page, kv_heads, dim = keys.shape
    heads, room = q.shape[1], len(table[0]) * page
    value = after.cpu().double().clone().flatten()
    bound = torch.zeros_like(value)
    flat = keys.reshape(pages * page, kv_heads, dim)
    old = None if before is None else before.cpu().double().flatten()
    for r, length in enumerate(kv_lengths):
        length = max(0, length)
        held = min(length, room)
        n = q_offsets[r + 1] - q_offsets[r]
        ahead = length - n
        slots = slots_of(table[r], held, page, pages)
        have = [j for j in range(held) if slots[j] >= 0]
        if not have:
            continue
        at = torch.tensor([slots[j] for j in have])
        total, off = torch.zeros(len(have), dtype=torch.float64), torch.zeros(len(have), dtype=torch.float64)
        terms = 0
        for h in range(heads):
            k = flat[at, h // (heads // kv_heads)]
            for i in range(n):
                l = lse64[h, q_offsets[r] + i]
                if l == -math.inf:
                    continue
                row = q[q_offsets[r] + i, h]
                if tree is None:
                    seen = torch.tensor([j <= ahead + i for j in have])
                else:
                    word = tree[q_offsets[r] + i] % (1 << 64)
                    seen = torch.tensor([j < ahead or (j - ahead < 64 and bool(word >> (j - ahead) & 1)) for j in have])
                score = k @ row * scale
                size = k.abs() @ row.abs() * scale
                w = torch.where(seen, torch.exp(score - l), 0.0)
                total += w
                off += w * ((dim + 8) * 2.0 ** -23 * (size + 1.0) + 2.0 ** -22 * (score.abs() + l.abs() + 1.0))
                terms += 1
        off += total.abs() * 2.0 ** -23 * (terms + 2)
        k = ahead if known is None else known[r]
        if old is not None:
            add = torch.tensor([j < k for j in have]) * old[at] * decay
            total, off = total + add, off + add.abs() * 2.0 ** -22 + total.abs() * 2.0 ** -23
        value[at], bound[at] = total, off
    return value.view(pages, page), bound.view(pages, page)


# ---- eviction ------------------------------------------------------------------------------------
def release(kv_lengths, keep_lengths, page, table, shifts=None, most_moves=None):
    kept, out_shifts, pages = [], [], []
    for r, (n, k) in enumerate(zip(kv_lengths, keep_lengths)):
        n, k = max(0, n), max(0, k)
        k = min(n, k)
        if most_moves is not None and min(k, n - k) > most_moves:
            k = n
        kept.append(k)
        out_shifts.append((shifts[r] if shifts else 0) + n - k)
        pages += [c for c in table[r][-(-k // page):-(-n // page)] if c >= 0]
    return kept, out_shifts, pages


def evict(weight, position, table, page, kv_lengths, kept_lengths, first, recent, shifts, width):
    """Moves [requests][width] from flat lists of slots' weights and positions."""
    pages = len(weight) // page
    moves_from, moves_to = [], []
    for r, length in enumerate(kv_lengths):
        length = max(0, length)
        n = min(length, len(table[r]) * page)
        keep = min(max(0, kept_lengths[r]), n)
        slots = slots_of(table[r], n, page, pages)
        late = shifts[r] + length - recent if recent else math.inf

        def key(j):
            s = slots[j]
            if s < 0:
                return (0, 0.0, -j)
            if position is not None and (position[s] < first or position[s] >= late):
                return (3, 0.0, -j)
            return (1, 0.0, -j) if math.isnan(weight[s]) else (2, weight[s] + 0.0, -j)

        stays = set(sorted(range(n), key=key, reverse=True)[:keep])
        source = [slots[j] for j in range(keep, n) if j in stays]
        target = [slots[j] for j in range(keep) if j not in stays]
        assert len(source) == len(target) <= min(keep, n - keep)
        pad = lambda x: (x + [-1] * width)[:width]
        moves_from.append(pad(source))
        moves_to.append(pad(target))
    return moves_from, moves_to


# ---- the recurrence ------------------------------------------------------------------------------
def _step_error(l, a, size, x):
    """Of one step of 32 bits, with `size` a bound on |h| before it: exp(l) - 1 is good to 2^-21 of itself, or exp(l) to
    2^-21 of itself, and two sums round; twice that, as a state that comes from a chunk before it is made in two ways."""
    small = l.abs() <= 0.0625
    return 2.0 ** -20 * torch.where(small, l.abs(), a) * size + 2.0 ** -21 * (torch.where(small, size, a * size) + x.abs())


def recurrence(x, log_decay, lengths, initial=None, dout=None, dfinal=None):
    """(value, bound) of out and final, and with dout of dx, dlog_decay and dinitial."""
    u, tiny = ROUNDOFF[x.dtype], TINY[x.dtype]
    x, l = x.cpu().double(), log_decay.cpu().double()
    a = l.exp()
    count, channels = len(lengths), x.shape[1]
    first = torch.zeros(count, channels, dtype=torch.float64) if initial is None else initial.cpu().double()
    out, off, final, final_off = torch.zeros_like(x), torch.zeros_like(x), first.clone(), torch.zeros_like(first)
    begin = 0
    for b, n in enumerate(lengths):
        h, e, size = first[b].clone(), torch.zeros(channels, dtype=torch.float64), first[b].abs()
        for t in range(begin, begin + n):
            e = a[t] * e + _step_error(l[t], a[t], size, x[t])
            h, size = a[t] * h + x[t], a[t] * size + x[t].abs()
            out[t], off[t] = h, e
        final[b], final_off[b] = h, e
        begin += n
    result = {"out": (out, off + u * out.abs() + tiny), "final": (final, final_off + tiny)}
    if dout is None:
        return result
    dout = dout.cpu().double()
    dx, dl, dx_off, dl_off = (torch.zeros_like(x) for _ in range(4))
    last = torch.zeros_like(first) if dfinal is None else dfinal.cpu().double()
    dfirst, dfirst_off = last.clone(), torch.zeros_like(first)
    begin = sum(lengths)
    for b in range(count - 1, -1, -1):
        c, e, size = last[b].clone(), torch.zeros(channels, dtype=torch.float64), last[b].abs()
        begin -= lengths[b]
        for t in range(begin + lengths[b] - 1, begin - 1, -1):
            g, g_size, g_off = dout[t] + c, dout[t].abs() + size, e + 2.0 ** -22 * (dout[t].abs() + size)
            c, size = a[t] * g, a[t] * g_size
            e = a[t] * g_off + _step_error(l[t], a[t], g_size, torch.zeros_like(g))
            h, h_off = (out[t - 1], off[t - 1] + u * out[t - 1].abs() + tiny) if t > begin else (first[b], torch.zeros_like(g))
            dx[t], dx_off[t] = g, g_off + u * g.abs() + tiny
            dl[t], dl_off[t] = c * h, u * (c * h).abs() * (1 + u) + (c.abs() + e) * h_off + e * h.abs() + tiny
        dfirst[b], dfirst_off[b] = c, e
    return result | {"dx": (dx, dx_off), "dlog_decay": (dl, dl_off), "dinitial": (dfirst, dfirst_off + tiny)}


# ---- comparing -----------------------------------------------------------------------------------
def check(name, got, want):
    """Every item within its bound of the value."""
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    if not got.numel():
        return
    over = ((got - value).abs() - bound).nan_to_num(nan=math.inf)
    worst = over.argmax()
    assert over.flatten()[worst] <= 0, \
        f"{name}: item {int(worst)} is {float(got.flatten()[worst])}, not {float(value.flatten()[worst])} +- {float(bound.flatten()[worst])}"
