"""Requests served for long in bounded memory: a recurrent layer with a pool of states and an attention layer with a paged cache that is
cut as it grows, step by step, against a plain record of every key that is still there.  And a training step of both layers."""
import math
import random

import pytest
import torch

import attention_oracle
import long_request_oracle as oracle
from gpu_util import log

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, ROTARY, PAGE, PAGES, CHANNELS = 6, 2, 64, 32, 8, 90, 80


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).cuda()


class Server:
    """The library's calls of a step, in the order that a program makes them; buffers of a fixed capacity."""

    def __init__(self, hip, requests, capacity, width=40):
        self.hip, self.count = hip, requests
        empty = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device="cuda")
        self.table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
        self.free = list(range(PAGES))
        random.Random(4).shuffle(self.free)
        self.cached, self.shifts = empty(requests), empty(requests)
        self.offsets, self.kv, self.kept, self.counts = empty(requests + 1), empty(requests), empty(requests), empty(2)
        self.request, self.position, self.slot = empty(capacity), empty(capacity), empty(capacity, dtype=torch.int64)
        self.released, self.released_counts = empty(PAGES), empty(2)
        self.moves = [empty(requests, 60, dtype=torch.int64) for _ in range(2)]
        self.keys, self.values = (torch.zeros(PAGES, PAGE, KV_HEADS, DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.weights = torch.full((PAGES, PAGE), 1e9, device="cuda")  # (what a page held before does not count)
        self.slot_positions = torch.full((PAGES, PAGE), -1, dtype=torch.int32, device="cuda")
        self.states = torch.zeros(requests + 2, CHANNELS, device="cuda")
        self.rows = ints(list(range(requests + 1, 1, -1)))
        self.frequencies = hip.rotary_frequencies(ROTARY, scaling="bands", scale=4.0, trained=64.0)
        self.q_out = torch.zeros(capacity, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
        self.out, self.lse = torch.zeros_like(self.q_out), torch.zeros(HEADS, capacity, device="cuda")
        self.mixed = torch.zeros(capacity, CHANNELS, dtype=torch.bfloat16, device="cuda")

    def step(self, new, q, k, v, x, log_decay):
        hip = self.hip
        free = ints(self.free)
        hip.page_plan(self.cached, ints(new), PAGE, free, self.table, self.offsets, self.kv, self.request, self.position, self.slot, self.counts)
        hip.recurrence("bf16", x, log_decay, self.offsets, self.mixed, initial=self.states, final=self.states, rows=self.rows)
        hip.paged_write_rotary("bf16", q, k, v, self.position, self.frequencies, self.slot, self.q_out, self.keys, self.values,
                               slot_positions=self.slot_positions, requests=self.request, shifts=self.shifts, factor=1.1)
        hip.attention_paged("bf16", self.q_out, self.keys, self.values, self.table, self.offsets, self.kv, self.out, self.lse)
        hip.attention_paged_weights("bf16", self.q_out, self.keys, self.table, self.offsets, self.kv, self.lse, self.weights,
                                    weights_in=self.weights, known_lengths=self.cached, decay=0.9)

    def cut(self, keep, first, recent):
        hip, before = self.hip, self.shifts.clone()
        hip.page_release(self.kv, ints(keep), PAGE, self.table, self.kept, self.released, self.released_counts, shifts=self.shifts,
                         shifts_out=self.shifts, most_moves=self.moves[0].shape[1])
        hip.evict_plan(self.weights, self.slot_positions, self.table, self.kv, self.kept, *self.moves, first=first, recent=recent,
                       shifts=before)
        hip.paged_move("bf16", *self.moves, self.keys, self.values, weights=self.weights, positions=self.slot_positions)
        taken, given = int(self.counts[1]), int(self.released_counts[0])
        self.free = self.free[taken:] + self.released[:given].tolist()
        self.cached.copy_(self.kept)


def test_requests_that_outgrow_their_budget(hip, dev):
    rng, g = random.Random(1), torch.Generator().manual_seed(2)
    count, capacity, budget = 3, 200, 40
    server = Server(hip, count, capacity)
    record = [dict() for _ in range(count)]  # position: (key row, value row, sum of weights)
    states = torch.zeros(count, CHANNELS, dtype=torch.float64)
    state_bound = torch.zeros(count, CHANNELS, dtype=torch.float64)
    seen = [0] * count
    evictions = 0
    for step in range(26):
        new = [50, 9, 130] if step == 0 else [rng.choice([1, 1, 1, 0, 3]) for _ in range(count)]
        total = sum(new)
        randn = lambda *s: torch.randn(*s, generator=g)
        q, k, v = ((randn(capacity, h, DIM)).to(torch.bfloat16).cuda() for h in (HEADS, KV_HEADS, KV_HEADS))
        x = randn(capacity, CHANNELS).to(torch.bfloat16).cuda()
        log_decay = (-0.3 * randn(capacity, CHANNELS).abs()).to(torch.bfloat16).cuda()
        server.q_out.fill_(5.0)
        server.mixed.fill_(5.0)
        lengths_before = server.cached.tolist()
        server.step(new, q, k, v, x, log_decay)
        torch.cuda.synchronize()
        log(f"step {step} new {new} lengths {server.kv.tolist()} free {len(server.free)}")

        # The recurrent layer goes on from where it was.
        want = oracle.recurrence(x[:total], log_decay[:total], new, states)
        spread = [b for b, n in enumerate(new) for _ in range(n)]
        value, bound = want["out"]
        oracle.check("recurrent layer", server.mixed[:total], (value, bound + state_bound[spread]))  # (decays only shrink what was off)
        states, bound = want["final"]
        state_bound = state_bound + bound
        assert bool((server.mixed[total:] == 5.0).all()) and bool((server.q_out[total:] == 5.0).all())

        # Rows are turned by the positions that they have in their requests, evicted ones counted.
        positions = [p for b, n in enumerate(new) for p in range(seen[b], seen[b] + n)]
        turned = oracle.turn(q[:total], torch.tensor(positions, dtype=torch.int32), server.frequencies, False, 1.1)
        oracle.check("queries", server.q_out[:total], turned)
        slots = server.slot[:total].tolist()
        assert min(slots + [0]) >= 0 and server.slot[total:].eq(-1).all()
        keys, values = server.keys.cpu().view(PAGES * PAGE, KV_HEADS, DIM), server.values.cpu().view(PAGES * PAGE, KV_HEADS, DIM)
        oracle.check("keys", keys[slots], oracle.turn(k[:total], torch.tensor(positions, dtype=torch.int32), server.frequencies, False, 1.1))
        assert torch.equal(values[slots], v[:total].cpu())

        # Attention of each row to the keys that are there, and what they gained.
        sums = server.weights.cpu().flatten()
        at, q_out = 0, server.q_out.cpu()
        for b, n in enumerate(new):
            for i in range(n):
                record[b][seen[b] + i] = [keys[slots[at + i]], values[slots[at + i]], 0.0, 0.0]
            old = sorted(p for p in record[b] if p < seen[b])
            order = old + [seen[b] + i for i in range(n)]
            assert len(order) == lengths_before[b] + n
            if not order:
                continue
            gain, gain_off = torch.zeros(len(order), dtype=torch.float64), torch.zeros(len(order), dtype=torch.float64)
            visible = torch.ones(n, len(order), dtype=torch.bool).tril(len(order) - n)
            for h in range(HEADS) if n else ():
                kv_head = h // (HEADS // KV_HEADS)
                kk = torch.stack([record[b][p][0][kv_head] for p in order]).double()
                vv = torch.stack([record[b][p][1][kv_head] for p in order]).double()
                qq = q_out[at:at + n, h].double()
                out, lse, weight, bound, relative, score = attention_oracle.head(qq, kk, vv, visible, DIM ** -0.5, torch.bfloat16)
                oracle.check("attention", server.out[at:at + n, h], (out, bound))
                gain += weight.sum(0)
                # The scores of both passes and the log-sum are off by their bounds.
                gain_off += (weight * (2 * relative + 2 * score + 2.0 ** -17)[:, None]).sum(0)
            for p, w, o in zip(order, gain.tolist(), gain_off.tolist()):
                r = record[b][p]
                r[2], r[3] = (0.9 * r[2] if p < seen[b] else 0.0) + w, (0.9 * r[3] if p < seen[b] else 0.0) + o + 1e-6 * (r[2] + w)
            at += n
            seen[b] += n

        # Sums, by the slots' positions.
        table, kv = server.table.tolist(), server.kv.tolist()
        where = server.slot_positions.cpu().flatten().tolist()
        held = [oracle.slots_of(table[b], kv[b], PAGE, PAGES) for b in range(count)]
        for b in range(count):
            assert sorted(where[s] for s in held[b]) == sorted(record[b])
            for s in held[b]:
                value, off = record[b][where[s]][2:]
                assert abs(float(sums[s]) - value) <= off + 1e-6, (b, where[s])

        # Cut what has grown past the budget by a few keys.
        keep = [budget if n > budget + 4 else n for n in kv]
        evictions += sum(k < n for k, n in zip(keep, kv))
        ranked = []
        for b in range(count):
            late = seen[b] - 6
            by = sorted(range(kv[b]), key=lambda j: (where[held[b][j]] < 2 or where[held[b][j]] >= late, float(sums[held[b][j]]), -j), reverse=True)
            stay = {where[held[b][j]] for j in by[:keep[b]]}
            ranked.append(stay if keep[b] < kv[b] else set(record[b]))
        server.cut(keep, first=2, recent=6)
        torch.cuda.synchronize()
        assert server.kept.tolist() == keep
        table = server.table.tolist()
        where = server.slot_positions.cpu().flatten().tolist()
        keys, values, moved = server.keys.cpu().view(-1, KV_HEADS, DIM), server.values.cpu().view(-1, KV_HEADS, DIM), server.weights.cpu().flatten()
        used = []
        for b in range(count):
            record[b] = {p: r for p, r in record[b].items() if p in ranked[b]}
            slots = oracle.slots_of(table[b], keep[b], PAGE, PAGES)
            assert {where[s] for s in slots} == ranked[b] and len(slots) == len(ranked[b])
            for s in slots:
                assert torch.equal(keys[s], record[b][where[s]][0]) and torch.equal(values[s], record[b][where[s]][1])
                assert abs(float(moved[s]) - record[b][where[s]][2]) <= record[b][where[s]][3] + 1e-6
            used += table[b][:-(-keep[b] // PAGE)]
            assert server.shifts[b] == seen[b] - keep[b]
        assert sorted(used + server.free) == list(range(PAGES))
    assert evictions >= 6


def test_a_training_step(hip, dev):
    """x -> recurrence -> heads -> rotary -> attention over packed sequences and back, its gradients against differences of a plain
    form in 64 bits."""
    lengths, heads, dim, width = [20, 1, 33], 2, 32, 64
    tokens, g = sum(lengths), torch.Generator().manual_seed(5)
    offsets = ints([0, 20, 21, 54])
    x = torch.randn(tokens, width, generator=g).to(torch.bfloat16).cuda()
    log_decay = (-0.5 * torch.rand(tokens, width, generator=g)).to(torch.bfloat16).cuda()
    value = torch.randn(tokens, heads, dim, generator=g).to(torch.bfloat16).cuda()
    dout = torch.randn(tokens, heads, dim, generator=g).to(torch.bfloat16).cuda()
    positions = ints(list(range(20)) + [0] + list(range(33)))
    f = hip.rotary_frequencies(dim)
    h, turned, out, dturned, dk, dv, dh, dx, dl = (torch.empty(tokens, width, dtype=torch.bfloat16, device=dev) for _ in range(9))
    rows = lambda t: t.view(tokens, heads, dim)
    lse = torch.empty(heads, tokens, device=dev)
    hip.recurrence("bf16", x, log_decay, offsets, h)
    hip.rotary("bf16", rows(h), None, positions, f, rows(turned), None)
    hip.attention_packed("bf16", rows(turned), rows(turned), value, offsets, offsets, rows(out), lse)
    hip.attention_packed_backward("bf16", rows(turned), rows(turned), value, rows(out), lse, dout, offsets, offsets, rows(dturned), rows(dk), rows(dv))
    dturned += dk  # the same rows are queries and keys
    hip.rotary("bf16", rows(dturned), None, positions, f, rows(dh), None, inverse=True)
    hip.recurrence_backward("bf16", log_decay, h, dh, offsets, dx, dl)

    def loss(x, l):
        angle = positions.cpu().double()[:, None, None] * f.cpu()
        total, at = 0.0, 0
        for n in lengths:
            state, hs = torch.zeros(width, dtype=torch.float64), []
            for t in range(at, at + n):
                state = l[t].exp() * state + x[t]
                hs.append(state)
            r = torch.stack(hs).view(n, heads, dim)
            a, b, c, s = r[..., :16], r[..., 16:], angle[at:at + n].cos(), angle[at:at + n].sin()
            r = torch.cat([a * c - b * s, a * s + b * c], -1).transpose(0, 1)
            scores = (r @ r.transpose(-1, -2) * dim ** -0.5).masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
            o = scores.softmax(-1) @ value[at:at + n].cpu().double().transpose(0, 1)
            total = total + (o * dout[at:at + n].cpu().double().transpose(0, 1)).sum()
            at += n
        return total

    leaves = [t.cpu().double().requires_grad_() for t in (x, log_decay)]
    want = torch.autograd.grad(loss(*leaves), leaves)
    step, v = 1e-6, torch.randn(tokens, width, generator=g, dtype=torch.float64)
    for i, w in enumerate(want):
        moved = lambda s: [t.detach() + (s * v if i == j else 0.0) for j, t in enumerate(leaves)]
        difference = float(loss(*moved(step)) - loss(*moved(-step))) / (2 * step)
        assert abs(difference - float((w * v).sum())) <= 1e-5 * float((w * v).abs().sum())
    # Seven tensors on the way are rounded to 16 bits, 2^-8 of an item each at most; scores of a size of about 5 carry two of them into
    # their weights, and the recurrence adds up some ten tokens' worth: norm by norm a twentieth holds all of it.
    for got, w in zip((dx, dl), want):
        assert float((got.cpu().double() - w).norm()) <= 0.05 * float(w.norm())
