"""Sums of attention weights over a paged cache, and eviction by them, against plain forms."""
import math
import random

import pytest
import torch

import long_request_oracle as oracle
from attention_oracle import offsets_of
from gpu_util import log

pytestmark = pytest.mark.gpu

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).cuda()


def tables(lengths, page, seed=1, spare=3, width=None, missing=()):
    """Block table rows over shuffled pages, and how many pages there are; (request, cell) in `missing` have none."""
    used = [-(-max(0, n) // page) for n in lengths]
    pages = sum(used) + spare
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    width = max(used + [1]) if width is None else width
    table, at = [], 0
    for r, n in enumerate(used):
        row = order[at:at + n]
        at += n
        table.append([-1 if (r, c) in missing else row[c] if c < n else -1 for c in range(width)])
    return table, pages


# ---- sums of weights -----------------------------------------------------------------------------
def plain_lse(q, keys, table, q_offsets, lengths, page, scale, tree):
    """Log-sums of what each row sees, rounded from 64 bits."""
    heads, group = q.shape[1], q.shape[1] // keys.shape[2]
    lse = torch.full((heads, q.shape[0]), -math.inf, dtype=torch.float64)
    flat = keys.cpu().double().flatten(0, 1)
    for r, length in enumerate(lengths):
        length = max(0, length)
        n = q_offsets[r + 1] - q_offsets[r]
        slots = oracle.slots_of(table[r], min(length, len(table[r]) * page), page, keys.shape[0])
        for i in range(n):
            word = None if tree is None else tree[q_offsets[r] + i] % (1 << 64)
            ahead = length - n
            seen = [s for j, s in enumerate(slots) if s >= 0 and (
                j <= ahead + i if tree is None else j < ahead or (j - ahead < 64 and word >> (j - ahead) & 1))]
            if seen:
                for h in range(heads):
                    lse[h, q_offsets[r] + i] = torch.logsumexp(flat[seen, h // group] @ q[q_offsets[r] + i, h].cpu().double() * scale, 0)
    return lse.float().cuda()


def check_weights(hip, suffix, lengths, new, heads, kv_heads, dim, page, decay=0.9, known=None, tree=None, before=True, seed=1, missing=(),
                  stated=None, order=(0, 1, 2, 3), scale=None, width=None):
    log(f"{suffix} lengths {lengths[:8]} new {new[:8]} heads {heads}/{kv_heads} dim {dim} page {page}")
    g = torch.Generator().manual_seed(seed)
    dtype = DTYPE[suffix]
    table, pages = tables(lengths, page, seed, missing=missing, width=width)
    q_offsets = [0]
    for n in new:
        q_offsets.append(q_offsets[-1] + n)
    q = (torch.randn(q_offsets[-1], heads, dim, generator=g) * 1.5).to(dtype).cuda()
    shape = [(pages, page, kv_heads, dim)[a] for a in order]
    back = [order.index(a) for a in range(4)]
    keys = torch.randn(shape, generator=g).to(dtype).cuda().permute(back)
    old = torch.rand(pages, page, generator=g).cuda() if before else None
    after = torch.full((pages, page), -5.0, device="cuda")
    used = dim ** -0.5 if scale is None else scale
    lse = plain_lse(q, keys, table, q_offsets, lengths, page, used, tree)
    words = None if tree is None else ints([w - (1 << 64) if w >> 63 else w for w in tree], torch.int64)
    hip.attention_paged_weights(suffix, q, keys, ints(table), ints(q_offsets), ints(lengths), lse, after, weights_in=old,
                                known_lengths=None if known is None else ints(known), decay=decay, tree=words, max_kv_length=stated,
                                scale=scale)
    want = oracle.weights(q, keys, table, q_offsets, lengths, known, lse, old, torch.full((pages, page), -5.0), used, decay, tree)
    oracle.check("weights", after, want)
    return q, keys, table, q_offsets, lse, old, after


@pytest.mark.parametrize("suffix", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [8, 32, 64, 72, 80, 96, 104, 120, 128])
def test_head_sizes(hip, dev, suffix, dim):
    check_weights(hip, suffix, [70, 1, 33], [1, 1, 3], 4, 2, dim, 16)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 1), (3, 3), (6, 2), (5, 5), (14, 2), (16, 1), (40, 1), (8, 8), (12, 4)])
def test_groups(hip, dev, heads, kv_heads):
    check_weights(hip, "bf16", [100, 17], [1, 5], heads, kv_heads, 64, 16)
    check_weights(hip, "bf16", [70], [33], heads, kv_heads, 32, 8)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 256])
def test_pages_that_end_inside_a_tile(hip, dev, page):
    check_weights(hip, "f16", [1, 15, 16, 17, 63, 64, 65, 129, 300], [1] * 9, 4, 2, 64, page)
    check_weights(hip, "bf16", [200, 77], [40, 77], 2, 1, 32, page)


def test_lengths(hip, dev):
    check_weights(hip, "bf16", [0, 1, 2, 0, 64, 500], [0, 1, 2, 0, 0, 1], 4, 2, 32, 16)
    check_weights(hip, "bf16", [3, 10], [5, 10], 4, 2, 32, 16)       # fewer keys than new rows: the first see none
    check_weights(hip, "bf16", [-4, 20], [1, 1], 4, 2, 32, 16)
    check_weights(hip, "bf16", [60], [1], 4, 2, 32, 16, width=2)     # keys past the table
    check_weights(hip, "bf16", [700, 90], [1, 2], 4, 2, 32, 16, stated=1)
    check_weights(hip, "bf16", [700, 90], [1, 2], 4, 2, 32, 16, stated=1 << 20)


def test_many_requests(hip, dev):
    rng = random.Random(3)
    check_weights(hip, "bf16", [rng.randrange(1, 40) for _ in range(300)], [1] * 300, 2, 1, 32, 16)


@pytest.mark.parametrize("suffix", ["bf16", "f16"])
def test_units_dealt_out_over_all_requests(hip, dev, suffix):
    """Lengths stated long enough that a request's own workgroups would be few; more requests than are counted at once."""
    rng = random.Random(5)
    lengths = [rng.choice((0, 1, 17, rng.randrange(1, 90), 130)) for _ in range(299)]
    few = [min(n, 1) for n in lengths]
    check_weights(hip, suffix, lengths + [700], few + [1], 2, 1, 32, 16, stated=1 << 20)
    check_weights(hip, suffix, [700] + lengths, [40] + few, 4, 2, 64, 16, stated=1 << 20)       # one of many rows
    check_weights(hip, suffix, lengths + [700], few + [300], 4, 2, 72, 24, stated=1 << 20)
    check_weights(hip, suffix, lengths + [300], [min(n, 20) for n in lengths] + [250], 4, 2, 32, 16, stated=1 << 20)
    check_weights(hip, suffix, lengths + [300], [0] * 299 + [140], 4, 2, 32, 16, stated=1 << 20)  # no row but one request's


@pytest.mark.parametrize("suffix,dim", [("bf16", 64), ("f16", 128), ("bf16", 40)])
def test_rows_that_workgroups_share(hip, dev, suffix, dim):
    check_weights(hip, suffix, [700], [600], 4, 2, dim, 16)
    check_weights(hip, suffix, [1], [257], 4, 2, dim, 16)
    check_weights(hip, suffix, [700, 90, 0, 50], [600, 3, 0, 0], 4, 2, dim, 24)
    check_weights(hip, suffix, [700, 300], [600, 210], 4, 2, dim, 16, stated=1)   # more units than the partial sums have room for
    check_weights(hip, suffix, [90, 2000], [1, 1000], 3, 1, dim, 64, known=[20, 999])


def test_shared_rows_are_the_same_every_time_in_a_graph(hip, dev):
    q, keys, table, q_offsets, lse, old, first = check_weights(hip, "bf16", [700, 90], [600, 3], 4, 2, 64, 16)
    after = torch.full_like(first, -5.0)
    arguments = ints(table), ints(q_offsets), ints([700, 90])
    size = hip.attention_paged_weights_temp_bytes(2, 603, arguments[0].shape[1] * 16, 4, 2, 64)
    assert size > 0
    temp = torch.full((size,), 0x7F, dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip.attention_paged_weights("bf16", q, keys, *arguments, lse, after, weights_in=old, decay=0.9, temp=temp)
    for _ in range(3):
        after.fill_(-5.0)
        temp.fill_(0x7F)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(after, first)


def test_orders_of_the_cache(hip, dev):
    for order in ((0, 1, 2, 3), (2, 0, 1, 3), (1, 0, 2, 3), (0, 2, 1, 3)):
        check_weights(hip, "bf16", [90, 40], [1, 2], 4, 2, 40, 16, order=order)


def test_known_keys_and_missing_pages(hip, dev):
    check_weights(hip, "bf16", [90, 40, 33], [1, 2, 1], 4, 2, 64, 16, known=[0, 25, 99], scale=0.3)
    check_weights(hip, "bf16", [90, 40, 33], [1, 2, 1], 4, 2, 64, 16, before=False)
    check_weights(hip, "bf16", [90, 40, 33], [1, 2, 1], 4, 2, 64, 16, decay=0.0)
    check_weights(hip, "bf16", [90, 40, 33], [1, 2, 1], 4, 2, 64, 16, missing={(0, 1), (1, 2), (2, 0)})


def test_trees(hip, dev):
    rng, words = random.Random(5), []
    new = [5, 64, 1, 70]
    for n in new:
        mask = []
        for i in range(n):
            parent = rng.randrange(-1, i)
            mask.append(((mask[parent] if parent >= 0 else 0) | 1 << min(i, 63)) if i % 11 else 0)
        words += mask
    check_weights(hip, "bf16", [100, 64, 30, 200], new, 4, 2, 32, 16, tree=words)


def test_a_row_that_sees_nothing_weighs_nothing(hip, dev):
    q, keys, table, q_offsets, lse, old, _ = check_weights(hip, "bf16", [90], [2], 2, 1, 32, 16)
    lse[:, 1] = -math.inf
    after = torch.zeros_like(old)
    hip.attention_paged_weights("bf16", q, keys, ints(table), ints(q_offsets), ints([90]), lse, after)
    oracle.check("weights", after, oracle.weights(q, keys, table, q_offsets, [90], None, lse, None, torch.zeros(after.shape), 32 ** -0.5, 1.0))


def test_not_finite_stays_with_what_meets_it(hip, dev):
    q, keys, table, q_offsets, lse, old, clean = check_weights(hip, "bf16", [90, 80], [1, 1], 2, 1, 32, 16)
    slots = oracle.slots_of(table[0], 90, 16, keys.shape[0])
    free = [p for p in range(keys.shape[0]) if p not in table[0] + table[1]]
    keys[free[0]] = math.nan                               # no request's
    keys.view(-1, 1, 32)[slots[89] + 1 if slots[89] % 16 < 15 else slots[0]] = math.nan  # past the end, in the last page
    keys.view(-1, 1, 32)[slots[20]] = math.inf
    after = torch.full_like(old, -5.0)
    call = lambda: hip.attention_paged_weights("bf16", q, keys, ints(table), ints(q_offsets), ints([90, 80]), lse, after, weights_in=old,
                                               decay=0.9)
    call()
    same = torch.ones(old.numel(), dtype=torch.bool)
    same[slots[20]] = False
    assert torch.equal(after.flatten()[same.cuda()], clean.flatten()[same.cuda()])
    q[0, 1, 3] = math.nan
    call()
    mine = torch.zeros(old.numel(), dtype=torch.bool)
    mine[slots] = True
    assert bool(after.flatten()[mine.cuda()].isnan().all()) and torch.equal(after.flatten()[~mine.cuda()], clean.flatten()[~mine.cuda()])


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lengths,new,tree,stated", [
    ([90, 80], [3, 1], False, None),                # few rows
    ([90, 80], [3, 1], True, None),
    ([300, 50], [40, 9], False, None),              # many
    ([300, 50], [40, 9], True, None),
    ([700, 90], [600, 3], False, None),             # rows that workgroups share
    ([700] + [20] * 299, [40] + [1] * 299, False, 1 << 20),  # units dealt out, of both kinds
])
def test_rows_without_a_log_sum_may_hold_anything(hip, dev, bad, lengths, new, tree, stated):
    """They give no weight, to the keys before the new ones either, the first row of a request among them."""
    words = [2 ** min(i + 1, 64) - 1 for n in new for i in range(n)] if tree else None
    q, keys, table, q_offsets, lse, old, _ = check_weights(hip, "bf16", lengths, new, 4, 2, 64, 16, tree=words, stated=stated)
    out_of_it = sorted({0, 2, q_offsets[1] - 1} | ({37, 301, 302} & set(range(q_offsets[1]))))
    lse[:, out_of_it] = -math.inf
    lse[1, q_offsets[1] - 2] = -math.inf  # one head of a row
    results = []
    for value in (0.0, bad):
        q[out_of_it] = value
        q[q_offsets[1] - 2, 1] = value
        after = torch.full_like(old, -5.0)
        hip.attention_paged_weights("bf16", q, keys, ints(table), ints(q_offsets), ints(lengths), lse, after, weights_in=old, decay=0.9,
                                    tree=None if words is None else ints([w - (1 << 64) if w >> 63 else w for w in words], torch.int64),
                                    max_kv_length=stated)
        results.append(after)
    assert torch.equal(*results)


@pytest.mark.parametrize("kv_heads", [31, 32, 33, 40, 63, 64, 65, 70, 130])
def test_many_key_heads(hip, dev, kv_heads):
    """More than have their log-sums (32) or the places of their rows (64) at hand at once; with as many rows as fit beside them, and more."""
    check_weights(hip, "bf16", [40, 3, 17], [1, 1, 1], kv_heads, kv_heads, 16, 8)
    check_weights(hip, "f16", [40, 30], [20, 9], kv_heads, kv_heads, 16, 8)
    check_weights(hip, "bf16", [70, 9], [50, 1], kv_heads, kv_heads, 8, 16)


def test_weights_from_the_framework_s_attention(hip, dev):
    """With the lse that attention_paged gave, a step's weights add up to the number of its rows and heads."""
    lengths, new = [300, 77, 1000], [1, 3, 20]
    q, keys, table, q_offsets, _, _, _ = check_weights(hip, "bf16", lengths, new, 8, 2, 64, 16)
    out, lse = torch.empty_like(q), torch.empty(8, q.shape[0], device=dev)
    hip.attention_paged("bf16", q, keys, keys, ints(table), ints(q_offsets), ints(lengths), out, lse)
    after = torch.zeros(keys.shape[:2], device=dev)
    hip.attention_paged_weights("bf16", q, keys, ints(table), ints(q_offsets), ints(lengths), lse, after)
    for r, n in enumerate(new):
        slots = oracle.slots_of(table[r], lengths[r], 16, keys.shape[0])
        # Scores of both passes are off by (64 + 8) 2^-23 of at most 100 each, and the sums by 2^-18.
        assert abs(float(after.flatten()[slots].double().sum()) - 8 * n) <= 8 * n * (2 * 72 * 100 * 2.0 ** -23 + 2.0 ** -18)


# ---- lengths and pages ---------------------------------------------------------------------------
def check_release(hip, kv, keep, page, shifts=None, most=None, missing=(), capacity=None, seed=1):
    table, _ = tables(kv, page, seed, missing=missing)
    count = len(kv)
    kept, pages, counts, moved = (torch.full((n,), -9, dtype=torch.int32, device="cuda")
                                  for n in (count, 4000 if capacity is None else capacity, 2, count))
    hip.page_release(ints(kv), ints(keep), page, ints(table).view(count, -1) if count else ints([[]]), kept, pages, counts,
                     shifts=None if shifts is None else ints(shifts), shifts_out=moved, most_moves=most)
    want = oracle.release(kv, keep, page, table, shifts, most)
    assert kept.tolist() == want[0] and moved.tolist() == want[1] and counts.tolist() == [len(want[2]), sum(want[0])]
    n = min(len(want[2]), pages.numel())
    assert pages.tolist() == want[2][:n] + [-9] * (pages.numel() - n)


@pytest.mark.parametrize("page", [1, 16, 24])
def test_release(hip, dev, page):
    check_release(hip, [40, 17, 0, 100, 16], [20, 17, 5, 0, 15], page)
    check_release(hip, [40, 17, 0, 100, 16], [20, 3, 5, 70, 99], page, shifts=[5, 0, -2, 1 << 30, 7])
    check_release(hip, [40, 17, 100, 16], [20, 3, 70, 99], page, most=20)
    check_release(hip, [40, 17, 100, 16], [20, 3, 30, 4], page, most=0)
    check_release(hip, [40, -5, 100], [20, 3, -30], page)
    check_release(hip, [400, 170, 100], [20, 3, 30], page, missing={(0, 2), (0, 3), (1, 1), (2, 5)})
    check_release(hip, [400, 170, 100], [20, 3, 30], page, capacity=4)
    check_release(hip, [400, 170, 100], [20, 3, 30], page, capacity=0)
    check_release(hip, [], [], page)


def test_release_of_many(hip, dev):
    rng = random.Random(2)
    for count in (1, 63, 64, 1000, 1023, 1024, 1025, 3000):
        kv = [rng.randrange(0, 60) for _ in range(count)]
        check_release(hip, kv, [rng.randrange(0, 70) for _ in kv], 16, capacity=9000)
    check_release(hip, [9001], [17], 1, capacity=9000)
    check_release(hip, [20000, 3, 20000], [10, 1, 9000], 2, capacity=30000)


# ---- which keys stay -----------------------------------------------------------------------------
def check_plan(hip, lengths, keep, page, first=0, recent=0, shifts=None, values="random", seed=1, width=None, missing=(), stated=None,
               table_width=None):
    log(f"lengths {lengths[:8]} keep {keep[:8]} page {page} first {first} recent {recent} {values}")
    rng = random.Random(seed)
    table, pages = tables(lengths, page, seed, missing=missing, width=table_width)
    count = pages * page
    weight = {"random": lambda: [rng.expovariate(1.0) for _ in range(count)],
              "few": lambda: [float(rng.randrange(3)) for _ in range(count)],
              "same": lambda: [2.5] * count,
              "signed": lambda: [rng.choice([0.0, -0.0, 1e-42, -1e-42, -3.0, 3.0, math.inf, -math.inf, math.nan, 1e38, rng.gauss(0, 1)])
                                 for _ in range(count)]}[values]()
    weight = torch.tensor(weight, dtype=torch.float32).tolist()
    shifts = [0] * len(lengths) if shifts is None else shifts
    position = [-1] * count
    for r, n in enumerate(lengths):
        order = list(range(shifts[r], shifts[r] + n))
        for _ in range(n // 8):
            a, b = rng.randrange(n), rng.randrange(n)
            order[a], order[b] = order[b], order[a]
        for slot, p in zip(oracle.slots_of(table[r], n, page, pages), order):
            if slot >= 0:
                position[slot] = p
    width = max([1] + [min(max(0, k), n - max(0, k)) for k, n in zip(keep, lengths) if k < n]) + 2 if width is None else width
    moves = [torch.full((len(lengths), width), 99, dtype=torch.int64, device="cuda") for _ in range(2)]
    protected = bool(first or recent)
    hip.evict_plan(torch.tensor(weight, dtype=torch.float32).view(pages, page).cuda(),
                   ints(position).view(pages, page) if protected else None, ints(table), ints(lengths), ints(keep), *moves, first=first,
                   recent=recent, shifts=ints(shifts), max_kv_length=stated)
    want = oracle.evict(weight, position if protected else None, table, page, lengths, keep, first, recent, shifts, width)
    assert moves[0].tolist() == want[0] and moves[1].tolist() == want[1]


@pytest.mark.parametrize("values", ["random", "few", "same", "signed"])
@pytest.mark.parametrize("page", [1, 16, 24, 64])
def test_plan(hip, dev, page, values):
    check_plan(hip, [40, 17, 1, 100, 16], [20, 17, 1, 7, 15], page, values=values)
    check_plan(hip, [40, 17, 1, 100, 16], [20, 0, 0, 99, 1], page, values=values, first=4, recent=10)
    check_plan(hip, [1500, 1025, 3000, 64, 63, 65], [700, 1024, 100, 32, 62, 1], page, values=values, first=2, recent=64,
               shifts=[0, 70, 5, 0, 1000, 3])


@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 1023, 1024, 1025, 2047, 2048, 2049, 4096, 4097, 8191, 8193, 16384, 16385, 20000])
def test_plan_lengths(hip, dev, length):
    for keep in sorted({1, length // 3, length // 2, length - 1, length}):
        check_plan(hip, [length], [keep], 16, recent=5, seed=length)
        check_plan(hip, [length, 5], [keep, 3], 64, values="few", seed=length)


def test_plan_of_long_requests(hip, dev):
    check_plan(hip, [70000, 131072, 9], [9000, 100000, 3], 64, first=4, recent=256, shifts=[0, 9, 0])
    check_plan(hip, [140001], [70000], 64, values="few")
    check_plan(hip, [140001], [4097], 128, values="signed")


def test_plan_of_requests_longer_than_stated(hip, dev):
    check_plan(hip, [140001, 30, 17000], [70000, 3, 1], 64, stated=20000, first=3, recent=9)
    check_plan(hip, [20000, 16385, 100], [300, 16384, 99], 16, stated=16385, values="few")


def test_the_latest_keys_stay_when_requests_are_cut_again_and_again(hip, dev):
    """Lengths, pages, plan and moves as a program makes them, in two arrays of shifts by turns and no copy: a plan takes the shifts
    that page_release read.  (With what it wrote, each cut of more keys than are protected would protect none of the latest.)"""
    page, recent, first, keep, new = 8, 6, 2, [30, 17], [25, 20]
    table = torch.arange(2 * 12, dtype=torch.int32, device=dev).view(2, 12)
    keys, values = (torch.zeros(24, page, 1, 8, dtype=torch.bfloat16, device=dev) for _ in range(2))
    weights, positions = torch.zeros(24, page, device=dev), torch.full((24, page), -1, dtype=torch.int32, device=dev)
    shifts, later = torch.zeros(2, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    kept, released, counts = torch.zeros(2, dtype=torch.int32, device=dev), torch.zeros(24, dtype=torch.int32, device=dev), ints([0, 0])
    moves = [torch.empty(2, 40, dtype=torch.int64, device=dev) for _ in range(2)]
    seen = [0, 0]
    for cut in range(5):
        lengths = [int(k) + n for k, n in zip(kept.tolist(), new)]
        for r, n in enumerate(lengths):
            slots = table[r, 0].item() * page + torch.arange(n - new[r], n, device=dev)
            positions.flatten()[slots] = torch.arange(seen[r], seen[r] + new[r], dtype=torch.int32, device=dev)
            weights.flatten()[slots] = -1.0 - torch.arange(new[r], device=dev)  # the later, the lighter: without protection the latest go
            seen[r] += new[r]
        kv = ints(lengths)
        hip.page_release(kv, ints(keep), page, table, kept, released, counts, shifts=shifts, shifts_out=later)
        hip.evict_plan(weights, positions, table, kv, kept, *moves, first=first, recent=recent, shifts=shifts)
        hip.paged_move("bf16", *moves, keys, values, weights=weights, positions=positions)
        shifts, later = later, shifts
        assert kept.tolist() == [min(n, k) for n, k in zip(lengths, keep)]
        assert shifts.tolist() == [a - b for a, b in zip(seen, kept.tolist())]
        for r, n in enumerate(kept.tolist()):
            mine = positions[table[r].long()].flatten()[:n].tolist()
            assert set(range(seen[r] - recent, seen[r])) | set(range(first)) <= set(mine) and len(set(mine)) == n, (cut, r, sorted(mine))


def test_plan_corners(hip, dev):
    check_plan(hip, [50, 50, 50], [10, 60, -4], 16)
    check_plan(hip, [50, 0], [10, 10], 16)
    check_plan(hip, [50], [10], 16, recent=50)          # more protected than kept
    check_plan(hip, [50], [10], 16, first=1000)
    check_plan(hip, [50, 80], [10, 30], 16, missing={(0, 0), (1, 2), (1, 4)}, recent=9)
    check_plan(hip, [50, 80], [10, 30], 16, width=3)    # moves past the width are left out
    check_plan(hip, [50, 80], [10, 30], 16, table_width=3)
    check_plan(hip, [50, 3000], [10, 30], 16, stated=1)
    check_plan(hip, [50, 300], [10, 30], 16, stated=1 << 21)
    check_plan(hip, [30] * 700, [20] * 700, 16, recent=4, seed=9)


# ---- moving rows ---------------------------------------------------------------------------------
@pytest.mark.parametrize("suffix,kv_heads,dim,page", [("bf16", 2, 64, 16), ("f16", 8, 128, 16), ("bf16", 1, 8, 1), ("f16", 3, 80, 24),
                                                      ("bf16", 40, 128, 8), ("f16", 5, 1032, 4)])
@pytest.mark.parametrize("count", [1, 7, 64, 1000])
def test_move(hip, dev, suffix, kv_heads, dim, page, count):
    g = torch.Generator().manual_seed(count)
    pages = -(-2 * count // page) + 2
    make = lambda: torch.randn(kv_heads, pages, page, dim, generator=g).to(DTYPE[suffix]).cuda().permute(1, 2, 0, 3)
    caches = [make(), make()]
    weights, positions = torch.randn(pages, page, generator=g).cuda(), torch.arange(pages * page, dtype=torch.int32).view(pages, page).cuda()
    slots = torch.randperm(2 * count, generator=g)
    source, target = slots[:count].clone(), slots[count:].clone()
    source[::5] = -1
    target[3::7] = -1
    if count > 20:
        source[11], target[12] = pages * page + 3, 1 << 40
    want = [c.cpu().clone().reshape(pages * page, -1) for c in caches] + [weights.cpu().clone().flatten(), positions.cpu().clone().flatten()]
    real = (source >= 0) & (target >= 0) & (source < pages * page) & (target < pages * page)
    for w in want:
        w[target[real]] = w[source[real]].clone()
    hip.paged_move(suffix, source.cuda(), target.cuda(), *caches, weights=weights, positions=positions)
    for w, got in zip(want, caches + [weights, positions]):
        assert torch.equal(got.cpu().reshape(w.shape), w)
    hip.paged_move(suffix, source[:0].cuda(), target[:0].cuda(), *caches)


@pytest.mark.parametrize("suffix,kv_heads,dim,page,count", [("bf16", 8, 128, 16, 70_001), ("f16", 3, 80, 24, 280_007), ("bf16", 40, 128, 8, 14_003)])
def test_many_moves(hip, dev, suffix, kv_heads, dim, page, count):
    """Two moves a thread, and rows of less and of more than a workgroup's chunks."""
    log(f"{suffix} {kv_heads} heads of {dim}, pages of {page}, {count} moves")
    g = torch.Generator(device=dev).manual_seed(count)
    pages = -(-2 * count // page) + 2
    make = lambda: torch.randn(pages, page, kv_heads, dim, generator=g, device=dev).to(DTYPE[suffix])
    caches = [make(), make()]
    weights, positions = torch.randn(pages, page, generator=g, device=dev), torch.arange(pages * page, dtype=torch.int32, device=dev).view(pages, page)
    slots = torch.randperm(2 * count, generator=g, device=dev)
    source, target = slots[:count].clone(), slots[count:].clone()
    source[::5], target[3::7] = -1, -1
    source[11], target[12], source[-1], target[-3] = pages * page, 1 << 40, pages * page + 3, -7
    real = (source >= 0) & (target >= 0) & (source < pages * page) & (target < pages * page)
    want = [t.clone().flatten(0, 1) for t in caches + [weights, positions]]
    for w in want:
        w[target[real]] = w[source[real]].clone()
    hip.paged_move(suffix, source, target, *caches, weights=weights, positions=positions)
    for w, got in zip(want, caches + [weights, positions]):
        assert torch.equal(got.flatten(0, 1), w)


def test_graph(hip, dev):
    """Weights, plan and moves of a step in one graph, replayed with other queries."""
    lengths, page, keep = [200, 70, 129], 16, [100, 70, 64]
    q, keys, table, q_offsets, lse, old, after = check_weights(hip, "bf16", lengths, [1, 1, 1], 4, 2, 64, page)
    table_d, offsets_d, kv, want_kept = ints(table), ints(q_offsets), ints(lengths), ints(keep)
    kept, pages, counts = torch.empty(3, dtype=torch.int32, device=dev), torch.empty(40, dtype=torch.int32, device=dev), ints([0, 0])
    moves = [torch.empty(3, 100, dtype=torch.int64, device=dev) for _ in range(2)]
    values, start = keys.clone(), keys.clone()

    def step(stream=None):
        hip.attention_paged_weights("bf16", q, keys, table_d, offsets_d, kv, lse, after, weights_in=old, stream=stream)
        hip.page_release(kv, want_kept, page, table_d, kept, pages, counts, stream=stream)
        hip.evict_plan(after, None, table_d, kv, kept, *moves, stream=stream)
        hip.paged_move("bf16", *moves, keys, values, weights=after, stream=stream)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(turn)))
        results = []
        for run in (graph.replay, step):
            keys.copy_(start)
            values.copy_(start)
            run()
            torch.cuda.synchronize()
            results.append([t.clone() for t in (keys, values, after, kept, counts, *moves)])
        assert all(torch.equal(a, b) for a, b in zip(*results)), turn
    stream = torch.cuda.Stream()
    keys.copy_(start)
    values.copy_(start)
    stream.wait_stream(torch.cuda.current_stream())
    step(stream)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(results[0], (keys, values, after, kept, counts, *moves)))
