"""A paged cache's plan, writes and attention, against a plain planner and plain 64-bit attention."""
import math
import random

import pytest
import torch

import attention_oracle as oracle
from gpu_util import log

pytestmark = pytest.mark.gpu

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---- plans ---------------------------------------------------------------------------------------
def run_plan(hip, cached, new, page, free, table, capacity):
    ints = lambda x, dtype=torch.int32: torch.tensor(x, dtype=dtype).cuda()
    width = len(table[0]) if table else 0
    s = {"table": ints(table).view(len(table), width), "offsets": torch.full((len(cached) + 1,), 77, dtype=torch.int32).cuda(),
         "kv": torch.full((len(cached),), 77, dtype=torch.int32).cuda()}
    for name in ("request", "position"):
        s[name] = torch.full((capacity,), 77, dtype=torch.int32).cuda()
    s["slot"] = torch.full((capacity,), 77, dtype=torch.int64).cuda()
    s["counts"] = torch.full((2,), 77, dtype=torch.int32).cuda()
    hip.page_plan(ints(cached), ints(new), page, ints(free), s["table"], s["offsets"], s["kv"], s["request"], s["position"],
                  s["slot"], s["counts"])
    torch.cuda.synchronize()
    return s


def check_plan(hip, cached, new, page, width, spare=10, extra=3, capacity=None):
    rng = random.Random(len(cached) * 31 + page)
    table = [[-5] * width for _ in cached]
    pages = list(range(sum(-(-(max(c, 0) + max(n, 0)) // page) for c, n in zip(cached, new)) + 50))
    rng.shuffle(pages)
    for row, c in zip(table, cached):
        for cell in range(min(width, -(-max(c, 0) // page))):
            row[cell] = pages.pop()
    need = sum(min(width, -(-(max(c, 0) + max(n, 0)) // page)) - min(width, -(-max(c, 0) // page)) for c, n in zip(cached, new))
    free = [pages.pop() for _ in range(max(0, need + spare))]
    capacity = sum(max(n, 0) for n in new) + extra if capacity is None else capacity
    got = run_plan(hip, cached, new, page, free, table, capacity)
    want = oracle.plan(cached, new, page, free, table, capacity)
    for name, value in want.items():
        assert got[name].cpu().tolist() == value, name


@pytest.mark.parametrize("page", [1, 2, 16, 24, 64])
def test_plan_small(hip, dev, page):
    check_plan(hip, [0, 5, 16, 17, 31, 32], [1, 1, 1, 1, 1, 1], page, 60)
    check_plan(hip, [0, 0, 7, 100, 3], [40, 0, 9, 1, 33], page, 200)
    check_plan(hip, [-3, 4, 0], [2, -9, 0], page, 8)
    check_plan(hip, [3], [5], page, 8)
    check_plan(hip, [0, 0], [0, 0], page, 2)


@pytest.mark.parametrize("requests", [63, 64, 65, 255, 256, 257, 1000, 1023, 1025, 2049, 4096, 4097, 5000, 5120, 5121, 9000, 11000])
def test_plan_request_counts(hip, dev, requests):
    rng = random.Random(requests)
    cached = [rng.choice([0, rng.randrange(40)]) for _ in range(requests)]
    new = [rng.choice([0, 1, 1, 1, rng.randrange(30)]) for _ in range(requests)]
    check_plan(hip, cached, new, 16, 6)


def test_plan_one_long_prompt(hip, dev):
    check_plan(hip, [0, 3000, 1], [20_000, 1, 4001], 16, 1300)


@pytest.mark.parametrize("low,high", [(0, 300), (1, 3), (2000, 3000)])
def test_plan_many_tokens(hip, dev, low, high):
    """More tokens than one a thread: threads take several, across requests, pages and the end of the buffers."""
    rng = random.Random(high)
    requests = 300_000 // (high // 2 + 1) + 1
    requests = min(requests, 8192)
    cached = [rng.randrange(60) for _ in range(requests)]
    new = [rng.randrange(low, high + 1) for _ in range(requests)]
    for page, extra in ((16, 0), (24, 3), (1, 300_000)):
        if page == 1 and high > 3:
            continue
        check_plan(hip, cached, new, page, -(-(60 + high) // page), extra=max(extra, 263_000 - sum(new)))


def test_plan_where_pages_run_out(hip, dev):
    """A free list that is too short, or empty, and rows that are too narrow: -1, and the rest as before."""
    check_plan(hip, [0, 5, 30], [40, 40, 40], 8, 20, spare=-6)
    check_plan(hip, [0, 5, 30], [40, 40, 40], 8, 20, spare=-100)
    check_plan(hip, [0, 5, 30, 100], [40, 40, 40, 4], 8, 4)
    check_plan(hip, [9], [9], 4, 0)


def test_plan_capacity_below_the_tokens(hip, dev):
    check_plan(hip, [0, 5, 30], [40, 40, 40], 8, 20, capacity=57)
    check_plan(hip, [0, 5, 30], [40, 40, 40], 8, 20, capacity=0)


def test_plan_no_requests(hip, dev):
    got = run_plan(hip, [], [], 8, [], [], 4)
    assert got["offsets"].tolist() == [0] and got["counts"].tolist() == [0, 0] and got["slot"].tolist() == [-1] * 4


def test_plan_slots_past_32_bits(hip, dev):
    page = 1 << 20
    got = run_plan(hip, [page - 1], [2], page, [40_000], [[30_000, -1]], 2)
    assert got["slot"].tolist() == [30_001 * page - 1, 40_000 * page]


def test_plan_again_and_in_a_graph(hip, dev):
    """The same lengths give the same plan again (the table's new entries are written, not appended to), and a recorded
    plan follows its inputs."""
    requests, page, width = 300, 16, 40
    ints = lambda n, dtype=torch.int32: torch.zeros(n, dtype=dtype, device="cuda")
    cached, new, free = ints(requests), ints(requests), torch.arange(9000, dtype=torch.int32, device="cuda")
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    outs = [ints(requests + 1), ints(requests), ints(4000), ints(4000), ints(4000, torch.int64), ints(2)]
    temp = torch.empty(max(16, hip.page_plan_temp_bytes(requests)), dtype=torch.uint8, device="cuda")
    step = lambda: hip.page_plan(cached, new, page, free, table, *outs, temp=temp)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        cached.copy_(torch.randint(0, 500, (requests,), generator=g))
        new.copy_(torch.randint(0, 14, (requests,), generator=g))
        table.fill_(3)
        step()
        want = [x.clone() for x in outs + [table]]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs + [table], want):
            assert torch.equal(a, b)


# ---- writes --------------------------------------------------------------------------------------
@pytest.mark.parametrize("suffix", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 1, 8, 1), (37, 3, 40, 16), (300, 8, 128, 24), (5000, 2, 64, 16)])
def test_write(hip, dev, suffix, tokens, heads, dim, page):
    g = torch.Generator().manual_seed(tokens)
    pages = -(-tokens // page) + 3
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[::7] = -1
    slots[3::11] = pages * page + 5  # past the cache
    key = torch.randn(tokens, heads, dim, generator=g).to(DTYPE[suffix])
    value = torch.randn(tokens, heads, dim, generator=g).to(DTYPE[suffix])
    caches = [torch.full((pages, page, heads, dim), 7.0, dtype=DTYPE[suffix]) for _ in range(2)]
    on_gpu = [c.cuda() for c in caches]
    hip.paged_write(suffix, key.cuda(), value.cuda(), slots.cuda(), *on_gpu)
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < pages * page:
            caches[0][slot // page, slot % page], caches[1][slot // page, slot % page] = key[t], value[t]
    torch.cuda.synchronize()
    for got, want in zip(on_gpu, caches):
        assert torch.equal(got.cpu(), want)


def test_write_strides(hip, dev):
    """Rows inside a fused projection, into caches with heads before tokens."""
    fused = torch.randn(20, 6, 64, dtype=torch.float16, device="cuda")
    key, value = fused[:, 2:4], fused[:, 4:]
    caches = [torch.zeros(5, 2, 8, 64, dtype=torch.float16, device="cuda").transpose(1, 2) for _ in range(2)]
    slots = torch.arange(39, -1, -2, device="cuda")
    hip.paged_write("f16", key, value, slots, *caches)
    torch.cuda.synchronize()
    for cache, x in zip(caches, (key, value)):
        flat = cache.reshape(40, 2, 64)
        assert torch.equal(flat[1::2].flip(0), x) and not flat[::2].any()


# ---- attention -----------------------------------------------------------------------------------
def make(suffix, kv, new, heads, kv_heads, dim, page, seed=1, tree=None, filled=math.nan, gain=1.5):
    """A cache whose unused places hold `filled`, and rows for the new tokens."""
    dtype, g = DTYPE[suffix], torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in kv]
    pages, width = sum(used) + 3, max(used + [1])
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(kv), width), -1, dtype=torch.int32)
    key_cache = torch.full((pages, page, kv_heads, dim), filled, dtype=dtype)
    value_cache = key_cache.clone()
    at = 0
    for r, n in enumerate(kv):
        table[r, :used[r]] = order[at:at + used[r]]
        at += used[r]
        for position in range(n):
            p = int(table[r, position // page])
            key_cache[p, position % page] = torch.randn(kv_heads, dim, generator=g).to(dtype)
            value_cache[p, position % page] = torch.randn(kv_heads, dim, generator=g).to(dtype)
    q = (torch.randn(sum(new), heads, dim, generator=g) * gain).to(dtype)
    words = None
    if tree == "random":
        rng, words = random.Random(seed), []
        for n in new:
            masks = []
            for i in range(n):
                parent = rng.randrange(-1, i)
                masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
            words += masks
    elif tree is not None:
        words = list(tree)
    if words is not None:
        words = torch.tensor([w - (1 << 64) if w >> 63 & 1 else w for w in words], dtype=torch.int64)
    return dict(q=q, key_cache=key_cache, value_cache=value_cache, table=table, q_offsets=oracle.offsets_of(new),
                kv=torch.tensor(kv, dtype=torch.int32), tree=words)


def run_paged(hip, suffix, s, max_kv=None, scale=None):
    d = {k: None if v is None else v.cuda() for k, v in s.items()}
    out = torch.full_like(d["q"], 7.0)
    lse = torch.full((out.shape[1], out.shape[0]), 7.0, device="cuda")
    hip.attention_paged(suffix, d["q"], d["key_cache"], d["value_cache"], d["table"], d["q_offsets"], d["kv"], out, lse,
                        tree=d["tree"], max_kv_length=max_kv, scale=scale)
    torch.cuda.synchronize()
    return out, lse


def compare(hip, suffix, kv, new, heads, kv_heads, dim, page, max_kv=None, **more):
    s = make(suffix, kv, new, heads, kv_heads, dim, page, **more)
    out, lse = run_paged(hip, suffix, s, max_kv)
    want = oracle.paged(s["q"], s["key_cache"], s["value_cache"], s["table"], s["q_offsets"], s["kv"], s["tree"], dim ** -0.5)
    oracle.check("lse", lse, want["lse"])
    oracle.check("out", out, want["out"])


@pytest.mark.parametrize("suffix", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 96, 120, 128])
def test_decode_head_sizes(hip, dev, suffix, dim):
    compare(hip, suffix, [70, 1, 33], [1, 1, 1], 4, 2, dim, 16)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (6, 2), (5, 1), (32, 2), (40, 1), (8, 8)])
def test_decode_head_layouts(hip, dev, heads, kv_heads):
    compare(hip, "bf16", [70, 131], [1, 1], heads, kv_heads, 128, 16)


@pytest.mark.parametrize("page", [1, 7, 8, 24, 64, 256])
def test_page_sizes(hip, dev, page):
    compare(hip, "bf16", [1, 31, 32, 33, 127, 129, 300], [1] * 7, 4, 2, 64, page)


@pytest.mark.parametrize("max_kv", [None, 1, 100, 5000, 200_000])
def test_parts(hip, dev, max_kv):
    """One request over one to many parts, joined; lengths past the stated maximum are right too."""
    compare(hip, "bf16", [2777, 1, 900], [1, 1, 1], 2, 1, 64, 16, max_kv=max_kv)
    compare(hip, "f16", [1025], [3], 4, 1, 128, 32, max_kv=max_kv)


@pytest.mark.parametrize("suffix", ["bf16", "f16"])
def test_trees(hip, dev, suffix):
    compare(hip, suffix, [5, 64, 65, 100, 400], [5, 64, 33, 48, 12], 4, 2, 128, 16, tree="random")
    compare(hip, suffix, [90, 700], [17, 64], 8, 1, 64, 24, tree="random", max_kv=3000)


def test_tree_words(hip, dev):
    """Rows that see nothing, everything, only the last; bits past the new tokens mean nothing."""
    words = [0, (1 << 64) - 1, 1 << 63, 1 << 2, 1, 6]
    compare(hip, "bf16", [3, 3], [3, 3], 2, 1, 64, 16, tree=words)       # no context: word 0 sees nothing
    compare(hip, "bf16", [50, 131], [3, 3], 2, 1, 64, 16, tree=words)


def test_chains(hip, dev):
    """Several new tokens without a tree: each sees the ones up to itself (also a whole prompt in pages)."""
    compare(hip, "bf16", [4, 200, 130], [4, 7, 130], 4, 2, 64, 16)
    compare(hip, "f16", [300], [300], 3, 3, 128, 24)
    compare(hip, "bf16", [500, 77], [1, 70], 16, 2, 128, 16)


def test_no_keys_and_no_rows(hip, dev):
    compare(hip, "bf16", [0, 5, 0, 9], [1, 0, 2, 1], 2, 2, 64, 16)
    compare(hip, "bf16", [2, 40], [5, 1], 2, 1, 64, 16)  # fewer keys than new tokens: the first rows see nothing


@pytest.mark.parametrize("requests", [65, 300])
def test_many_requests(hip, dev, requests):
    kv = [1 + (i * 13) % 40 for i in range(requests)]
    compare(hip, "bf16", kv, [1] * requests, 8, 2, 64, 16)


def test_pages_that_are_not_there(hip, dev):
    """Entries outside the cache hide their keys; lengths past the table end with it."""
    s = make("bf16", [100, 60], [1, 2], 2, 1, 64, 16, filled=math.nan)
    s["table"][0, 2], s["table"][0, 5], s["table"][1, 0] = -1, s["key_cache"].shape[0], -7
    s["kv"][0] = 5000
    s["table"] = s["table"][:, :6].contiguous()
    out, lse = run_paged(hip, "bf16", s)
    # 5000 counts as the table's 96: the new token is the last of those, in the page that is not there.
    want = oracle.paged(s["q"], s["key_cache"], s["value_cache"], s["table"], s["q_offsets"], s["kv"], None, 0.125)
    oracle.check("lse", lse, want["lse"])
    oracle.check("out", out, want["out"])


def test_cache_orders(hip, dev):
    """Heads before tokens inside a page, keys and values in one array, a table wider than its rows."""
    s = make("f16", [300, 41], [1, 1], 4, 2, 64, 16)
    want = oracle.paged(s["q"], s["key_cache"], s["value_cache"], s["table"], s["q_offsets"], s["kv"], None, 0.125)
    both = torch.stack([s["key_cache"], s["value_cache"]], 1).transpose(2, 3).contiguous().cuda()  # [P, 2, H, page, D]
    wide = torch.full((2, s["table"].shape[1] + 9), -1, dtype=torch.int32)
    wide[:, :s["table"].shape[1]] = s["table"]
    out = torch.empty(2, 4, 64, dtype=torch.float16, device="cuda")
    hip.attention_paged("f16", s["q"].cuda(), both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2),
                        wide.cuda()[:, :s["table"].shape[1]], s["q_offsets"].cuda(), s["kv"].cuda(), out)
    torch.cuda.synchronize()
    oracle.check("out", out, want["out"])


def test_cache_past_4_gib(hip, dev):
    """Pages whose bytes lie past 2^32: the same pages at the end of a large cache give the same bits."""
    s = make("bf16", [500], [1], 4, 2, 128, 16)
    near, _ = run_paged(hip, "bf16", s)
    pages = s["key_cache"].shape[0]
    large = (9 << 30) // (16 * 2 * 128 * 2)
    caches = []
    for name in ("key_cache", "value_cache"):
        c = torch.empty(large, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
        c[-pages:] = s[name].cuda()
        caches.append(c)
    table = torch.where(s["table"] >= 0, s["table"] + large - pages, -1)
    out = torch.empty_like(near)
    hip.attention_paged("bf16", s["q"].cuda(), *caches, table.cuda(), s["q_offsets"].cuda(), s["kv"].cuda(), out)
    torch.cuda.synchronize()
    assert torch.equal(out, near)
    key = torch.randn(2, 2, 128, device="cuda").to(torch.bfloat16)
    slots = torch.tensor([large * 16 - 1, (large - 2) * 16 + 3], device="cuda")
    hip.paged_write("bf16", key, key, slots, *caches)
    torch.cuda.synchronize()
    for c in caches:
        assert torch.equal(c[-1, 15], key[0]) and torch.equal(c[-2, 3], key[1])


def test_same_bits_again_on_another_stream_and_in_a_graph(hip, dev):
    s = make("bf16", [3000, 77], [4, 1], 8, 2, 128, 16)
    first, first_lse = run_paged(hip, "bf16", s)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again, again_lse = run_paged(hip, "bf16", s)
    side.synchronize()
    assert torch.equal(first, again) and torch.equal(first_lse, again_lse)
    d = {k: None if v is None else v.cuda() for k, v in s.items()}
    out = torch.empty_like(first)
    temp = torch.empty(max(16, hip.attention_paged_temp_bytes(2, 5, 3000, 8, 2, 128)), dtype=torch.uint8, device="cuda")
    step = lambda: hip.attention_paged("bf16", d["q"], d["key_cache"], d["value_cache"], d["table"], d["q_offsets"], d["kv"],
                                       out, max_kv_length=3000, temp=temp)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        d["q"].copy_(torch.randn(d["q"].shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16))
        d["kv"].copy_(torch.tensor([3000 - 900 * seed, 77 - 30 * seed], dtype=torch.int32))
        step()
        want = out.clone()
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("heads,max_kv", [(2, 400), (2, 9000), (16, 400)])
def test_infinities_and_nan_reach_the_rows_that_see_them(hip, dev, heads, max_kv):
    """A drafted token whose value is not finite: its siblings do not see it.  One row of parts, several, and wide tiles."""
    words = [1, 3, 5, 9, 0b10011]  # a root, three children, and a child of the first child
    s = make("bf16", [900, 305], [5, 5], heads, 1, 64, 16, tree=words * 2)
    want = oracle.paged(s["q"], s["key_cache"], s["value_cache"], s["table"], s["q_offsets"], s["kv"], s["tree"], 0.125)
    place = 305 - 5 + 2  # the second child of the second request
    page = int(s["table"][1, place // 16])
    for bad in (math.nan, math.inf):
        s["value_cache"][page, place % 16, 0, 7] = bad
        out, lse = run_paged(hip, "bf16", s, max_kv)
        sees = torch.zeros(10, dtype=torch.bool)
        sees[7] = True
        oracle.check("lse", lse, want["lse"])
        oracle.check("out", out.cpu()[~sees], (want["out"][0][~sees], want["out"][1][~sees]))
        mine = out.cpu()[sees].float()
        assert torch.isnan(mine[:, :, 7]).all() if math.isnan(bad) else (mine[:, :, 7] == bad).all()
        assert torch.isfinite(mine[:, :, :7]).all() and torch.isfinite(mine[:, :, 8:]).all()


@pytest.mark.parametrize("heads,tree", [(2, None), (16, None), (2, "random")])
def test_lengths_past_the_table(hip, dev, heads, tree):
    """New tokens keep their places where the table ends before their request does: the keys past it are not seen, those
    before are."""
    s = make("bf16", [100, 60, 90], [5, 20, 60], heads, 1, 64, 16, tree=tree)
    ends = s["table"].clone()
    ends[:, 4:] = -1
    want = oracle.paged(s["q"], s["key_cache"], s["value_cache"], ends, s["q_offsets"], s["kv"], s["tree"], 0.125)
    s["table"] = s["table"][:, :4].contiguous()
    out, lse = run_paged(hip, "bf16", s)
    oracle.check("lse", lse, want["lse"])
    oracle.check("out", out, want["out"])


@pytest.mark.parametrize("max_kv", [None, 9000])
def test_long_chunks(hip, dev, max_kv):
    """A part of a prompt over what came before it: tiles of rows that see some of the new keys, all or none."""
    compare(hip, "bf16", [700, 1300], [400, 150], 4, 1, 64, 16, max_kv=max_kv)
    compare(hip, "f16", [600], [290], 2, 2, 128, 24, max_kv=max_kv)


def test_scratch_belongs_to_the_stream_of_the_call(hip, dev):
    """Calls on a given stream, without temporary storage of the caller's, beside the current stream's own allocations."""
    s = make("bf16", [2777, 900], [1, 1], 4, 1, 64, 16)
    d = {k: None if v is None else v.cuda() for k, v in s.items()}
    want, want_lse = run_paged(hip, "bf16", s, 200_000)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    need = hip.attention_paged_temp_bytes(2, 2, 200_000, 4, 1, 64)
    assert need > 0
    for _ in range(5):
        out, lse = torch.full_like(want, 7.0), torch.full_like(want_lse, 7.0)
        side.wait_stream(torch.cuda.current_stream())
        hip.attention_paged("bf16", d["q"], d["key_cache"], d["value_cache"], d["table"], d["q_offsets"], d["kv"], out, lse,
                            max_kv_length=200_000, stream=side)
        busy = torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # would be the call's storage, if it were this stream's
        del busy
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
