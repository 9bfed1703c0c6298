"""max_kv_length says how much temporary storage there is.  What is split, and so the order of sums and the time, goes by the
requests' own lengths: a captured graph and a wide block table state far more than a step's requests have."""
import pytest
import torch

import attention_oracle as oracle

pytestmark = pytest.mark.gpu

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


def batch(dtype, kv, new, heads, kv_heads, dim, page, width):
    g = torch.Generator(device="cuda").manual_seed(sum(kv))
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=g).to(dtype)
    used = [-(-n // page) for n in kv]
    pages = sum(used) + 2
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(kv), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(used):
        table[r, :n] = order[at:at + n]
        at += n
    return dict(q=randn(sum(new), heads, dim), key_cache=randn(pages, page, kv_heads, dim), value_cache=randn(pages, page, kv_heads, dim),
                block_table=table, q_offsets=oracle.offsets_of(new).cuda(), kv_lengths=torch.tensor(kv, dtype=torch.int32, device="cuda"))


def run(hip, suffix, s, stated, tree=None):
    out = torch.full_like(s["q"], 7.0)
    lse = torch.full((out.shape[1], out.shape[0]), 7.0, device="cuda")
    hip.attention_paged(suffix, **s, out=out, lse=lse, tree=tree, max_kv_length=stated)
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("suffix,kv,new,heads,kv_heads,dim", [
    ("bf16", [8000], [1], 32, 8, 128),
    ("f16", [2777, 1, 900], [1, 1, 1], 2, 1, 64),
    ("bf16", [300, 5000, 0, 1200], [1, 1, 1, 1], 16, 4, 80),
    ("f16", [4000, 700], [40, 9], 8, 2, 128),       # wide tiles
    ("bf16", [3000], [500], 4, 1, 64),              # a chunk of a prompt
    ("bf16", [1 + 37 * i % 900 for i in range(150)], [1] * 150, 2, 2, 64),  # more requests than lanes
])
def test_the_same_bits_whatever_is_stated(hip, dev, suffix, kv, new, heads, kv_heads, dim):
    """The same parts make the same sums.  (They are joined one after another where the statement allows for up to 16, in 16 groups
    where it allows for more: it is 17 parts of 256 keys or more here.)"""
    s = batch(DTYPE[suffix], kv, new, heads, kv_heads, dim, 16, 1 << 14)
    least = max(max(kv), 17 * 256)
    want = run(hip, suffix, s, least)
    for stated in (least + 1, 2 * least, 131_072, None, 1 << 22):  # None: what the table holds, 2^18
        got = run(hip, suffix, s, stated)
        for name, a, b in zip(("out", "lse"), got, want):
            assert torch.equal(a, b), f"{name} with {stated} stated"


def test_trees_whatever_is_stated(hip, dev):
    kv, new = [6000, 800, 2500], [48, 5, 20]
    s = batch(torch.bfloat16, kv, new, 8, 2, 128, 32, 1 << 12)
    tree = torch.cat([(1 << torch.arange(1, n + 1)) - 1 for n in new]).cuda()
    want = run(hip, "bf16", s, max(kv), tree)
    for stated in (9000, 131_072):
        assert all(torch.equal(a, b) for a, b in zip(run(hip, "bf16", s, stated, tree), want))


def test_a_graph_recorded_for_long_requests_follows_short_ones(hip, dev):
    s = batch(torch.bfloat16, [30_000, 9000], [1, 1], 8, 2, 128, 16, 1 << 13)
    out, lse = torch.empty_like(s["q"]), torch.empty(8, 2, device="cuda")
    temp = torch.empty(hip.attention_paged_temp_bytes(2, 2, 131_072, 8, 2, 128), dtype=torch.uint8, device="cuda")
    step = lambda: hip.attention_paged("bf16", **s, out=out, lse=lse, max_kv_length=131_072, temp=temp)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for kv in ([30_000, 9000], [700, 9000], [1, 2], [0, 5000]):
        s["kv_lengths"].copy_(torch.tensor(kv, dtype=torch.int32))
        want, want_lse = run(hip, "bf16", s, max(kv))
        out.fill_(7.0)
        lse.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse), kv
