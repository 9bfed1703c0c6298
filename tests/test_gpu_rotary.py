"""Rotary positions and the paged write that turns keys, against a plain 64-bit form."""
import math

import pytest
import torch

import long_request_oracle as oracle
from gpu_util import log

pytestmark = pytest.mark.gpu

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


def rows(seed, tokens, heads, dim, dtype, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(tokens, heads, dim, generator=g) * gain).to(dtype).cuda()


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).cuda()


def spread(tokens, most, seed=3):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, most, (tokens,), generator=g).to(torch.int32).cuda()


def check_turn(hip, suffix, tokens, heads, kv_heads, dim, rotary, interleaved, most=4096, factor=1.0, inverse=False, seed=1, gap=0):
    """`gap`: rows lie in a wider projection."""
    dtype = DTYPE[suffix]
    fused = rows(seed, tokens, heads + kv_heads + gap, dim, dtype)
    q, k = fused[:, :heads], fused[:, heads:heads + kv_heads]
    p, f = spread(tokens, most), hip.rotary_frequencies(rotary)
    q_out, k_out = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    hip.rotary(suffix, q, k, p, f, q_out, k_out, interleaved=interleaved, inverse=inverse, factor=factor)
    for name, got, x in (("q", q_out, q), ("k", k_out, k)):
        oracle.check(name, got, oracle.turn(x, p, f, interleaved, factor, inverse))
    return q_out, k_out


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 64), (64, 64), (80, 80), (96, 48), (8, 8), (8, 2), (32, 18), (120, 20), (256, 256),
                                        (128, 126), (1024, 1024), (1016, 1016), (80, 16), (112, 50)])
def test_head_layouts(hip, dev, dim, rotary, interleaved):
    log(f"dim {dim} rotary {rotary} interleaved {interleaved}")
    check_turn(hip, "bf16", 37, 6, 2, dim, rotary, interleaved)
    check_turn(hip, "f16", 5, 3, 1, dim, rotary, interleaved, inverse=True, factor=1.25)


@pytest.mark.parametrize("tokens", [1, 2, 63, 64, 65, 255, 257, 1000, 4099])
def test_token_counts(hip, dev, tokens):
    for heads, kv_heads, dim in ((8, 2, 64), (1, 1, 8), (5, 5, 128), (32, 8, 128)):
        check_turn(hip, "bf16", tokens, heads, kv_heads, dim, dim, False, gap=3)
    check_turn(hip, "f16", tokens, 7, 1, 80, 24, True, gap=1)


def test_many_rows(hip, dev):
    """Sizes of the kernel that takes four units a thread."""
    check_turn(hip, "bf16", 6007, 24, 8, 128, 128, False)
    check_turn(hip, "f16", 9001, 16, 4, 128, 64, True)
    check_turn(hip, "bf16", 30011, 8, 2, 64, 36, False)


@pytest.mark.parametrize("most", [1 << 17, 1 << 24, (1 << 31) - 1])
def test_far_positions(hip, dev, most):
    check_turn(hip, "f16", 300, 4, 4, 128, 128, False, most=most)
    check_turn(hip, "bf16", 300, 4, 4, 64, 64, True, most=most)


def test_negative_and_extreme_positions(hip, dev):
    p, f = ints([-1, -100000, 0, (1 << 31) - 1, -(1 << 31)]), hip.rotary_frequencies(64)
    q = rows(5, 5, 2, 64, torch.float16)
    out = torch.empty_like(q)
    hip.rotary("f16", q, None, p, f, out, None)
    oracle.check("q", out, oracle.turn(q, p, f, False))


@pytest.mark.parametrize("interleaved,rotary", [(False, 64), (True, 64), (False, 36), (False, 32)])
def test_in_place(hip, dev, interleaved, rotary):
    x = rows(8, 700, 5, 64, torch.bfloat16)
    q, k = x[:, :4], x[:, 4:]
    p, f = spread(700, 9000), hip.rotary_frequencies(rotary)
    want = [oracle.turn(t, p, f, interleaved) for t in (q, k)]
    hip.rotary("bf16", q, k, p, f, q, k, interleaved=interleaved)
    for got, w in zip((q, k), want):
        oracle.check("in place", got, w)


def test_the_gradient_is_the_inverse_turn(hip, dev):
    """Against the formula, and against differences: the turn is linear, so <dout, turn(v)> is the derivative along v."""
    tokens, dim, rotary = 50, 64, 48
    p, f = spread(tokens, 3000), hip.rotary_frequencies(rotary)
    dout = rows(11, tokens, 3, dim, torch.bfloat16)
    v = rows(12, tokens, 3, dim, torch.bfloat16)
    dx, turned = torch.empty_like(dout), torch.empty_like(v)
    hip.rotary("bf16", dout, None, p, f, dx, None, inverse=True, factor=0.75)
    hip.rotary("bf16", v, None, p, f, turned, None, factor=0.75)
    oracle.check("dx", dx, oracle.turn(dout, p, f, False, 0.75, True))
    left, right = (dout.double() * turned.double()).sum(), (dx.double() * v.double()).sum()
    # Each side is a sum of products of which one factor is rounded (2^-8 of it, and the turn's own 2^-19).
    slack = (2.0 ** -8 + 2.0 ** -19) * ((dout.double() * turned.double()).abs().sum() + (dx.double() * v.double()).abs().sum())
    assert abs(left - right) <= slack
    # An input that needs a gradient twice over (heads that share it): the caller sums; a turn of a turn back is the identity.
    back = torch.empty_like(v)
    hip.rotary("bf16", turned, None, p, f, back, None, inverse=True, factor=1 / 0.75)
    size = v.double().abs()
    pair = size.clone()
    pair[..., :24] += size[..., 24:48]
    pair[..., 24:48] += size[..., :24]
    pair[..., 48:] = size[..., 48:]
    # Two roundings, 2^-8 of a value that is at most 1 / 0.75 times 0.75 of the pair's sum each.
    assert bool(((back.double() - v.double()).abs()[..., :48] <= 2.0 ** -6.5 * pair[..., :48]).all())
    assert torch.equal(back[..., 48:], v[..., 48:])


def test_rows_of_no_request_are_left(hip, dev):
    tokens, f = 40, hip.rotary_frequencies(128)
    q, k = rows(1, tokens, 4, 128, torch.float16), rows(2, tokens, 2, 128, torch.float16)
    requests = [t // 5 if t % 7 else -1 for t in range(tokens)]
    shifts = [0, 100, -3, 7777, 1, 1 << 20]  # requests 6 and 7 have none
    p = spread(tokens, 500)
    q_out, k_out = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
    hip.rotary("f16", q, k, p, f, q_out, k_out, requests=ints(requests), shifts=ints(shifts))
    moved = p.cpu() + torch.tensor([shifts[r] if 0 <= r < len(shifts) else 0 for r in requests], dtype=torch.int32)
    real = torch.tensor([r >= 0 for r in requests])
    for got, x in ((q_out, q), (k_out, k)):
        oracle.check("rows", got[real.cuda()], oracle.turn(x.cpu()[real], moved[real], f, False))
        assert bool((got[~real.cuda()] == 9.0).all())


def test_no_rows(hip, dev):
    f, none = hip.rotary_frequencies(64), torch.empty(0, 4, 64, dtype=torch.bfloat16, device=dev)
    hip.rotary("bf16", none, none, ints([]), f, none, none)
    hip.rotary("bf16", none, None, ints([]), f, none, None)


def test_infinities_stay_in_their_pair(hip, dev):
    q = rows(1, 20, 2, 64, torch.bfloat16)
    q[3, 1, 5], q[7, 0, 40], q[9, 1, 63] = math.inf, math.nan, -math.inf
    p, f = spread(20, 100), hip.rotary_frequencies(64)
    for interleaved in (False, True):
        out = torch.empty_like(q)
        hip.rotary("bf16", q, None, p, f, out, None, interleaved=interleaved)
        partner = (lambda i: i ^ 1) if interleaved else (lambda i: (i + 32) % 64)
        touched = torch.zeros(20, 2, 64, dtype=torch.bool)
        for t, h, i in ((3, 1, 5), (7, 0, 40), (9, 1, 63)):
            touched[t, h, i] = touched[t, h, partner(i)] = True
        assert bool(out.cpu()[~touched].isfinite().all()) and not bool(out.cpu()[touched].isfinite().any())


@pytest.mark.parametrize("suffix,interleaved,rotary,page", [("bf16", False, 128, 16), ("f16", True, 64, 24), ("bf16", False, 36, 1), ("f16", False, 128, 64)])
@pytest.mark.parametrize("tokens", [1, 64, 333, 5000])
def test_paged_write(hip, dev, suffix, interleaved, rotary, page, tokens):
    dtype, heads, kv_heads, dim = DTYPE[suffix], 6, 2, 128
    fused = rows(tokens, tokens, heads + 2 * kv_heads, dim, dtype)
    q, key, value = fused[:, :heads], fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:]
    pages = -(-tokens // page) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(5))
    t = torch.arange(tokens)
    slots = order[t // page] * page + t % page
    slots[::11] = -1
    if tokens > 40:
        slots[13] = pages * page + 5  # past the last page
    requests = torch.where(t % 9 == 4, -1, t % 4).to(torch.int32)
    shifts, p = ints([0, 5, 100000, -2]), spread(tokens, 70000)
    f = hip.rotary_frequencies(rotary)
    q_out = torch.full((tokens, heads, dim), 3.0, dtype=dtype, device=dev)
    caches = [torch.full((kv_heads, pages, page, dim), 3.0, dtype=dtype, device=dev).permute(1, 2, 0, 3) for _ in range(2)]
    where = torch.full((pages, page), -7, dtype=torch.int32, device=dev)
    hip.paged_write_rotary(suffix, q, key, value, p, f, slots.cuda(), q_out, *caches, slot_positions=where,
                           requests=requests.cuda(), shifts=shifts, interleaved=interleaved, factor=1.5)
    moved = p.cpu() + shifts.cpu()[requests.clamp_min(0).long()]
    real = requests >= 0
    oracle.check("q", q_out.cpu()[real], oracle.turn(q.cpu()[real], moved[real], f, interleaved, 1.5))
    assert bool((q_out.cpu()[~real] == 3.0).all())
    put = real & (slots >= 0) & (slots < pages * page)
    flat = [c.cpu().reshape(pages * page, kv_heads, dim) for c in caches]
    oracle.check("keys", flat[0][slots[put]], oracle.turn(key.cpu()[put], moved[put], f, interleaved, 1.5))
    assert torch.equal(flat[1][slots[put]], value.cpu()[put])
    wanted = torch.full((pages * page,), -7, dtype=torch.int32)
    wanted[slots[put]] = moved[put]
    assert torch.equal(where.cpu().flatten(), wanted)
    free = torch.ones(pages * page, dtype=torch.bool)
    free[slots[put]] = False
    assert all(bool((c[free] == 3.0).all()) for c in flat)


@pytest.mark.parametrize("suffix,interleaved,rotary,page", [("bf16", False, 128, 16), ("f16", True, 64, 24), ("bf16", False, 36, 8)])
def test_many_rows_into_pages(hip, dev, suffix, interleaved, rotary, page):
    """Four units a thread."""
    test_paged_write(hip, dev, suffix, interleaved, rotary, page, 20011)


def test_the_write_is_rotary_and_paged_write(hip, dev):
    """Bit for bit, on a stream of its own, replayed from a graph with other inputs."""
    tokens, f = 70, hip.rotary_frequencies(64)
    q, k, v = (rows(s, tokens, h, 64, torch.bfloat16) for s, h in ((1, 4), (2, 2), (3, 2)))
    p, slots = spread(tokens, 1000), torch.randperm(96)[:tokens].cuda()
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    caches = [torch.zeros(6, 16, 2, 64, dtype=torch.bfloat16, device=dev) for _ in range(4)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = torch.empty_like(q)
    hip.paged_write_rotary("bf16", q, k, v, p, f, slots, got, caches[0], caches[1], stream=stream)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip.paged_write_rotary("bf16", q, k, v, p, f, slots, got, caches[0], caches[1])
    for turn in range(3):
        q.copy_(rows(20 + turn, tokens, 4, 64, torch.bfloat16))
        p.copy_(spread(tokens, 1000, seed=turn))
        graph.replay()
        torch.cuda.synchronize()
        hip.rotary("bf16", q, k, p, f, q_out, k_out)
        hip.paged_write("bf16", k_out, v, slots, caches[2], caches[3])
        torch.cuda.synchronize()
        assert torch.equal(got, q_out) and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
