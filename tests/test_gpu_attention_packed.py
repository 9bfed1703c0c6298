"""Packed attention and its gradients against plain 64-bit attention, element by element within derived bounds."""
import math

import pytest
import torch

import attention_oracle as oracle
from gpu_util import log

pytestmark = pytest.mark.gpu

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


def rows(dtype, tokens, heads, dim, seed, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(tokens, heads, dim, generator=g) * gain).to(dtype)


def run(hip, suffix, q, k, v, q_offsets, k_offsets, causal, scale=None, dout=None):
    dev = lambda x: x.cuda()
    q, k, v, q_offsets, k_offsets = map(dev, (q, k, v, q_offsets, k_offsets))
    out, lse = torch.full_like(q, 7.0), torch.full((q.shape[1], q.shape[0]), 7.0, device="cuda")
    hip.attention_packed(suffix, q, k, v, q_offsets, k_offsets, out, lse, causal=causal, scale=scale)
    got = {"out": out, "lse": lse}
    if dout is not None:
        got |= {"dq": torch.full_like(q, 7.0), "dk": torch.full_like(k, 7.0), "dv": torch.full_like(v, 7.0)}
        hip.attention_packed_backward(suffix, q, k, v, out, lse, dout.cuda(), q_offsets, k_offsets, got["dq"], got["dk"],
                                      got["dv"], causal=causal, scale=scale)
    torch.cuda.synchronize()
    return got


def compare(hip, suffix, lengths, keys, heads, kv_heads, dim, causal, seed=1, gain=1.5, scale=None):
    dtype = DTYPE[suffix]
    q, k, v = (rows(dtype, sum(lengths), heads, dim, seed, gain), rows(dtype, sum(keys), kv_heads, dim, seed + 1),
               rows(dtype, sum(keys), kv_heads, dim, seed + 2))
    dout = rows(dtype, sum(lengths), heads, dim, seed + 3)
    q_offsets, k_offsets = oracle.offsets_of(lengths), oracle.offsets_of(keys)
    got = run(hip, suffix, q, k, v, q_offsets, k_offsets, causal, scale, dout)
    want = oracle.packed(q, k, v, q_offsets, k_offsets, causal, scale or dim ** -0.5, dout)
    for name in ("lse", "out", "dv", "dq", "dk"):
        oracle.check(name, got[name], want[name])


@pytest.mark.parametrize("suffix", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [8, 32, 40, 64, 72, 80, 96, 120, 128])
def test_head_sizes(hip, dev, suffix, dim):
    compare(hip, suffix, [67, 130], [67, 130], 2, 1, dim, True)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (6, 2), (5, 1), (16, 2), (7, 7)])
def test_head_layouts(hip, dev, heads, kv_heads):
    compare(hip, "bf16", [70, 33], [70, 33], heads, kv_heads, 64, True)
    compare(hip, "f16", [70, 33], [81, 12], heads, kv_heads, 128, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,keys", [
    ([1], [1]), ([1], [300]), ([300], [1]), ([31, 32, 33], [31, 32, 33]), ([63, 64, 65], [64, 65, 63]),
    ([127, 128, 129], [127, 128, 129]), ([255, 257], [257, 255]), ([5, 0, 7, 0], [5, 0, 7, 0]), ([0, 9, 4], [3, 0, 700]),
    ([40, 513], [200, 640]), ([200, 3], [40, 1]), ([1] * 70, [1] * 70), ([2, 1] * 40, [3, 9] * 40), ([0, 0, 1], [0, 0, 1]),
])
def test_lengths(hip, dev, causal, lengths, keys):
    compare(hip, "bf16", lengths, keys, 4, 2, 64, causal)
    compare(hip, "f16", lengths, keys, 2, 2, 128, causal)


def test_long_sequence(hip, dev):
    compare(hip, "bf16", [1500], [2100], 2, 1, 128, True)
    compare(hip, "f16", [2050], [2050], 1, 1, 64, True)


def test_many_sequences(hip, dev):
    """More sequences than lanes of a wave, and than its square, so that a tile's owner takes one to three steps to find."""
    for count in (65, 200, 4100):
        lengths = [(i * 7) % 5 for i in range(count)]
        compare(hip, "bf16", lengths, lengths, 1, 1, 32, True)


@pytest.mark.parametrize("gain,scale", [(40.0, None), (1.0, 1e-3), (0.0, None)])
def test_score_ranges(hip, dev, gain, scale):
    """Weights all on one key, all alike, and in between; the running maximum moves or stays."""
    compare(hip, "bf16", [200], [200], 2, 1, 64, True, gain=gain, scale=scale)


def test_rising_scores_move_the_maximum(hip, dev):
    """Every key outweighs the ones before it, by far and by a little."""
    for step in (0.05, 3.0):
        n, dim = 300, 64
        q = torch.zeros(n, 1, dim)
        q[:, :, 0] = 1.0
        k = torch.zeros(n, 1, dim)
        k[:, 0, 0] = torch.arange(n) * step
        q, k, v, dout = (x.to(torch.bfloat16) for x in (q, k, torch.randn(n, 1, dim), torch.randn(n, 1, dim)))
        o = oracle.offsets_of([n])
        got = run(hip, "bf16", q, k, v, o, o, True, 1.0, dout)
        want = oracle.packed(q, k, v, o, o, True, 1.0, dout)
        for name in want:
            oracle.check(name, got[name], want[name])


def test_strides(hip, dev):
    """Rows inside a fused projection, heads before tokens, and padded rows."""
    n, heads, kv_heads, dim = 150, 4, 2, 64
    fused = rows(torch.bfloat16, n, heads + 2 * kv_heads, dim, 5).cuda()
    q, k, v = fused[:, :heads], fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:]
    out = torch.full((heads, n, dim + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    view = out[:, :, :dim].transpose(0, 1)
    lse = torch.empty(heads, n, device="cuda")
    o = oracle.offsets_of([100, 50])
    hip.attention_packed("bf16", q, k, v, o.cuda(), o.cuda(), view, lse)
    dout = rows(torch.bfloat16, n, heads, dim, 6)
    grad = torch.full((n, heads + 2 * kv_heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    dq, dk, dv = grad[:, :heads], grad[:, heads:heads + kv_heads], grad[:, heads + kv_heads:]
    dout_heads = dout.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    hip.attention_packed_backward("bf16", q, k, v, view, lse, dout_heads, o.cuda(), o.cuda(), dq, dk, dv)
    want = oracle.packed(q.cpu(), k.cpu(), v.cpu(), o, o, True, dim ** -0.5, dout)
    for name, got in (("out", view), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        oracle.check(name, got, want[name])
    assert bool((out[:, :, dim:] == 7.0).all())


def test_rows_of_no_sequence_are_left_alone(hip, dev):
    """Rows before the first offset and after the last: not read (they hold NaN), not written."""
    n, dim = 100, 64
    make = lambda seed: rows(torch.bfloat16, n, 1, dim, seed)
    q, k, v, dout = (make(s) for s in range(4))
    for x in (q, k, v, dout):
        x[:9] = math.nan
        x[80:] = math.nan
    o = torch.tensor([9, 40, 80], dtype=torch.int32)
    got = run(hip, "bf16", q, k, v, o, o, True, None, dout)
    inner = torch.tensor([0, 31, 71], dtype=torch.int32)
    want = oracle.packed(*(x[9:80] for x in (q, k, v)), inner, inner, True, dim ** -0.5, dout[9:80])
    for name in ("out", "dq", "dk", "dv"):
        oracle.check(name, got[name][9:80], want[name])
        assert bool((got[name][:9] == 7.0).all()) and bool((got[name][80:] == 7.0).all())
    oracle.check("lse", got["lse"][:, 9:80], want["lse"])


def test_a_sequence_of_nan_stays_its_own(hip, dev):
    lengths, dim = [50, 20, 70], 64
    o = oracle.offsets_of(lengths)
    make = lambda seed, bad: torch.where(torch.tensor([[[False]]] * 50 + [[[True]]] * 20 + [[[False]]] * 70),
                                         torch.tensor(bad, dtype=torch.bfloat16), rows(torch.bfloat16, 140, 2, dim, seed))
    clean = [rows(torch.bfloat16, 140, 2, dim, s) for s in range(4)]
    want = oracle.packed(clean[0], clean[1], clean[2], o, o, True, dim ** -0.5, clean[3])
    for bad in (math.nan, math.inf):
        got = run(hip, "bf16", make(0, bad), make(1, bad), make(2, bad), o, o, True, None, make(3, bad))
        keep = torch.tensor([True] * 50 + [False] * 20 + [True] * 70)
        for name in ("out", "dq", "dk", "dv"):
            oracle.check(name, got[name].cpu()[keep], (want[name][0][keep], want[name][1][keep]))
            assert not torch.isfinite(got[name].cpu()[~keep].float()).all()


@pytest.mark.parametrize("suffix", ["bf16", "f16"])
def test_gradients_against_differences(hip, dev, suffix):
    """<gradient, direction> against the central difference of the 64-bit loss sum(dout * out) along the direction; what
    the rounded gradients may be off is their bounds along it."""
    dtype, lengths, keys, heads, kv_heads, dim = DTYPE[suffix], [45, 30], [50, 26], 4, 2, 40
    q, k, v = (rows(dtype, sum(lengths), heads, dim, 11), rows(dtype, sum(keys), kv_heads, dim, 12),
               rows(dtype, sum(keys), kv_heads, dim, 13))
    dout = rows(dtype, sum(lengths), heads, dim, 14)
    qo, ko, scale = oracle.offsets_of(lengths), oracle.offsets_of(keys), dim ** -0.5
    got = run(hip, suffix, q, k, v, qo, ko, True, None, dout)
    bounds = oracle.packed(q, k, v, qo, ko, True, scale, dout)

    def loss(q, k, v):
        total = 0.0
        for b in range(2):
            r, c = slice(int(qo[b]), int(qo[b + 1])), slice(int(ko[b]), int(ko[b + 1]))
            visible = torch.ones(lengths[b], keys[b], dtype=torch.bool).tril(keys[b] - lengths[b])
            for h in range(heads):
                o = oracle.head(q[r, h], k[c, h // 2], v[c, h // 2], visible, scale, dtype)[0]
                total += (o * dout[r, h].double()).sum()
        return float(total)

    base = [x.double() for x in (q, k, v)]
    for i, name in enumerate(("dq", "dk", "dv")):
        direction = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(20 + i), dtype=torch.float64)
        step, moved = 1e-4, [list(base), list(base)]
        moved[0][i], moved[1][i] = base[i] + step * direction, base[i] - step * direction
        slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
        along = float((got[name].cpu().double() * direction).sum())
        allowed = float((bounds[name][1] * direction.abs()).sum()) + 1e-5 * abs(slope) + 1e-6
        log(f"{name}: {along:.6f} along the direction, difference {slope:.6f}, allowed {allowed:.4f}")
        assert abs(along - slope) <= allowed


def test_same_bits_again_and_on_another_stream(hip, dev):
    dtype, lengths = torch.bfloat16, [333, 90]
    q, k, v, dout = (rows(dtype, 423, h, 128, s) for s, h in ((1, 8), (2, 2), (3, 2), (4, 8)))
    o = oracle.offsets_of(lengths)
    first = run(hip, "bf16", q, k, v, o, o, True, None, dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(hip, "bf16", q, k, v, o, o, True, None, dout)
    side.synchronize()
    for name in first:
        assert torch.equal(first[name], again[name]), name


def test_recorded_into_a_graph(hip, dev):
    """Forward and backward in one graph, replayed on fresh inputs with eager work in between."""
    lengths, dim = [130, 61], 64
    o = oracle.offsets_of(lengths).cuda()
    q, k, v, dout = (rows(torch.bfloat16, 191, h, dim, s).cuda() for s, h in ((1, 4), (2, 2), (3, 2), (4, 4)))
    out, lse = torch.empty_like(q), torch.empty(4, 191, device="cuda")
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    temp = torch.empty(max(16, hip.attention_packed_backward_temp_bytes(2, 191, 191, 4, 2, dim),
                           hip.attention_packed_temp_bytes(2, 191, 191, 4, 2, dim)), dtype=torch.uint8, device="cuda")

    def step():
        hip.attention_packed("bf16", q, k, v, o, o, out, lse, temp=temp)
        hip.attention_packed_backward("bf16", q, k, v, out, lse, dout, o, o, dq, dk, dv, temp=temp)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (50, 60, 70):
        for i, x in enumerate((q, k, v, dout)):
            x.copy_(rows(torch.bfloat16, 191, x.shape[1], dim, seed + i))
        step()
        want = [x.clone() for x in (out, lse, dq, dk, dv)]
        for x in (out, lse, dq, dk, dv):
            x.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip((out, lse, dq, dk, dv), want):
            assert torch.equal(got, w)


def test_no_lse_and_nothing_to_do(hip, dev):
    q = rows(torch.bfloat16, 5, 2, 64, 1).cuda()
    o = oracle.offsets_of([5]).cuda()
    out = torch.full_like(q, 7.0)
    hip.attention_packed("bf16", q, q, q, o, o, out)
    want = oracle.packed(q, q, q, o.cpu(), o.cpu(), True, 0.125)
    oracle.check("out", out, want["out"])
    empty = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    none = oracle.offsets_of([0]).cuda()
    hip.attention_packed("bf16", empty, empty, empty, none, none, empty)
    out.fill_(7.0)
    lse = torch.full((2, 5), 7.0, device="cuda")
    hip.attention_packed("bf16", q, empty, empty, o, none, out, lse)  # rows without keys
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    dk, dv = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    hip.attention_packed_backward("bf16", empty, q, q, empty, torch.empty(2, 0, device="cuda"), empty, none, o, empty, dk, dv)
    assert bool((dk == 0).all()) and bool((dv == 0).all())  # keys without rows


@pytest.mark.parametrize("suffix,dim", [("bf16", 64), ("f16", 128), ("bf16", 80)])
@pytest.mark.parametrize("where", [0, 37, 64, 127, 199])
def test_infinities_and_nan_reach_the_rows_that_see_them(hip, dev, suffix, dim, where):
    """A key or value that is not finite, inside a causal sequence: rows before it are as if it were zero, the others hold
    what the formula gives."""
    dtype, n = DTYPE[suffix], 200
    q, k, v = (rows(dtype, n, h, dim, s) for s, h in ((1, 4), (2, 2), (3, 2)))
    o = oracle.offsets_of([n])
    clean = [x.clone() for x in (k, v)]
    for x in clean:
        x[where] = 0
    want = oracle.packed(q, clean[0], clean[1], o, o, True, dim ** -0.5)
    before = torch.arange(n) < where
    for bad in (math.nan, math.inf, -math.inf):
        broken = v.clone()
        broken[where, 1, 5] = bad
        got = run(hip, suffix, q, k, broken, o, o, True)
        for name, axis in (("out", 0), ("lse", 1)):
            pick = lambda x: x.cpu().index_select(axis, before.nonzero()[:, 0])
            oracle.check(name, pick(got[name]), (pick(want[name][0]), pick(want[name][1])))
        after = got["out"].cpu()[~before].float()
        column = after[:, 2:, 5]
        assert torch.isnan(column).all() if math.isnan(bad) else (column == bad).all()
        after[:, 2:, 5] = 0
        assert torch.isfinite(after).all() and torch.isfinite(got["lse"]).all()
        broken = k.clone()
        broken[where, 0, 3] = math.nan
        got = run(hip, suffix, q, broken, v, o, o, True)
        oracle.check("out", got["out"].cpu()[before], (want["out"][0][before], want["out"][1][before]))
        assert torch.isnan(got["out"].cpu()[~before][:, :2].float()).all()
        assert torch.isfinite(got["out"].cpu()[:, 2:].float()).all()


@pytest.mark.parametrize("suffix,n,heads,kv_heads,dim", [("bf16", 200, 4, 2, 128), ("f16", 200, 4, 2, 64), ("bf16", 700, 8, 1, 80),
                                                         ("f16", 300, 3, 1, 128)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_gradients_pass_infinities_and_nan_along_what_is_seen(hip, dev, suffix, n, heads, kv_heads, dim, bad):
    """A row or key that is not finite inside a causal sequence: the gradients of what does not meet it are as if it were
    zero."""
    dtype, group = DTYPE[suffix], heads // kv_heads
    tensors = [rows(dtype, n, h, dim, s) for s, h in enumerate((heads, kv_heads, kv_heads, heads))]  # q, k, v, dout
    o, place = oracle.offsets_of([n]), torch.arange(n)
    for which, name in enumerate(("q", "k", "v", "dout")):
        log(name)
        of_keys = name in "kv"
        h = (kv_heads if of_keys else heads) - 1
        own = slice(h * group, heads) if of_keys else slice(h, heads)  # the query heads that meet it, and their key head
        for where in (0, 45, 64, n - 1):
            clean, broken = [x.clone() for x in tensors], [x.clone() for x in tensors]
            clean[which][where, h] = 0
            broken[which][where, h, 5] = bad
            want = oracle.packed(*clean[:3], o, o, True, dim ** -0.5, clean[3])
            got = run(hip, suffix, *broken[:3], o, o, True, None, broken[3])
            row_hit = place >= where if of_keys else place == where
            key_hit = torch.ones(n, dtype=torch.bool) if of_keys else place <= where
            for gradient in ("dq", "dk", "dv"):
                hit = torch.zeros(got[gradient].shape[:2], dtype=torch.bool)
                if gradient == "dq":
                    hit[:, own] = row_hit[:, None]
                elif not (gradient == "dv" and name == "v"):  # (dV does not depend on V)
                    hit[:, kv_heads - 1] = key_hit
                value = got[gradient].cpu()
                oracle.check(f"{gradient} of {name} at {where}", value[~hit], (want[gradient][0][~hit], want[gradient][1][~hit]))
                if hit.any() and math.isnan(bad):
                    assert not torch.isfinite(value[hit].float()).all(1).any()


def test_rows_that_see_nothing_pass_nothing(hip, dev):
    """Fewer keys than rows: what the first rows hold, NaN too, reaches no gradient."""
    n, m, dim = 100, 70, 128
    q, k, v, dout = (rows(torch.bfloat16, t, 2, dim, s) for s, t in enumerate((n, m, m, n)))
    qo, ko = oracle.offsets_of([n]), oracle.offsets_of([m])
    want = oracle.packed(q, k, v, qo, ko, True, dim ** -0.5, dout)
    q[:n - m], dout[:n - m] = math.nan, math.nan
    got = run(hip, "bf16", q, k, v, qo, ko, True, None, dout)
    for name in ("lse", "out", "dv", "dq", "dk"):
        oracle.check(name, got[name], want[name])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("sequences", [2, 63, 64, 65])
def test_batches_of_more_workgroups_than_run_at_once(hip, dev, causal, sequences):
    """Tiles are then taken in the order of their keys, up to 64 sequences: short and long ones, empty ones, keys with a head
    start, and fewer keys than rows."""
    lengths = [(37 * i * i) % 140 + (i % 5 == 0) * 150 for i in range(sequences)]
    lengths[1], lengths[-1] = 0, 300
    keys = [max(0, n + (-40, 0, 170)[i % 3]) for i, n in enumerate(lengths)]
    heads = 32 if sequences > 2 else 260
    assert sum(-(-n // 128) for n in lengths) * heads > 512
    compare(hip, "bf16", lengths, keys, heads, heads // 4, 32, causal)
