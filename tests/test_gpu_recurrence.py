"""The gated recurrence and its gradients, against a plain 64-bit form that goes token by token."""
import math

import pytest
import torch

import long_request_oracle as oracle
from attention_oracle import offsets_of
from gpu_util import log

pytestmark = pytest.mark.gpu

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def made(seed, suffix, lengths, channels, span=200.0, gap=0):
    """x, log_decay, dout [tokens, channels] and states; `gap`: rows of a wider array."""
    g = torch.Generator().manual_seed(seed)
    tokens, dtype = sum(lengths), DTYPE[suffix]
    randn = lambda *s: torch.randn(*s, generator=g)
    remember = torch.exp(-math.log(span) * torch.rand(channels, generator=g))
    wide = lambda x: torch.nn.functional.pad(x.to(dtype), (0, gap)).cuda()[:, :channels]
    x, dout = wide(randn(tokens, channels)), wide(randn(tokens, channels))
    l = wide(-0.7 * remember * torch.exp(0.5 * randn(tokens, channels)))
    return x, l, dout, randn(len(lengths), channels).cuda(), randn(len(lengths), channels).cuda()


def run(hip, suffix, lengths, x, l, dout, initial=None, dfinal=None, temp=None):
    offsets = offsets_of(lengths).cuda()
    out, dx, dl = (torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda") for _ in range(3))
    final, dinitial = (torch.full((len(lengths), x.shape[1]), 7.0, device="cuda") for _ in range(2))
    hip.recurrence(suffix, x, l, offsets, out, initial=initial, final=final, temp=temp)
    hip.recurrence_backward(suffix, l, out, dout, offsets, dx, dl, initial=initial, dfinal=dfinal, dinitial=dinitial, temp=temp)
    torch.cuda.synchronize()
    return {"out": out, "final": final, "dx": dx, "dlog_decay": dl, "dinitial": dinitial}


def check(hip, suffix, lengths, channels, seed=1, states=True, **kind):
    log(f"{suffix} lengths {lengths[:12]} channels {channels}")
    x, l, dout, initial, dfinal = made(seed, suffix, lengths, channels, **kind)
    initial, dfinal = (initial, dfinal) if states else (None, None)
    got = run(hip, suffix, lengths, x, l, dout, initial, dfinal)
    want = oracle.recurrence(x, l, lengths, initial, dout, dfinal)
    for name, value in want.items():
        oracle.check(name, got[name], value)
    return got


@pytest.mark.parametrize("suffix", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("channels", [1, 2, 3, 7, 64, 65, 127, 130, 256, 258, 513, 1000])
def test_widths(hip, dev, suffix, channels):
    check(hip, suffix, [5, 0, 130, 1, 33], channels)


@pytest.mark.parametrize("suffix", ["bf16", "f32"])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1025, 2500])
def test_lengths(hip, dev, suffix, length):
    check(hip, suffix, [length], 72)
    check(hip, suffix, [length, 3, length], 36, states=False)


@pytest.mark.parametrize("suffix", ["bf16", "f16", "f32"])
def test_strides(hip, dev, suffix):
    for gap in (1, 2, 3, 4, 8, 100):
        check(hip, suffix, [40, 300], 68, gap=gap)
        check(hip, suffix, [40, 300], 33, gap=gap)


@pytest.mark.parametrize("suffix", ["bf16", "f32"])
def test_ragged(hip, dev, suffix):
    check(hip, suffix, [0, 0, 700, 0, 1, 1, 260, 128, 0, 256, 2, 0], 260, seed=4)
    check(hip, suffix, [1] * 300, 40, seed=5)
    check(hip, suffix, [3, 1, 4, 1, 5, 9, 2, 6] * 40, 24, seed=6)
    check(hip, suffix, [6000, 50, 50], 16, seed=7, span=3000.0)


@pytest.mark.parametrize("suffix", ["bf16", "f16", "f32"])
def test_steps_of_serving(hip, dev, suffix):
    """Around a token a sequence, where a sequence is walked: among them ones of none and of many."""
    for channels in (1, 33, 130, 260):
        check(hip, suffix, [1] * 70 + [60], channels, seed=3)
        check(hip, suffix, [0] * 200 + [240, 1, 0], channels, seed=4)
        check(hip, suffix, [1, 2, 0, 7, 8, 9, 16, 17, 1], channels, seed=5, gap=3)
        check(hip, suffix, [4] * 50 + [63] + [0, 25, 24], channels, seed=7, states=False)
    check(hip, suffix, [1] * 70 + [66], 64, seed=6)


def test_no_tokens_and_no_sequences(hip, dev):
    none = torch.empty(0, 12, dtype=torch.bfloat16, device=dev)
    states = torch.randn(3, 12, device=dev)
    final, dinitial = torch.zeros_like(states), torch.zeros_like(states)
    offsets = torch.zeros(4, dtype=torch.int32, device=dev)
    hip.recurrence("bf16", none, none, offsets, none, initial=states, final=final)
    hip.recurrence_backward("bf16", none, none, none, offsets, none, none, initial=states, dfinal=states, dinitial=dinitial)
    assert torch.equal(final, states) and torch.equal(dinitial, states)
    hip.recurrence("bf16", none, none, offsets, none, final=final)
    assert not bool(final.any())
    hip.recurrence("bf16", none, none, offsets[:1], none)


def test_rows_of_no_sequence_are_left(hip, dev):
    """Offsets that begin past the first row and end before the last."""
    x, l, dout, _, _ = made(3, "f32", [100], 20)
    offsets = torch.tensor([7, 40, 90], dtype=torch.int32).cuda()
    out, dx, dl = (torch.full_like(x, 5.0) for _ in range(3))
    hip.recurrence("f32", x, l, offsets, out)
    hip.recurrence_backward("f32", l, out, dout, offsets, dx, dl)
    want = oracle.recurrence(x[7:90], l[7:90], [33, 50], None, dout[7:90])
    for name, got in (("out", out), ("dx", dx), ("dlog_decay", dl)):
        oracle.check(name, got[7:90], want[name])
        assert bool((got[:7] == 5.0).all()) and bool((got[90:] == 5.0).all())


def test_state_rows(hip, dev):
    """Serving: a pool of states, kept in place; a request without a row starts from zero and is not kept."""
    lengths, channels = [1, 1, 40, 1, 0], 96
    x, l, _, _, _ = made(9, "bf16", lengths, channels)
    pool = torch.randn(8, channels, device=dev)
    before = pool.clone()
    rows = torch.tensor([5, 0, 7, -1, 2], dtype=torch.int32).cuda()
    out = torch.empty_like(x)
    hip.recurrence("bf16", x, l, offsets_of(lengths).cuda(), out, initial=pool, final=pool, rows=rows)
    first = before[rows.clamp_min(0).long()] * (rows >= 0)[:, None]
    want = oracle.recurrence(x, l, lengths, first)
    oracle.check("out", out, want["out"])
    for b, row in enumerate(rows.tolist()):
        if row >= 0:
            oracle.check("state", pool[row], (want["final"][0][b], want["final"][1][b]))
    for row in (1, 3, 4, 6):
        assert torch.equal(pool[row], before[row])
    rows[1] = 8  # past the pool: as -1
    again = torch.empty_like(x)
    hip.recurrence("bf16", x, l, offsets_of(lengths).cuda(), again, initial=before, rows=rows)
    first[1] = 0
    oracle.check("out", again, oracle.recurrence(x, l, lengths, first)["out"])


def test_token_by_token_is_the_scan(hip, dev):
    """A sequence fed one token a call, or in pieces, comes out as the whole one within both bounds."""
    length, channels = 300, 64
    x, l, _, _, _ = made(2, "f32", [length], channels)
    want = oracle.recurrence(x, l, [length])
    for pieces in ([1] * length, [128, 1, 2, 169], [299, 1]):
        state, at = torch.zeros(1, channels, device=dev), 0
        out = torch.empty_like(x)
        for n in pieces:
            hip.recurrence("f32", x[at:at + n], l[at:at + n], offsets_of([n]).cuda(), out[at:at + n], initial=state, final=state)
            at += n
        oracle.check("out", out, want["out"])
        oracle.check("final", state, want["final"])


def test_long_memories_that_decay_alike(hip, dev):
    """Roundings of either sign add up like a random walk, 2^-24 times the square root of the 10,000 tokens that a state remembers: 6e-6.
    One of the same sign in every token or chunk would be a hundred or ten times that."""
    tokens, channels = 20000, 64
    x = torch.randn(tokens, channels, generator=torch.Generator().manual_seed(1)).cuda()
    l = -torch.logspace(-4, -1, channels).cuda().expand(tokens, channels).contiguous()
    out, final = torch.empty_like(x), torch.empty(1, channels, device=dev)
    hip.recurrence("f32", x, l, offsets_of([tokens]).cuda(), out, final=final)
    state, decay = torch.zeros(channels, dtype=torch.float64, device=dev), l[0].double().exp()
    for row in x.double():
        state = decay * state + row
    assert float((final[0].double() - state).norm()) <= 6e-6 * float(state.norm())


def test_forgetting_and_growing(hip, dev):
    """-infinity forgets the state exactly; 0 keeps it; growth by a little is the formula's."""
    x, _, dout, initial, dfinal = made(5, "f32", [400, 70], 40)
    l = torch.full_like(x, -0.01)
    l[50], l[300], l[430] = -math.inf, -math.inf, -math.inf
    l[60:200] = 0.0
    l[200:260] = 0.02
    l[:, ::5] = -90.0
    l[:, 1::5] = -0.0625
    l[:, 2::5] = -0.0624
    got = run(hip, "f32", [400, 70], x, l, dout, initial, dfinal)
    want = oracle.recurrence(x, l, [400, 70], initial, dout, dfinal)
    for name, value in want.items():
        oracle.check(name, got[name], value)
    for t in (50, 300):
        forgot = l[t] == -math.inf  # channels 3 and 4 of five
        assert torch.equal(got["out"][t, forgot], x[t, forgot])


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_not_finite_stays_in_its_channel_and_sequence(hip, dev, bad):
    lengths, channels = [300, 300, 40], 130
    x, l, dout, initial, dfinal = made(6, "bf16", lengths, channels)
    clean = run(hip, "bf16", lengths, x, l, dout, initial, dfinal)
    x[310, 17] = bad
    dout[450, 90] = bad
    got = run(hip, "bf16", lengths, x, l, dout, initial, dfinal)
    for name in got:
        broken = ~got[name].isfinite()
        if name in ("out", "dx", "dlog_decay"):
            channel, first, last = {"out": (17, 310, 600), "dx": (90, 300, 451), "dlog_decay": (17, 311, 600)}[name]
            assert bool(broken[first:last, channel].all()), name
        allowed = torch.zeros_like(broken)
        if broken.shape[0] == 3:
            allowed[1, [17, 90]] = True
        else:
            allowed[300:600, [17, 90]] = True
        assert not bool((broken & ~allowed).any()), name
        assert torch.equal(got[name][~allowed], clean[name][~allowed]), name


@pytest.mark.parametrize("limit", [0, 1])
def test_chunks_that_are_not_waited_for(hip, dev, limit):
    """With no patience a workgroup makes what it needs of the chunks before its own itself: the same bits."""
    lengths = [3000, 10, 900]
    x, l, dout, initial, dfinal = made(7, "bf16", lengths, 300, span=2000.0)
    want = run(hip, "bf16", lengths, x, l, dout, initial, dfinal)
    before = hip.lib().lcpp_hip_get_lookback_spin_limit()
    try:
        hip.check(hip.lib().lcpp_hip_set_lookback_spin_limit(limit))
        got = run(hip, "bf16", lengths, x, l, dout, initial, dfinal)
    finally:
        hip.check(hip.lib().lcpp_hip_set_lookback_spin_limit(before))
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_the_same_bits_again(hip, dev):
    lengths = [5000, 1, 2000, 4000]
    x, l, dout, initial, dfinal = made(8, "bf16", lengths, 600, span=2000.0)
    want = run(hip, "bf16", lengths, x, l, dout, initial, dfinal)
    for _ in range(4):
        got = run(hip, "bf16", lengths, x, l, dout, initial, dfinal)
        assert all(torch.equal(got[name], want[name]) for name in want)


def test_differences(hip, dev):
    """dx: the loss is linear in x, so a difference along a direction is the derivative.  dlog_decay: the central difference is
    off by a sixth of the step squared times the third derivative, for which the oracle's difference of the same step stands."""
    lengths, channels, step = [90, 200], 24, 2.0 ** -7
    x, l, dout, initial, dfinal = made(11, "f32", lengths, channels, span=30.0)
    got = run(hip, "f32", lengths, x, l, dout, initial, dfinal)
    v = torch.randn(x.shape, generator=torch.Generator().manual_seed(3)).cuda()

    def loss(x, l, initial):
        r = run(hip, "f32", lengths, x, l, dout, initial, dfinal)
        return float((r["out"].double() * dout).sum() + (r["final"].double() * dfinal).sum())

    def plain(x, l, initial):
        w = oracle.recurrence(x, l, lengths, initial)
        value = float((w["out"][0] * dout.cpu().double()).sum() + (w["final"][0] * dfinal.cpu().double()).sum())
        return value, float((w["out"][1] * dout.cpu().double().abs()).sum() + (w["final"][1] * dfinal.cpu().double().abs()).sum())

    for name, up, down, direction in (
            ("dx", (x + step * v, l, initial), (x - step * v, l, initial), (v, x + step * v, x - step * v)),
            ("dlog_decay", (x, l + step * v, initial), (x, l - step * v, initial), (v, l + step * v, l - step * v)),
            ("dinitial", (x, l, initial + 1.0), (x, l, initial - 1.0), (None, initial + 1.0, initial - 1.0))):
        moved = (direction[1].double() - direction[2].double()) / 2
        along = float((got[name].double() * moved).sum())
        a, b = plain(*up), plain(*down)
        measured, exact = (loss(*up) - loss(*down)) / 2, (a[0] - b[0]) / 2
        assert abs(measured - exact) <= (a[1] + b[1]) / 2, name
        want = oracle.recurrence(x, l, lengths, initial, dout, dfinal)[name]
        remainder = abs(exact - float((want[0] * moved.cpu()).sum()))
        size = float((want[0].abs() * moved.cpu().abs()).sum())
        assert remainder <= (1e-12 if name != "dlog_decay" else 0.02) * size, name
        assert abs(along - measured) <= float((want[1] * moved.cpu().abs()).sum()) + (a[1] + b[1]) / 2 + remainder, name


def test_graphs_and_streams(hip, dev):
    """Two graphs that share a workspace, replayed with other inputs between eager calls; and another stream."""
    lengths, channels = [600, 1, 300], 200
    offsets = offsets_of(lengths).cuda()
    x, l, dout, initial, dfinal = made(12, "bf16", lengths, channels)
    temp = torch.empty(max(16, hip.recurrence_temp_bytes(3, x.shape[0], channels)), dtype=torch.uint8, device=dev)
    run(hip, "bf16", lengths, x, l, dout, initial, dfinal, temp)
    out, dx, dl = (torch.empty_like(x) for _ in range(3))
    final, dinitial = torch.empty_like(initial), torch.empty_like(initial)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        hip.recurrence("bf16", x, l, offsets, out, initial=initial, final=final, temp=temp)
    with torch.cuda.graph(graphs[1]):
        hip.recurrence_backward("bf16", l, out, dout, offsets, dx, dl, initial=initial, dfinal=dfinal, dinitial=dinitial, temp=temp)
    for turn in range(3):
        fresh = made(30 + turn, "bf16", lengths, channels)
        x.copy_(fresh[0])
        l.copy_(fresh[1])
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        want = run(hip, "bf16", lengths, x, l, dout, initial, dfinal, temp)
        for name, got in (("out", out), ("final", final), ("dx", dx), ("dlog_decay", dl), ("dinitial", dinitial)):
            assert torch.equal(got, want[name]), (turn, name)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    other = torch.empty_like(x)
    hip.recurrence("bf16", x, l, offsets, other, initial=initial, stream=stream)
    stream.synchronize()
    assert torch.equal(other, want["out"])


@pytest.mark.parametrize("suffix", ["bf16", "f32"])
@pytest.mark.parametrize("lengths,channels", [([1], 40), ([40, 300], 33), ([700], 64)])
def test_rows_side_by_side_in_one_array(hip, dev, suffix, lengths, channels):
    """What is read and what is written as columns of one array: they share no item, and are not refused."""
    x, l, dout, initial, dfinal = made(14, suffix, lengths, channels)
    want = oracle.recurrence(x, l, lengths, initial, dout, dfinal)
    wide = torch.full((x.shape[0], 6 * channels + 1), 7.0, dtype=x.dtype, device=dev)
    columns = [wide[:, i * channels:(i + 1) * channels] for i in (4, 1, 5, 0, 3, 2)]
    for column, rows in zip(columns, (x, l, dout)):
        column.copy_(rows)
    out, dx, dl = columns[3:]
    offsets, final, dinitial = offsets_of(lengths).cuda(), torch.empty_like(initial), torch.empty_like(initial)
    hip.recurrence(suffix, columns[0], columns[1], offsets, out, initial=initial, final=final)
    hip.recurrence_backward(suffix, columns[1], out, columns[2], offsets, dx, dl, initial=initial, dfinal=dfinal, dinitial=dinitial)
    for name, got in (("out", out), ("final", final), ("dx", dx), ("dlog_decay", dl), ("dinitial", dinitial)):
        oracle.check(name, got, want[name])
    assert torch.equal(columns[0], x) and torch.equal(columns[1], l) and torch.equal(columns[2], dout) and bool((wide[:, -1] == 7.0).all())


@pytest.mark.parametrize("suffix", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lengths", [[3, 20, 1], [60, 50, 3], [700, 40], [2100]])  # walked, chunks of one wave, and of eight
def test_infinite_states_are_the_formula_s(hip, dev, suffix, lengths):
    """exp(l) times an infinity is one for every finite l: around 0, where exp(l) - 1 is taken, and far below, where a chunk's decay
    is 0 in 32 bits.  An infinity of the other sign makes NaN, and only what the formulas make infinite or NaN differs from the same
    call with finite items there."""
    dtype, tokens = DTYPE[suffix], sum(lengths)
    decays = [0.0, -2.0 ** -7, -0.0625, -0.5, -3.0, 2.0 ** -9]
    places = ["initial", "below", "x", "x, then the other", "dout", "dfinal", "none"]
    channels = len(decays) * len(places)
    x, l, dout, initial, dfinal = made(21, suffix, lengths, channels)
    l = torch.tensor(decays * len(places), dtype=dtype).cuda().expand(tokens, channels).contiguous()
    clean = run(hip, suffix, lengths, x, l, dout, initial, dfinal)
    begins = offsets_of(lengths).tolist()
    for i, place in enumerate(places):
        mine = slice(i * len(decays), (i + 1) * len(decays))
        for b, n in enumerate(lengths):
            if place in ("initial", "below"):
                initial[b, mine] = math.inf if place == "initial" else -math.inf
            if place.startswith("x"):
                x[begins[b] + n // 3, mine] = math.inf
            if place.endswith("other"):
                x[begins[b] + n // 3 + n // 2, mine] = -math.inf
            if place == "dout":
                dout[begins[b] + n // 2, mine] = -math.inf
            if place == "dfinal":
                dfinal[b, mine] = math.inf
    got = run(hip, suffix, lengths, x, l, dout, initial, dfinal)
    want = {name: value for name, (value, _) in oracle.recurrence(x, l, lengths, initial, dout, dfinal).items()}
    for name, value in want.items():
        mine = got[name].cpu().double()
        for what, a, b in (("NaN", mine.isnan(), value.isnan()), ("inf", mine == math.inf, value == math.inf),
                           ("-inf", mine == -math.inf, value == -math.inf)):
            assert torch.equal(a, b), f"{name}: {int((a != b).sum())} items are {what} or are not, in channels {(a != b).any(0).nonzero()[:, 0].tolist()}"
        finite = value.isfinite().cuda()
        assert torch.equal(got[name][finite], clean[name][finite]), name


def test_infinite_states_without_waiting(hip, dev):
    """As a workgroup makes them that reads its neighbours' rows itself."""
    before = hip.lib().lcpp_hip_get_lookback_spin_limit()
    try:
        hip.check(hip.lib().lcpp_hip_set_lookback_spin_limit(0))
        test_infinite_states_are_the_formula_s(hip, dev, "bf16", [2100])
    finally:
        hip.check(hip.lib().lcpp_hip_set_lookback_spin_limit(before))


# ---- large batches -------------------------------------------------------------------------------
def check_large(hip, lengths, sequences, channels, suffix="f32"):
    """Both directions of `sequences` of the lengths, which repeat, against 64 bits on the GPU, with the bounds of the oracle."""
    period, tokens = sum(lengths), sum(lengths) * (sequences // len(lengths))
    log(f"{suffix} {sequences} sequences {tokens} tokens {channels} channels")
    repeats, dtype, u, tiny = sequences // len(lengths), DTYPE[suffix], oracle.ROUNDOFF[DTYPE[suffix]], oracle.TINY[DTYPE[suffix]]
    g = torch.Generator(device="cuda").manual_seed(5)
    rows = lambda: torch.randn(tokens, channels, generator=g, device="cuda").to(dtype)
    states = lambda: torch.randn(sequences, channels, generator=g, device="cuda")
    x, dout, l = rows(), rows(), rows().abs_().mul_(-0.3)
    initial, dfinal = states(), states()
    count = torch.tensor([0] + lengths, device="cuda").cumsum(0)
    offsets = (torch.arange(repeats, device="cuda")[:, None] * period + count[:-1]).flatten()
    offsets = torch.cat([offsets, offsets.new_tensor([tokens])]).to(torch.int32)
    got = {name: torch.full_like(x, 7.0) for name in ("out", "dx", "dlog_decay")} | {n: torch.full_like(initial, 7.0) for n in ("final", "dinitial")}
    hip.recurrence(suffix, x, l, offsets, got["out"], initial=initial, final=got["final"])
    hip.recurrence_backward(suffix, l, got["out"], dout, offsets, got["dx"], got["dlog_decay"], initial=initial, dfinal=dfinal,
                            dinitial=got["dinitial"])
    torch.cuda.synchronize()

    def within(name, mine, value, bound):
        over = ((mine.double() - value).abs() - bound).nan_to_num(nan=math.inf).amax()
        assert float(over) <= 0, (name, float(over))

    token = lambda t, i: t.view(repeats, period, channels)[:, i].double()
    at = 0
    for b, n in enumerate(lengths):
        state = lambda t: t.view(repeats, len(lengths), channels)[:, b].double()
        h, size, e = state(initial), state(initial).abs(), torch.zeros(repeats, channels, dtype=torch.float64, device="cuda")
        before = []
        for i in range(at, at + n):
            before.append((h, e + u * h.abs() if i > at else e))
            li, xi = token(l, i), token(x, i)
            a = li.exp()
            e = a * e + oracle._step_error(li, a, size, xi)
            h, size = a * h + xi, a * size + xi.abs()
            within("out", token(got["out"], i), h, e + u * h.abs() + tiny)
        within("final", state(got["final"]), h, e + tiny)
        c, size, e = state(dfinal), state(dfinal).abs(), torch.zeros_like(e)
        for i in range(at + n - 1, at - 1, -1):
            li, d = token(l, i), token(dout, i)
            a = li.exp()
            gr, g_size, g_off = d + c, d.abs() + size, e + 2.0 ** -22 * (d.abs() + size)
            c, size, e = a * gr, a * g_size, a * g_off + oracle._step_error(li, a, g_size, torch.zeros_like(gr))
            h, h_off = before[i - at]
            within("dx", token(got["dx"], i), gr, g_off + u * gr.abs() + tiny)
            within("dlog_decay", token(got["dlog_decay"], i), c * h, u * (c * h).abs() * (1 + u) + (c.abs() + e) * (h_off + tiny) + e * h.abs() + tiny)
        within("dinitial", state(got["dinitial"]), c, e + tiny)
        at += n


# More workgroups of 64 channels than 2^31 threads of eight waves each are; those of one channel, more than one launch holds.
@pytest.mark.parametrize("name,lengths,sequences,channels,suffix", [
    ("walked, 4,096 channels", [1], 70_000, 4096, "bf16"),
    ("walked", [1], 34_000_000, 1, "bf16"),
    ("chunks of a wave, 4,096 channels", [1, 1, 1, 1, 1, 17, 2, 1], 60_000, 4096, "bf16"),
    ("chunks of a wave", [2] * 63 + [40], 64 * 453_200, 1, "f32"),
    ("chunks of eight waves", [130, 2, 66], 3 * 1_350_000, 1, "f32"),
])
def test_large_batches(hip, dev, name, lengths, sequences, channels, suffix):
    check_large(hip, lengths, sequences, channels, suffix)
    torch.cuda.empty_cache()
