"""Refusals of rotary positions, eviction and the recurrence through the C-ABI and the binding, on a machine without a GPU:
arguments are checked before any HIP call."""
import types

import pytest
import torch

ALIGNED = 1 << 20  # a made-up device address: refused calls do not look at it


def message(hip):
    return hip.lib().lcpp_hip_last_error().decode()


def rows(hip, data=ALIGNED, token=64, head=64):
    return hip.Rows(data, token, head)


def pages(hip, data=ALIGNED, page=1024, token=64, head=64):
    return hip.Pages(data, page, token, head)


def steps(hip, data=ALIGNED, token=64):
    return hip.Steps(data, token)


def rotary(hip, q=None, k=None, positions=ALIGNED, requests=None, shifts=None, num_shifts=0, frequencies=ALIGNED, q_out=None, k_out=None,
           tokens=4, heads=2, kv_heads=1, dim=64, rotary_dim=64, factor=1.0):
    q, k, q_out, k_out = (rows(hip) if x is None else x for x in (q, k, q_out, k_out))
    return hip.lib().lcpp_hip_rotary_bf16(q, k, positions, requests, shifts, num_shifts, frequencies, q_out, k_out, tokens, heads, kv_heads,
                                          dim, rotary_dim, 0, 0, factor, None)


def write(hip, q=None, key=None, value=None, positions=ALIGNED, requests=None, shifts=None, frequencies=ALIGNED, slots=ALIGNED, q_out=None,
          key_cache=None, value_cache=None, tokens=4, heads=2, kv_heads=1, dim=64, rotary_dim=64, factor=1.0, page=16):
    q, key, value, q_out = (rows(hip) if x is None else x for x in (q, key, value, q_out))
    key_cache, value_cache = (pages(hip) if x is None else x for x in (key_cache, value_cache))
    return hip.lib().lcpp_hip_paged_write_rotary_f16(q, key, value, positions, requests, shifts, 0, frequencies, slots, q_out, key_cache,
                                                     value_cache, None, tokens, heads, kv_heads, dim, rotary_dim, 0, factor, page, 9, None)


@pytest.mark.parametrize("call", [rotary, write])
@pytest.mark.parametrize("change,word", [
    (dict(rotary_dim=0), "even"), (dict(rotary_dim=7), "even"), (dict(rotary_dim=66), "even"), (dict(heads=70000), "heads"),
    (dict(kv_heads=70000), "heads"), (dict(heads=0, kv_heads=0), "heads"), (dict(tokens=1 << 31), "too many"),
    (dict(factor=float("nan")), "factor"), (dict(factor=float("inf")), "factor"), (dict(positions=None), "null"),
    (dict(frequencies=None), "null"), (dict(shifts=ALIGNED), "requests"),
])
def test_turns_refuse(hip, call, change, word):
    assert call(hip, **change) == hip.ERR_INVALID_ARGUMENT
    assert word in message(hip)


@pytest.mark.parametrize("dim", [0, 4, 60, 1032])
def test_head_sizes_that_are_not_turned(hip, dim):
    assert rotary(hip, dim=dim, rotary_dim=2) == hip.ERR_UNSUPPORTED and write(hip, dim=dim, rotary_dim=2) == hip.ERR_UNSUPPORTED
    assert "head size" in message(hip)


def test_turns_refuse_rows(hip):
    for bad in (rows(hip, None), rows(hip, ALIGNED + 8), rows(hip, token=60), rows(hip, head=4), rows(hip, token=-64)):
        for name in ("q", "k", "q_out", "k_out"):
            assert rotary(hip, **{name: bad}) == hip.ERR_INVALID_ARGUMENT, name
        for name in ("q", "key", "value", "q_out"):
            assert write(hip, **{name: bad}) == hip.ERR_INVALID_ARGUMENT, name
    assert rotary(hip, q_out=rows(hip, token=128)) == hip.ERR_INVALID_ARGUMENT
    assert "in place" in message(hip)
    for bad in (pages(hip, None), pages(hip, ALIGNED + 2), pages(hip, page=1020), pages(hip, token=4)):
        assert write(hip, key_cache=bad) == hip.ERR_INVALID_ARGUMENT and write(hip, value_cache=bad) == hip.ERR_INVALID_ARGUMENT
    assert write(hip, page=0) == hip.ERR_INVALID_ARGUMENT and write(hip, slots=None) == hip.ERR_INVALID_ARGUMENT
    assert write(hip, kv_heads=0) == hip.ERR_INVALID_ARGUMENT


def weights(hip, q=None, cache=None, table=ALIGNED, stride=4, width=4, qo=ALIGNED, kv=ALIGNED, lse=ALIGNED, out=ALIGNED, requests=1, tokens=2,
            most=64, heads=2, kv_heads=1, dim=64, page=16, n_pages=9, scale=0.125, decay=1.0):
    return hip.lib().lcpp_hip_attention_paged_weights_bf16(
        None, 0, rows(hip) if q is None else q, pages(hip) if cache is None else cache, table, stride, width, qo, kv, None, None, lse, None,
        out, requests, tokens, most, heads, kv_heads, dim, page, n_pages, scale, decay, None)


@pytest.mark.parametrize("change,word", [
    (dict(heads=3, kv_heads=2), "multiple"), (dict(heads=0), "multiple"), (dict(kv_heads=0), "multiple"), (dict(page=0), "page"),
    (dict(n_pages=1 << 31), "page"), (dict(width=5), "width"), (dict(tokens=1 << 31), "too many"), (dict(requests=1 << 24), "too many"),
    (dict(most=1 << 31), "long"), (dict(width=1 << 20, stride=1 << 20, page=4096), "long"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(decay=-0.1), "decay"), (dict(decay=float("nan")), "decay"),
    (dict(decay=float("inf")), "decay"), (dict(qo=None), "null"), (dict(kv=None), "null"), (dict(out=None), "null"), (dict(table=None), "null"),
    (dict(lse=None), "lse"),
])
def test_weights_refuse(hip, change, word):
    assert weights(hip, **change) == hip.ERR_INVALID_ARGUMENT
    assert word in message(hip)


def test_weights_of_a_cache_without_pages(hip):
    # No slot is there to add to, so that nothing is launched: the arguments name no memory.
    assert weights(hip, n_pages=0) == hip.OK
    assert weights(hip, n_pages=0, tokens=0) == hip.OK
    assert weights(hip, n_pages=0, cache=pages(hip, None)) == hip.ERR_INVALID_ARGUMENT


def test_weights_refuse_temp_storage(hip):
    size = hip.attention_paged_weights_temp_bytes
    # Decoding steps, steps of a tile of rows in all, and full grids share no rows; few units of many rows do.
    assert size(256, 256, 4000, 32, 8, 128) == 0 and size(1, 4, 1 << 20, 32, 8, 128) == 0 and size(64, 4096, 8192, 32, 8, 128) == 0
    assert size(0, 0, 0, 32, 8, 128) == 0 and size(1, 0, 64, 2, 1, 64) == 0
    assert size(1, 4096, 8192, 32, 8, 128) > 0
    def call(temp, given):
        return hip.lib().lcpp_hip_attention_paged_weights_bf16(
            temp, given, rows(hip), pages(hip), ALIGNED, 4, 4, ALIGNED, ALIGNED, None, None, ALIGNED, None, ALIGNED, 1, 600, 64, 2, 1, 64, 16, 9,
            0.125, 1.0, None)
    needed = size(1, 600, 64, 2, 1, 64)
    assert needed > 0
    for temp, given, word in ((None, 0, "small"), (None, needed, "small"), (ALIGNED, needed - 1, "small")):
        assert call(temp, given) == hip.ERR_TEMP_TOO_SMALL and word in message(hip)
    assert call(ALIGNED + 2, needed) == hip.ERR_INVALID_ARGUMENT and "aligned" in message(hip)


def test_weights_refuse_rows_and_head_sizes(hip):
    for dim in (0, 4, 60, 136):
        assert weights(hip, dim=dim) == hip.ERR_UNSUPPORTED
    assert weights(hip, q=rows(hip, None)) == hip.ERR_INVALID_ARGUMENT and "aligned" in message(hip)
    assert weights(hip, cache=pages(hip, token=4)) == hip.ERR_INVALID_ARGUMENT and "aligned" in message(hip)


def release(hip, kv=ALIGNED, keep=ALIGNED, requests=2, page=16, table=ALIGNED, stride=4, width=4, kept=ALIGNED, out=ALIGNED, capacity=9,
            counts=ALIGNED):
    return hip.lib().lcpp_hip_page_release(kv, keep, requests, page, table, stride, width, 5, None, kept, None, out, capacity, counts, None)


@pytest.mark.parametrize("change,word", [
    (dict(kv=None), "lengths"), (dict(keep=None), "lengths"), (dict(kept=None), "lengths"), (dict(page=0), "page"), (dict(page=1 << 31), "page"),
    (dict(requests=1 << 28), "too many"), (dict(width=5), "width"), (dict(table=None), "table"), (dict(out=None), "list"),
    (dict(capacity=1 << 31), "too many"), (dict(counts=None), "counts"),
])
def test_release_refuses(hip, change, word):
    assert release(hip, **change) == hip.ERR_INVALID_ARGUMENT
    assert word in message(hip)


def plan(hip, weight=ALIGNED, positions=ALIGNED, table=ALIGNED, stride=4, width=4, kv=ALIGNED, kept=ALIGNED, requests=2, most=64, page=16,
         n_pages=9, first=0, recent=0, source=ALIGNED, target=ALIGNED, moves=8):
    return hip.lib().lcpp_hip_evict_plan(None, 0, weight, positions, table, stride, width, kv, kept, None, requests, most, page, n_pages, first,
                                         recent, source, target, moves, None)


@pytest.mark.parametrize("change,word", [
    (dict(weight=None), "null"), (dict(kv=None), "null"), (dict(kept=None), "null"), (dict(table=None), "null"), (dict(source=None), "moves"),
    (dict(target=None), "moves"), (dict(page=0), "page"), (dict(n_pages=1 << 31), "pages"), (dict(moves=1 << 31), "moves"),
    (dict(first=1 << 31), "protected"), (dict(recent=1 << 31), "protected"), (dict(positions=None, first=1), "positions"),
    (dict(positions=None, recent=1), "positions"), (dict(width=5), "width"), (dict(most=1 << 31), "long"),
    (dict(width=1 << 20, stride=1 << 20, page=4096), "long"), (dict(requests=1 << 28), "too many"),
])
def test_plan_refuses(hip, change, word):
    assert plan(hip, **change) == hip.ERR_INVALID_ARGUMENT
    assert word in message(hip)


def move(hip, source=ALIGNED, target=ALIGNED, moves=4, key=None, value=None, heads=2, dim=64, page=16):
    return hip.lib().lcpp_hip_paged_move_bf16(source, target, moves, pages(hip) if key is None else key, pages(hip) if value is None else value,
                                              None, None, heads, dim, page, 9, None)


def test_move_refuses(hip):
    for change, word in ((dict(source=None), "moves"), (dict(target=None), "moves"), (dict(moves=1 << 31), "moves"), (dict(heads=0), "heads"),
                         (dict(heads=70000), "heads"), (dict(page=0), "page"), (dict(key=pages(hip, None)), "aligned"),
                         (dict(value=pages(hip, token=4)), "aligned"), (dict(heads=65535, dim=65536), "long")):
        assert move(hip, **change) == hip.ERR_INVALID_ARGUMENT and word in message(hip), change
    for dim in (0, 4, 65544):
        assert move(hip, dim=dim) == hip.ERR_UNSUPPORTED


def forward(hip, x=None, l=None, out=None, offsets=ALIGNED, states=0, sequences=2, tokens=4, channels=64):
    x, l, out = (steps(hip) if t is None else t for t in (x, l, out))
    need = hip.recurrence_temp_bytes(min(sequences, 9), min(tokens, 9), min(channels, 64)) + 16
    return hip.lib().lcpp_hip_recurrence_bf16(ALIGNED, need, x, l, offsets, None, None, states, out, None, sequences, tokens, channels, None)


def backward(hip, l=None, out=None, dout=None, dx=None, dl=None, offsets=ALIGNED, sequences=2, tokens=4, channels=64):
    l, out, dout, dx, dl = (steps(hip) if t is None else t for t in (l, out, dout, dx, dl))
    need = hip.recurrence_temp_bytes(min(sequences, 9), min(tokens, 9), min(channels, 64)) + 16
    return hip.lib().lcpp_hip_recurrence_backward_bf16(ALIGNED, need, l, out, dout, offsets, None, None, dx, dl, None, sequences, tokens,
                                                       channels, None)


def test_recurrence_refuses(hip):
    for call in (forward, backward):
        for change, word in ((dict(channels=0), "channels"), (dict(channels=1 << 27), "channels"), (dict(tokens=1 << 31), "tokens"),
                             (dict(sequences=1 << 28), "sequences"), (dict(offsets=None), "offsets")):
            assert call(hip, **change) == hip.ERR_INVALID_ARGUMENT and word in message(hip), change
    assert forward(hip, states=1 << 31) == hip.ERR_INVALID_ARGUMENT
    for bad in (steps(hip, None), steps(hip, ALIGNED + 1), steps(hip, token=63), steps(hip, token=-64), steps(hip, token=1 << 41)):
        for name in ("x", "l", "out"):
            assert forward(hip, **{name: bad}) == hip.ERR_INVALID_ARGUMENT and "channels apart" in message(hip)
        for name in ("l", "out", "dout", "dx", "dl"):
            assert backward(hip, **{name: bad}) == hip.ERR_INVALID_ARGUMENT and "channels apart" in message(hip)


@pytest.mark.parametrize("tokens,channels,stride", [(4, 64, 64), (70, 64, 200), (1, 64, 64), (1000, 10, 24), (8, 1, 1)])
def test_recurrence_refuses_rows_written_over_what_is_read(hip, tokens, channels, stride):
    """A workgroup that does not wait for its neighbours reads their rows itself, which they may have written by then."""
    need, sequences = hip.recurrence_temp_bytes(2, tokens, channels), 2
    far = lambda i, shift=0, step=stride: hip.Steps(ALIGNED + (i << 24) + 2 * shift, step)

    def forward(x, l, out):
        return hip.lib().lcpp_hip_recurrence_bf16(ALIGNED, need, x, l, ALIGNED, None, None, 0, out, None, sequences, tokens, channels, None)

    def backward(l, out, dout, dx, dl):
        return hip.lib().lcpp_hip_recurrence_backward_bf16(ALIGNED, need, l, out, dout, ALIGNED, None, None, dx, dl, None, sequences, tokens,
                                                           channels, None)

    # The same rows; rows that begin in others; rows that others begin in; the last row that another's first one is.
    shifts = [0, channels - 1, 1 - channels, (tokens - 1) * stride, (1 - tokens) * stride]
    if tokens > 2:
        shifts += [stride + channels - 1, 2 * stride - channels + 1, (2 - tokens) * stride + 1 - channels]
    for shift in shifts:
        for call in (lambda: forward(far(1), far(2), far(1, shift)), lambda: forward(far(1), far(2), far(2, shift)),
                     *(lambda a=a, b=b: backward(*[far(b, shift) if i == a else far(i) for i in range(5)])
                       for a, b in ((3, 0), (3, 1), (3, 2), (4, 0), (4, 1), (4, 2), (3, 4)))):
            assert call() == hip.ERR_INVALID_ARGUMENT and "share no memory" in message(hip), shift
    # First rows that share items, other rows further apart.
    assert forward(far(1), far(2), far(1, 0, stride + 1)) == hip.ERR_INVALID_ARGUMENT and "share no memory" in message(hip)


def test_temporary_storage(hip):
    """Enough of it, and aligned to the words that it holds."""
    need = hip.recurrence_temp_bytes(2, 1000, 64)
    r = hip.Steps(ALIGNED, 64)
    call = lambda temp, size: hip.lib().lcpp_hip_recurrence_bf16(temp, size, r, r, ALIGNED, None, None, 0, r, None, 2, 1000, 64, None)
    back = lambda temp, size: hip.lib().lcpp_hip_recurrence_backward_bf16(temp, size, r, r, r, ALIGNED, None, None, r, r, None, 2, 1000, 64, None)
    for run in (call, back):
        assert need > 0 and run(ALIGNED, need - 1) == hip.ERR_TEMP_TOO_SMALL and run(None, need) == hip.ERR_TEMP_TOO_SMALL
        assert run(ALIGNED + 4, need) == hip.ERR_INVALID_ARGUMENT and "8-byte" in message(hip)
    need = hip.evict_plan_temp_bytes(2, 100000)
    run = lambda temp, size: hip.lib().lcpp_hip_evict_plan(temp, size, ALIGNED, None, ALIGNED, 4, 4, ALIGNED, ALIGNED, None, 2, 100000, 16, 9, 0,
                                                           0, ALIGNED, ALIGNED, 8, None)
    assert need > 0 and run(ALIGNED, need - 1) == hip.ERR_TEMP_TOO_SMALL and run(None, need) == hip.ERR_TEMP_TOO_SMALL
    assert run(ALIGNED + 8, need) == hip.ERR_INVALID_ARGUMENT and "16-byte" in message(hip)
    assert hip.recurrence_temp_bytes(0, 0, 64) == 0 and hip.recurrence_temp_bytes(256, 256, 4096) == 0
    assert hip.evict_plan_temp_bytes(0, 100000) == 0 and hip.evict_plan_temp_bytes(256, 1040) == 0


# ---- the binding ---------------------------------------------------------------------------------
@pytest.fixture
def never(hip, monkeypatch):
    """Calls that reach the library fail the test: what the binding has to refuse, it refuses by itself."""
    def reached(name, *args):
        raise AssertionError(f"{name} was reached")
    monkeypatch.setattr(hip, "call", reached)
    monkeypatch.setattr(hip, "stream_handle", lambda stream=None: None)
    return types.SimpleNamespace(
        bf=lambda *s: torch.zeros(*s, dtype=torch.bfloat16), i32=lambda *s: torch.zeros(*s, dtype=torch.int32),
        i64=lambda *s: torch.zeros(*s, dtype=torch.int64), f32=lambda *s: torch.zeros(*s), f64=lambda *s: torch.zeros(*s, dtype=torch.float64))


def test_binding_of_turns(hip, never):
    q, k, p, f = never.bf(4, 2, 64), never.bf(4, 1, 64), never.i32(4), never.f64(32)
    call = lambda q=q, k=k, p=p, f=f, q_out=q, k_out=k, **more: hip.rotary("bf16", q, k, p, f, q_out, k_out, **more)
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(k=k[:3]), dict(k=never.bf(4, 1, 32)), dict(p=p.long()), dict(p=p[:3]), dict(f=f.float()),
                dict(f=f[:0]), dict(q_out=never.bf(5, 2, 64)), dict(k_out=never.bf(4, 2, 64)), dict(q_out=never.bf(1, 2, 64).expand(4, 2, 64)),
                dict(q=never.bf(4, 2, 128)[..., ::2]), dict(requests=p[:2]), dict(requests=p.long()), dict(shifts=p), dict(requests=p, shifts=p.long())):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(AssertionError, match="reached"):
        call()
    cache, slots = never.bf(3, 16, 1, 64), never.i64(4)
    put = lambda key=k, value=k, slots=slots, kc=cache, vc=cache, **more: hip.paged_write_rotary("bf16", q, key, value, p, f, slots, q, kc, vc,
                                                                                               **more)
    for bad in (dict(key=k[:2]), dict(value=k.float()), dict(slots=slots.int()), dict(slots=slots[:2]), dict(kc=cache[0]), dict(vc=cache[:2]),
                dict(slot_positions=never.i32(3, 15)), dict(slot_positions=never.i64(3, 16)), dict(kc=cache[:, :1].expand(3, 16, 1, 64))):
        with pytest.raises(ValueError):
            put(**bad)


def test_binding_of_weights_and_eviction(hip, never):
    q, cache, table = never.bf(4, 2, 64), never.bf(3, 16, 1, 64), never.i32(2, 2)
    qo, kv, lse, sums = never.i32(3), never.i32(2), never.f32(2, 4), never.f32(3, 16)
    call = lambda q=q, cache=cache, table=table, qo=qo, lse=lse, out=sums, **more: hip.attention_paged_weights("bf16", q, cache, table, qo, kv,
                                                                                                            lse, out, **more)
    for bad in (dict(q=q.float()), dict(cache=never.bf(3, 16, 1, 32)), dict(table=table.long()), dict(table=table[:1]), dict(qo=qo[:2]),
                dict(lse=never.f32(4, 2)), dict(lse=lse.double()), dict(out=sums[:2]), dict(out=sums.double()), dict(weights_in=sums[:2]),
                dict(known_lengths=kv[:1]), dict(tree=never.i64(3)), dict(tree=never.i32(4)), dict(table=never.i32(1, 2).expand(2, 2))):
        with pytest.raises(ValueError):
            call(**bad)
    moves = never.i64(2, 5)
    plan = lambda weights=sums, positions=never.i32(3, 16), table=table, kept=kv, a=moves, b=moves, **more: hip.evict_plan(
        weights, positions, table, kv, kept, a, b, **more)
    for bad in (dict(weights=sums.flatten()), dict(weights=sums.double()), dict(positions=never.i32(3, 15)), dict(table=table[:1]),
                dict(kept=kv[:1]), dict(a=never.i64(2, 4)), dict(a=moves[0], b=moves[0]), dict(a=never.i64(3, 5), b=never.i64(3, 5)),
                dict(a=moves.int(), b=moves.int()), dict(shifts=kv[:1])):
        with pytest.raises(ValueError):
            plan(**bad)
    free = lambda keep=kv, kept=kv, released=never.i32(4), counts=never.i32(2), **more: hip.page_release(kv, keep, 16, table, kept, released,
                                                                                                       counts, **more)
    for bad in (dict(keep=kv[:1]), dict(kept=kv.long()), dict(released=never.i64(4)), dict(counts=never.i32(1)), dict(shifts=kv[:1]),
                dict(shifts_out=kv.long())):
        with pytest.raises(ValueError):
            free(**bad)
    shift = lambda a=moves, b=moves, kc=cache, vc=cache, **more: hip.paged_move("bf16", a, b, kc, vc, **more)
    for bad in (dict(a=moves[:1]), dict(a=moves.int()), dict(b=moves.t()), dict(kc=cache.float()), dict(vc=cache[:2]), dict(weights=sums[:2]),
                dict(positions=never.i64(3, 16))):
        with pytest.raises(ValueError):
            shift(**bad)


def test_binding_of_the_recurrence(hip, never):
    x, offsets, states = never.bf(6, 10), never.i32(3), never.f32(2, 10)
    call = lambda x=x, l=x, offsets=offsets, out=x, **more: hip.recurrence("bf16", x, l, offsets, out, **more)
    for bad in (dict(x=x.float()), dict(x=x[0]), dict(l=x[:5]), dict(out=never.bf(6, 9)), dict(offsets=offsets.long()),
                dict(l=never.bf(1, 10).expand(6, 10)), dict(l=never.bf(6, 1).expand(6, 10)), dict(x=never.bf(10, 6).t()), dict(initial=states[:1]),
                dict(initial=states.double()), dict(final=never.f32(2, 9)), dict(final=never.f32(2, 20)[:, ::2]),
                dict(initial=states, final=never.f32(3, 10)), dict(initial=states, rows=never.i32(1)), dict(initial=states, rows=never.i64(2))):
        with pytest.raises(ValueError):
            call(**bad)
    back = lambda l=x, out=x, dout=x, dx=x, dl=x, **more: hip.recurrence_backward("bf16", l, out, dout, offsets, dx, dl, **more)
    for bad in (dict(l=x.float()), dict(out=x[0]), dict(dout=x[:5]), dict(dx=never.bf(6, 9)), dict(dl=x.t()), dict(initial=states[:1]),
                dict(dfinal=states.double()), dict(dinitial=never.f32(2, 9))):
        with pytest.raises(ValueError):
            back(**bad)
    with pytest.raises(KeyError):
        hip.recurrence("i32", x, x, offsets, x)
