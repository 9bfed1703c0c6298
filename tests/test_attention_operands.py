"""Operands whose strides the attention calls must not misread, as the binding sees them (no GPU: the library's entry points
are replaced by a recorder, or refuse before any HIP call)."""
import types

import pytest
import torch

STREAM = types.SimpleNamespace(cuda_stream=None)


@pytest.fixture
def calls(hip, monkeypatch):
    """What reaches the library, as (name, arguments)."""
    made = []
    monkeypatch.setattr(hip, "call", lambda name, *args: made.append((name, args)))
    return made


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def paged(hip, table, requests=4):
    q, cache = torch.zeros(requests, 2, 64, dtype=torch.bfloat16), torch.zeros(9, 16, 2, 64, dtype=torch.bfloat16)
    hip.attention_paged("bf16", q, cache, cache, table, ints(requests + 1), ints(requests), torch.zeros_like(q),
                        temp=torch.zeros(1 << 20, dtype=torch.uint8), stream=STREAM)


def plan(hip, table, requests=4):
    hip.page_plan(ints(requests), ints(requests), 16, ints(5), table, ints(requests + 1), ints(requests), ints(8), ints(8),
                  torch.zeros(8, dtype=torch.int64), ints(2), stream=STREAM)


SHARED_TABLES = {
    "one row for all": lambda: ints(1, 8).expand(4, 8),
    "rows that overlap": lambda: ints(64).as_strided((4, 8), (2, 1)),
    "rows that overlap in one entry": lambda: ints(64).as_strided((4, 8), (7, 1)),
    "one entry for all": lambda: ints(1, 1).expand(4, 1),
}


@pytest.mark.parametrize("name", SHARED_TABLES)
@pytest.mark.parametrize("run", [paged, plan])
def test_block_tables_whose_rows_share_entries_are_refused(hip, calls, run, name):
    with pytest.raises(ValueError, match="block_table"):
        run(hip, SHARED_TABLES[name]())
    assert not calls


@pytest.mark.parametrize("table,requests,stride,width", [
    (lambda: ints(4, 8), 4, 8, 8), (lambda: ints(4, 20)[:, :8], 4, 20, 8), (lambda: ints(8, 8)[::2], 4, 16, 8),
    (lambda: ints(4, 1), 4, 1, 1), (lambda: ints(4, 9)[:, :1], 4, 9, 1), (lambda: ints(1, 8), 1, 8, 8),
    (lambda: ints(64).as_strided((1, 8), (2, 1)), 1, 8, 8), (lambda: ints(4, 0), 4, None, 0),
])
@pytest.mark.parametrize("run,first", [(paged, 6), (plan, 9)])
def test_block_tables_are_passed_as_they_are(hip, calls, run, first, table, requests, stride, width):
    run(hip, table(), requests)
    (_, args), = calls
    assert args[first + 1] == width and (stride is None or args[first] == stride) and args[first] >= width


# ---- the last axis ---------------------------------------------------------------------------------
def repeated(*shape, step=0):
    """One item for all of the last axis; `step` items apart otherwise (0: one item for everything)."""
    strides = [step * n for n in (shape[1] if len(shape) == 3 else 1, 1)] if step else [0, 0]
    if len(shape) == 4:
        strides = [0, *strides]
    return torch.zeros(4096, dtype=torch.bfloat16).as_strided(shape, (*strides, 0))


@pytest.mark.parametrize("step", [0, 8])
@pytest.mark.parametrize("name", ["q", "k", "v", "dout", "out"])
def test_rows_that_repeat_one_item_are_refused(hip, calls, name, step):
    """What `out.sum()` hands back as the gradient of `out` is one item expanded over every axis."""
    n, heads, dim = 4, 2, 64
    rows = {k: torch.zeros(n, heads, dim, dtype=torch.bfloat16) for k in ("q", "k", "v", "out", "dout")}
    rows[name] = repeated(n, heads, dim, step=step)
    offsets, lse, grads = torch.tensor([0, n], dtype=torch.int32), torch.zeros(heads, n), [torch.zeros(n, heads, dim, dtype=torch.bfloat16)
                                                                                          for _ in range(3)]
    temp = torch.zeros(1 << 16, dtype=torch.uint8)
    with pytest.raises(ValueError, match=name):
        hip.attention_packed_backward("bf16", rows["q"], rows["k"], rows["v"], rows["out"], lse, rows["dout"], offsets, offsets, *grads,
                                      temp=temp, stream=STREAM)
    if name != "dout":
        with pytest.raises(ValueError, match=name):
            hip.attention_packed("bf16", rows["q"], rows["k"], rows["v"], offsets, offsets, rows["out"], lse, temp=temp, stream=STREAM)
    assert not calls


def test_caches_and_new_rows_that_repeat_one_item_are_refused(hip, calls):
    x, cache = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(9, 16, 2, 64, dtype=torch.bfloat16)
    bad = repeated(9, 16, 2, 64)
    for keys, values in ((bad, cache), (cache, bad)):
        with pytest.raises(ValueError, match="cache"):
            hip.attention_paged("bf16", x, keys, values, ints(4, 8), ints(5), ints(4), torch.zeros_like(x),
                                temp=torch.zeros(1 << 20, dtype=torch.uint8), stream=STREAM)
    for key, value in ((repeated(4, 2, 64), x), (x, repeated(4, 2, 64))):
        with pytest.raises(ValueError, match="key|value"):
            hip.paged_write("bf16", key, value, torch.zeros(4, dtype=torch.int64), cache, cache.clone(), stream=STREAM)
    assert not calls


def test_rows_broadcast_over_tokens_and_heads_are_passed(hip, calls):
    """Strides of zero before the last axis are what they say, where nothing is written."""
    q, offsets = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    one = torch.zeros(64, dtype=torch.bfloat16).expand(4, 2, 64)
    hip.attention_packed("bf16", one, one, one, offsets, offsets, q, stream=STREAM)
    (_, args), = calls
    assert all((r.token_stride, r.head_stride) == (0, 0) for r in args[2:5]) and args[7].token_stride == 128


def test_rows_that_are_not_there_may_have_any_strides(hip, calls):
    q, offsets = torch.zeros(0, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 0], dtype=torch.int32)
    none = torch.zeros((), dtype=torch.bfloat16).expand(0, 2, 64)
    hip.attention_packed("bf16", none, none, none, offsets, offsets, q, stream=STREAM)
    assert len(calls) == 1


def test_table_rows_too_far_apart_for_the_library(hip, calls):
    """A row stride that the paged call's 32 bits do not hold is refused, not cut off; a plan takes it."""
    far = torch.empty_strided((4, 8), ((1 << 32) + 8, 1), dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="block_table"):
        paged(hip, far)
    assert not calls
    plan(hip, far)
    assert calls[0][1][9] == (1 << 32) + 8


# ---- lse -------------------------------------------------------------------------------------------
def with_lse(hip, which, lse, n, heads):
    x, offsets = torch.zeros(n, heads, 64, dtype=torch.bfloat16), torch.tensor([0, n], dtype=torch.int32)
    temp = torch.zeros(1 << 20, dtype=torch.uint8)
    if which == "packed":
        hip.attention_packed("bf16", x, x, x, offsets, offsets, x.clone(), lse, temp=temp, stream=STREAM)
    elif which == "backward":
        hip.attention_packed_backward("bf16", x, x, x, x, lse, x, offsets, offsets, x.clone(), x.clone(), x.clone(), temp=temp, stream=STREAM)
    else:
        cache = torch.zeros(9, 16, heads, 64, dtype=torch.bfloat16)
        hip.attention_paged("bf16", x, cache, cache, ints(1, 8), ints(2), ints(1), x.clone(), lse, temp=temp, stream=STREAM)


@pytest.mark.parametrize("which", ["packed", "backward", "paged"])
@pytest.mark.parametrize("n,heads,shape", [(6, 4, (6, 4)), (6, 4, (4, 7)), (6, 4, (2, 12)), (6, 1, (2, 3)), (6, 4, (1, 6, 4)),
                                           (6, 4, (6, 4, 1))])
def test_lse_with_its_axes_the_wrong_way_is_refused(hip, calls, which, n, heads, shape):
    """[heads, tokens] is what is filled: another shape of as many items would be read as something else."""
    with pytest.raises(ValueError, match="lse"):
        with_lse(hip, which, torch.zeros(shape), n, heads)
    assert not calls


@pytest.mark.parametrize("which", ["packed", "backward", "paged"])
@pytest.mark.parametrize("n,heads,shape", [(6, 4, (4, 6)), (6, 4, (24,)), (6, 4, (30,)), (6, 4, (24, 1)), (6, 4, (5, 6)), (6, 1, (6, 1)), (1, 4, (1, 4)), (1, 4, (4, 1)),
                                           (6, 4, (1, 4, 6)), (6, 4, (4, 6, 1)), (6, 4, (2, 2, 6)), (4, 4, (4, 4))])
def test_lse_of_any_shape_in_the_same_order_is_taken(hip, calls, which, n, heads, shape):
    with_lse(hip, which, torch.zeros(shape), n, heads)
    assert len(calls) == 1


def test_a_backward_call_without_lse_says_so(hip):
    """(The library's own refusal, before any HIP call.)"""
    r = hip.Rows(1 << 20, 64, 64)
    need = hip.attention_packed_backward_temp_bytes(1, 4, 4, 2, 1, 64)
    status = hip.lib().lcpp_hip_attention_packed_backward_f16(1 << 20, need, r, r, r, r, None, r, 1 << 20, 1 << 20, r, r, r, 1, 4, 4, 2, 1, 64,
                                                              0.125, 1, None)
    assert status == hip.ERR_INVALID_ARGUMENT
    assert "lse" in hip.lib().lcpp_hip_last_error().decode() and "aligned" not in hip.lib().lcpp_hip_last_error().decode()
