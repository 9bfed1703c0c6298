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
