"""Attention's refusals through the C-ABI and the binding, on a machine without a GPU: arguments are checked before any HIP
call."""
import ctypes as C
import pathlib
import subprocess
import types

import pytest
import torch

ALIGNED = 1 << 20  # a made-up device address: refused calls do not look at it


def rows(hip, data=ALIGNED, token=64, head=64):
    return hip.Rows(data, token, head)


def packed(hip, temp=None, temp_bytes=0, q=None, k=None, v=None, qo=ALIGNED, ko=ALIGNED, out=None, lse=None, sequences=1, tq=4,
           tk=4, heads=2, kv_heads=1, dim=64, scale=0.125):
    q, k, v, out = (rows(hip) if x is None else x for x in (q, k, v, out))
    return hip.lib().lcpp_hip_attention_packed_bf16(temp, temp_bytes, q, k, v, qo, ko, out, lse, sequences, tq, tk, heads,
                                                    kv_heads, dim, scale, 1, None)


def paged(hip, temp=None, temp_bytes=0, table=ALIGNED, stride=4, width=4, requests=1, tokens=1, max_kv=16, heads=2, kv_heads=1,
          dim=64, page=16, pages=9, scale=0.125, cache=None, lengths=ALIGNED):
    cache = hip.Pages(ALIGNED, 1024, 64, 64) if cache is None else cache
    return hip.lib().lcpp_hip_attention_paged_f16(temp, temp_bytes, rows(hip), cache, cache, table, stride, width, ALIGNED,
                                                  lengths, None, rows(hip), None, requests, tokens, max_kv, heads, kv_heads,
                                                  dim, page, pages, scale, None)


@pytest.mark.parametrize("change,word", [
    (dict(heads=3, kv_heads=2), "multiple"), (dict(heads=0), "multiple"), (dict(kv_heads=0), "multiple"),
    (dict(heads=70000), "65535"), (dict(tq=1 << 31), "too many"), (dict(tk=1 << 31), "too many"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(qo=None), "offsets"), (dict(ko=None), "offsets"),
])
def test_packed_refuses(hip, change, word):
    assert packed(hip, **change) == hip.ERR_INVALID_ARGUMENT
    assert word in hip.lib().lcpp_hip_last_error().decode()


@pytest.mark.parametrize("name", ["q", "k", "v", "out"])
def test_packed_refuses_rows(hip, name):
    for bad in (rows(hip, None), rows(hip, ALIGNED + 8), rows(hip, token=60), rows(hip, head=4), rows(hip, token=-64)):
        assert packed(hip, **{name: bad}) == hip.ERR_INVALID_ARGUMENT
        assert "aligned" in hip.lib().lcpp_hip_last_error().decode()


@pytest.mark.parametrize("dim", [0, 4, 60, 136, 256])
def test_head_sizes_that_are_not_built(hip, dim):
    assert packed(hip, dim=dim) == hip.ERR_UNSUPPORTED
    assert paged(hip, dim=dim) == hip.ERR_UNSUPPORTED
    assert "head size" in hip.lib().lcpp_hip_last_error().decode()


def test_backward_refuses(hip):
    r = rows(hip)
    call = lambda temp, size, lse=ALIGNED, dq=r, dk=r: hip.lib().lcpp_hip_attention_packed_backward_bf16(
        temp, size, r, r, r, r, lse, r, ALIGNED, ALIGNED, dq, dk, r, 1, 4, 4, 2, 1, 64, 0.125, 1, None)
    need = hip.attention_packed_backward_temp_bytes(1, 4, 4, 2, 1, 64)
    assert need >= 2 * 4 * 4
    assert call(ALIGNED, need - 1) == hip.ERR_TEMP_TOO_SMALL
    assert call(None, need) == hip.ERR_TEMP_TOO_SMALL
    assert call(ALIGNED, need, lse=None) == hip.ERR_INVALID_ARGUMENT
    assert call(ALIGNED, need, dq=rows(hip, None)) == hip.ERR_INVALID_ARGUMENT
    assert call(ALIGNED, need, dk=rows(hip, ALIGNED + 2)) == hip.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("change,word", [
    (dict(heads=3, kv_heads=2), "multiple"), (dict(page=0), "page"), (dict(page=1 << 31), "page"),
    (dict(pages=1 << 31), "page"), (dict(width=5), "width"), (dict(tokens=1 << 31), "too many"),
    (dict(tokens=1 << 30, heads=8), "too many"), (dict(max_kv=1 << 31), "too long"), (dict(scale=0.0), "scale"),
    (dict(table=None), "block table"), (dict(lengths=None), "lengths"),
])
def test_paged_refuses(hip, change, word):
    assert paged(hip, **change) == hip.ERR_INVALID_ARGUMENT
    assert word in hip.lib().lcpp_hip_last_error().decode()


def test_paged_refuses_caches_and_small_temp(hip):
    for bad in (hip.Pages(None, 1024, 64, 64), hip.Pages(ALIGNED + 4, 1024, 64, 64), hip.Pages(ALIGNED, 1020, 64, 64),
                hip.Pages(ALIGNED, 1024, 4, 64), hip.Pages(ALIGNED, 1024, 64, -8)):
        assert paged(hip, cache=bad) == hip.ERR_INVALID_ARGUMENT
    need = hip.attention_paged_temp_bytes(1, 1, 100_000, 2, 1, 64)
    assert need > 0
    assert paged(hip, ALIGNED, need - 1, max_kv=100_000) == hip.ERR_TEMP_TOO_SMALL
    assert paged(hip, None, need, max_kv=100_000) == hip.ERR_TEMP_TOO_SMALL


def test_plan_and_write_refuse(hip):
    lib = hip.lib()
    a = ALIGNED
    need = hip.page_plan_temp_bytes(3)

    def plan(temp=a, size=need, requests=3, page=16, stride=4, width=4, free=a, num_free=1, table=a, lengths=a, slots=a,
             tokens=5, offsets=a):
        return lib.lcpp_hip_page_plan(temp, size, lengths, a, requests, page, free, num_free, table, stride, width, offsets, a, a,
                                      a, slots, tokens, a, None)

    for change in (dict(page=0), dict(requests=1 << 31), dict(width=5), dict(free=None), dict(table=None), dict(lengths=None),
                   dict(slots=None), dict(offsets=None), dict(tokens=1 << 31)):
        assert plan(**change) == hip.ERR_INVALID_ARGUMENT, change
    if need:
        assert plan(size=need - 1) == hip.ERR_TEMP_TOO_SMALL
        assert plan(temp=None) == hip.ERR_TEMP_TOO_SMALL
    cache = hip.Pages(a, 1024, 64, 64)
    write = lambda key=None, slots=a, heads=1, dim=64, page=16, c=cache, tokens=3: lib.lcpp_hip_paged_write_bf16(
        key or rows(hip), rows(hip), slots, tokens, c, cache, heads, dim, page, 4, None)
    assert write(dim=60) == hip.ERR_UNSUPPORTED
    for change in (dict(heads=0), dict(page=0), dict(slots=None), dict(key=rows(hip, a + 2)), dict(tokens=1 << 31),
                   dict(c=hip.Pages(a, 1024, 63, 64))):
        assert write(**change) == hip.ERR_INVALID_ARGUMENT, change


def test_nothing_to_do_is_no_error(hip):
    lib = hip.lib()
    none = hip.Rows(None, 0, 0)
    assert packed(hip, sequences=0, tq=0, tk=0, qo=None, ko=None) == hip.OK
    assert packed(hip, tq=0, q=none, out=none) == hip.OK
    assert paged(hip, requests=0, tokens=0, table=None) == hip.OK
    assert lib.lcpp_hip_paged_write_f16(none, none, None, 0, hip.Pages(None, 0, 0, 0), hip.Pages(None, 0, 0, 0), 1, 64, 16, 0,
                                        None) == hip.OK


def test_binding_refuses(hip):
    """Shapes, types and orders that the binding can see."""
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    o = torch.tensor([0, 4], dtype=torch.int32)
    temp, stream = torch.zeros(64, dtype=torch.uint8), types.SimpleNamespace(cuda_stream=None)
    call = lambda q=x, k=x, v=x, qo=o, ko=o, out=x, lse=None: hip.attention_packed("bf16", q, k, v, qo, ko, out, lse, temp=temp,
                                                                                  stream=stream)
    for change in (dict(q=x.half()), dict(v=x[:3]), dict(out=x[:, :1]), dict(k=x.transpose(1, 2)), dict(qo=o.long()),
                   dict(ko=o[:1]), dict(lse=torch.zeros(7)), dict(lse=torch.zeros(8, dtype=torch.float64)),
                   dict(q=x.transpose(1, 2).contiguous().transpose(1, 2)), dict(out=x[:1].expand(4, 2, 64))):
        with pytest.raises(ValueError):
            call(**change)
    cache = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    table, kv = torch.zeros(1, 3, dtype=torch.int32), torch.tensor([4], dtype=torch.int32)
    go = lambda cache=cache, table=table, kv=kv, tree=None: hip.attention_paged("bf16", x, cache, cache, table, o, kv, x,
                                                                                 tree=tree, temp=temp, stream=stream)
    for change in (dict(cache=cache.half()), dict(cache=cache[..., :32]), dict(table=table.long()), dict(table=table[0]),
                   dict(kv=kv.long()), dict(tree=torch.zeros(4, dtype=torch.int32)),
                   dict(tree=torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(ValueError):
            go(**change)
    with pytest.raises(hip.LcppHipError):
        call(q=torch.zeros(4, 3, 64, dtype=torch.bfloat16), out=torch.zeros(4, 3, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        hip.paged_write("bf16", x, x[:2], torch.zeros(4, dtype=torch.int64), cache, cache, stream=stream)


def test_temp_bytes_hold_their_parts(hip):
    """Temp storage grows with what is split, never past a few times the outputs, and is nothing for batches that fill the
    device."""
    assert hip.attention_packed_backward_temp_bytes(1, 0, 10, 8, 8, 128) == 0
    assert hip.attention_paged_temp_bytes(4096, 4096, 8000, 8, 8, 128) == 0
    one = hip.attention_paged_temp_bytes(1, 1, 131_000, 32, 8, 128)
    assert 0 < one < 64 << 20
    assert isinstance(C.sizeof(hip.Rows), int) and C.sizeof(hip.Rows) == 24 and C.sizeof(hip.Pages) == 32


def test_calls_that_need_no_scratch_take_none(hip, monkeypatch):
    """No allocation where none is needed; the caller's storage is passed on as it is."""
    calls = []
    monkeypatch.setattr(hip, "call", lambda name, *args: calls.append(args))
    monkeypatch.setattr(hip, "stream_handle", lambda stream=None: None)
    q, o = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    hip.attention_packed("bf16", q, q, q, o, o, q.clone())
    assert calls[0][:2] == (None, 0)
    mine = torch.zeros(10, dtype=torch.uint8)
    hip.attention_packed("bf16", q, q, q, o, o, q.clone(), temp=mine)
    assert calls[1][:2] == (mine.data_ptr(), 10)


def test_cpp_module_builds_and_lists_its_cases():
    repo = pathlib.Path(__file__).resolve().parents[1]
    subprocess.run(["make", "-s", "-C", str(repo / "tests" / "cpp")], check=True)
    out = subprocess.run([str(repo / "tests" / "cpp" / "bin" / "attention_test"), "--list"], check=True, capture_output=True,
                         text=True).stdout.split()
    assert out == ["packed_forward", "plan_write_and_paged", "packed_gradients", "refusals"]
