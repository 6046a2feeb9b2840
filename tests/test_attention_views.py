"""CPU: what the cache and attention wrappers hand to the C entry points for views of tensors (the
call itself is replaced, and host tensors stand in for device tensors)."""
import ctypes
import gc

import pytest
import torch

from inspark_proper_format_b200 import attention, kv_cache


class Device(torch.Tensor):
    """A host tensor that passes for a device tensor."""
    is_cuda = True


def device(t):
    return t.as_subclass(Device)


def i32(*v):
    return device(torch.tensor(v, dtype=torch.int32))


@pytest.fixture
def tables(monkeypatch):
    """The page tables that the calls would read, entry by entry, by the arguments they are given."""
    seen = []
    at = {"isp_kv_append": 9, "isp_kv_gather": 2, "isp_paged_decode": 5}

    def call(dev, name, *args):
        table, stride, width, _, batch = args[at[name]:at[name] + 5]
        holders = [t for t in gc.get_objects() if type(t) in (torch.Tensor, Device) and t.dtype == torch.int32]
        rows = []
        for b in range(batch):
            first, last = table + 4 * b * stride, table + 4 * (b * stride + width)
            inside = any(t.untyped_storage().data_ptr() <= first and
                         last <= t.untyped_storage().data_ptr() + t.untyped_storage().nbytes() for t in holders)
            assert inside, f"row {b} of the page table lies outside every tensor"
            rows.append(list((ctypes.c_int32 * width).from_address(first)))
        seen.append(rows)
    monkeypatch.setattr(kv_cache, "call", call)
    monkeypatch.setattr(attention, "call", call)
    return seen


def page_tables():
    base = torch.arange(64, dtype=torch.int32)
    yield "expanded", base[8:13][None].expand(3, 5)
    yield "overlapping", base[:20].as_strided((3, 5), (2, 1))
    yield "wide", base[:60].view(3, 20)[:, 2:7]
    yield "plain", base[:15].view(3, 5)
    yield "one column", base[:30].view(3, 10)[:, 4:5]
    yield "expanded column", base[3:4][None].expand(3, 1)


@pytest.mark.parametrize("name,table", list(page_tables()), ids=lambda v: v if isinstance(v, str) else "")
def test_page_tables_are_read_as_they_stand(tables, name, table):
    cache = kv_cache.PagedKVCache(70, 2, 64, page_size=4, fmt="bf16", device="cpu")
    x = device(torch.zeros(3, 2, 64, dtype=torch.bfloat16))
    lengths, cu = i32(1, 2, 3), i32(0, 1, 2, 3)

    class Workspace:
        buffer = torch.zeros(8)
    table = device(table)
    kv_cache.kv_append(cache, x, x, table, lengths, cu)
    kv_cache.kv_gather(cache, table, lengths, cu, tokens=3)
    attention.paged_decode_attention(x, cache, table, lengths, workspace=Workspace())
    assert tables == [table.tolist()] * 3
