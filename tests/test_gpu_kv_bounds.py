"""GPU: cumulative counts outside a cache call's rows, and calls without sequences."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    from inspark_proper_format_b200 import kv_cache
    return kv_cache


@pytest.fixture
def errors():
    from inspark_proper_format_b200 import _lib
    _lib.read_device_error(clear=True)
    return lambda: _lib.read_device_error(clear=True)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("batch", [3, 1500])                    # bounds in shared memory, and searched where they lie
@pytest.mark.parametrize("cu,good", [
    ([0, 5, 100, 100], [0]),                                   # past the rows
    ([0, 5, 12, 100], [0, 1]),                                 # the same, in a sequence whose rows all exist but the last
    ([-3, 5, 12, 12], [1]),                                    # before them
    ([0, 12, 12, 30], [0]),                                    # past them, without a row of its own
])
def test_counts_outside_the_rows_are_skipped_and_recorded(kv, errors, cu, good, batch):
    """12 rows; the sequences whose bounds are inside 0..12 are served, the others' cached tokens stay as they are."""
    from inspark_proper_format_b200 import _lib
    t, page = 12, 16
    cu = cu + [cu[-1]] * (batch - 3)
    lengths = _i32([100, 101, 102] + [0] * (batch - 3))
    table = torch.arange(7 * 3, device="cuda", dtype=torch.int32).view(3, 7)
    table = torch.cat([table, torch.zeros(batch - 3, 7, device="cuda", dtype=torch.int32)])
    cache = kv.PagedKVCache(21, 1, 64, page_size=page, fmt="bf16")
    cache.k.fill_(7.0)
    cache.v.fill_(7.0)
    rows = torch.arange(1, t + 1, device="cuda").float()[:, None, None].expand(t, 1, 64).bfloat16()
    kv.kv_append(cache, rows, -rows, table, lengths, _i32(cu))
    assert errors() == _lib.ISP_ERR_ARG
    want = torch.full((21 * page,), 7.0, device="cuda")
    back = torch.zeros(t, device="cuda")
    for b in good:
        n = cu[b + 1] - cu[b]
        at = 7 * page * b + int(lengths[b]) - n
        back[cu[b]:cu[b + 1]] = want[at:at + n] = rows[cu[b]:cu[b + 1], 0, 0].float()
    assert torch.equal(cache.k[:, 0, :, 0].flatten().float(), want)
    k, v = kv.kv_gather(cache, table, lengths, _i32(cu), tokens=t)
    assert errors() == _lib.ISP_ERR_ARG
    assert torch.equal(k[:, 0, 0].float(), back) and torch.equal(v, -k)


def test_descending_counts_are_recorded(kv, errors):
    """No row goes to the sequence whose end lies before its start."""
    from inspark_proper_format_b200 import _lib
    cache = kv.PagedKVCache(4, 1, 64, page_size=16, fmt="bf16")
    rows = torch.ones(12, 1, 64, device="cuda").bfloat16()
    table, lengths, cu = _i32([[0], [1], [2]]), _i32([9, 9, 9]), _i32([0, 5, 3, 3])
    kv.kv_append(cache, rows, rows, table, lengths, cu)
    assert errors() == _lib.ISP_ERR_ARG and not cache.k[1:].any() and not cache.k[0, :, :4].any()


def test_counts_inside_the_rows_are_not_recorded(kv, errors):
    """Rows before the first and behind the last sequence belong to nobody."""
    cache = kv.PagedKVCache(4, 1, 64, page_size=16, fmt="bf16")
    rows = torch.ones(12, 1, 64, device="cuda").bfloat16()
    table, lengths, cu = _i32([[0], [1]]), _i32([4, 5]), _i32([2, 6, 9])
    kv.kv_append(cache, rows, rows, table, lengths, cu)
    k, _ = kv.kv_gather(cache, table, lengths, cu, tokens=12)
    assert errors() == 0
    assert k[:, 0, 0].tolist() == [0] * 2 + [1] * 7 + [0] * 3 and int(cache.k[:, 0, :, 0].sum()) == 4 + 3


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
def test_rows_of_a_call_without_sequences_are_zeros(kv, errors, fmt):
    """Nobody claims them: through the wrapper and the C entry, whose index arrays may be NULL then."""
    from inspark_proper_format_b200 import _lib
    cache = kv.PagedKVCache(2, 3, 64, page_size=16, fmt=fmt)
    table, none, cu = torch.zeros(0, 2, dtype=torch.int32, device="cuda"), _i32([]), _i32([0])
    rows = torch.ones(5, 3, 64, device="cuda").bfloat16()
    kv.kv_append(cache, rows, rows, table, none, cu)
    assert not cache.k.view(torch.uint8).any() and not cache.v.view(torch.uint8).any()
    for got in kv.kv_gather(cache, table, none, cu, tokens=5):
        assert got.shape == (5, 3, 64) and not got.any()
    k, v = rows.clone(), rows.clone()
    status = _lib.load().isp_kv_gather(ctypes.byref(cache._struct), cu.data_ptr(), None, 2, 2, None, 0, 5, _lib.BF16,
                                       k.data_ptr(), v.data_ptr(), _lib.stream_handle())
    assert status == _lib.ISP_OK and not k.any() and not v.any() and errors() == 0
