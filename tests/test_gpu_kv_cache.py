"""GPU: the paged key-value cache, bit for bit against the row quantisers of the oracle."""
import numpy as np
import pytest
import torch

from oracle import normquant as onq
from oracle.formats import e4m3_decode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    from inspark_proper_format_b200 import kv_cache
    return kv_cache


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def quantise(x, fmt):
    """(codes, scales, values) of FP32 rows x [..., D] by the definition; numpy."""
    if fmt == "e4m3":
        shape = x.shape
        codes, scales = onq.quant_e4m3_row(x.reshape(-1, shape[-1]))
        codes, scales = codes.reshape(shape), scales.reshape(shape[:-1])
        return codes, scales, e4m3_decode(codes) * scales[..., None]
    scales = np.maximum(np.abs(x).max(-1) / np.float32(127), np.float32(1e-12)).astype(np.float32)
    codes = np.clip(np.rint((x / scales[..., None]).astype(np.float32)), -127, 127).astype(np.int8)
    return codes, scales, codes.astype(np.float32) * scales[..., None]


def layout(totals, page, seed, extra=2):
    """Random page table and pool size for sequences of these lengths."""
    need = [(n + page - 1) // page for n in totals]
    g = np.random.default_rng(seed)
    ids = g.permutation(sum(need) + extra)
    width = max(1, max(need)) + 1
    table = np.full((len(totals), width), -1, np.int32)          # unused entries are no pages
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return torch.from_numpy(table).cuda(), sum(need) + extra


def positions(totals, new):
    return [(b, t - n + i) for b, (t, n) in enumerate(zip(totals, new)) for i in range(n)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "bf16", "f16"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,dim,page,new,past", [
    (1, 64, 1, [1], [0]),
    (20, 64, 64, [256, 1, 63], [0, 64, 1]),
    (3, 128, 48, [0, 95, 1, 200], [7, 1, 0, 333]),
    (8, 128, 16, [1, 1, 1, 1, 1], [0, 15, 16, 17, 500]),
    (65, 64, 7, [30, 2], [3, 0]),                              # more heads than rows per block
])
def test_append_and_gather_bit_exact(kv, fmt, dtype, heads, dim, page, new, past):
    totals = [a + b for a, b in zip(new, past)]
    table, pages = layout(totals, page, 3)
    cache = kv.PagedKVCache(pages, heads, dim, page_size=page, fmt=fmt)
    t = sum(new)
    g = torch.Generator().manual_seed(t + dim)
    k, v = (torch.randn(t, heads, dim, generator=g).mul_(3).to(dtype) for _ in range(2))
    k[0, 0] = 0                                               # an all-zero row: the smallest scale
    cu = _i32(np.concatenate([[0], np.cumsum(new)]))
    kv.kv_append(cache, k.cuda(), v.cuda(), table, _i32(totals), cu)
    table_np = table.cpu().numpy()
    where = positions(totals, new)
    ids = np.array([table_np[b, p // page] for b, p in where])
    off = np.array([p % page for _, p in where])
    for x, pool, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        raw = pool.view(torch.uint8 if pool.element_size() == 1 else torch.int16).cpu().numpy()
        if scale is None:
            want = x.to(pool.dtype).view(torch.int16).numpy()
            np.testing.assert_array_equal(raw[ids, :, off], want)
            written = np.zeros(raw.shape[:3], bool)
        else:
            codes, s, _ = quantise(x.float().numpy(), fmt)
            np.testing.assert_array_equal(raw[ids, :, off], codes.view(np.uint8))
            np.testing.assert_array_equal(scale.cpu().numpy()[ids, :, off], s)
        written = np.zeros((pages, page), bool)
        written[ids, off] = True
        assert not raw.transpose(0, 2, 1, 3)[~written].any(), "a row outside the tokens was written"
    for out_dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = kv.kv_gather(cache, table, _i32(totals), cu, tokens=t, dtype=out_dtype)
        for x, y in zip((k, v), got):
            values = (torch.from_numpy(quantise(x.float().numpy(), fmt)[2]) if fmt in ("e4m3", "int8")
                      else x.to(kv.FORMATS[fmt]).float())
            assert torch.equal(y.cpu(), values.to(out_dtype))


def test_strided_rows_of_a_fused_projection(kv):
    heads, dim, t = 4, 64, 37
    qkv = torch.randn(t, 3 * heads * dim, device="cuda").bfloat16()
    k, v = (qkv[:, i * heads * dim:(i + 1) * heads * dim].view(t, heads, dim) for i in (1, 2))
    table, pages = layout([t], 16, 1)
    a, b = (kv.PagedKVCache(pages, heads, dim, page_size=16, fmt="e4m3") for _ in range(2))
    lens, cu = _i32([t]), _i32([0, t])
    kv.kv_append(a, k, v, table, lens, cu)
    kv.kv_append(b, k.contiguous(), v.contiguous(), table, lens, cu)
    # heads outermost, an unaligned base and a broadcast head are taken as well
    c = kv.PagedKVCache(pages, heads, dim, page_size=16, fmt="e4m3")
    odd = torch.empty(t * heads * dim + 1, device="cuda", dtype=torch.bfloat16)[1:].view(t, heads, dim).copy_(v)
    kv.kv_append(c, k.transpose(0, 1).contiguous().transpose(0, 1), odd, table, lens, cu)
    for x in (b, c):
        assert torch.equal(a.k.view(torch.uint8), x.k.view(torch.uint8))
        assert torch.equal(a.v.view(torch.uint8), x.v.view(torch.uint8))
        assert torch.equal(a.k_scale, x.k_scale) and torch.equal(a.v_scale, x.v_scale)
    one = k[:, :1].expand(t, heads, dim)
    kv.kv_append(a, one, one, table, lens, cu)
    got, _ = kv.kv_gather(a, table, lens, cu, tokens=t, dtype=torch.float32)
    assert torch.equal(got, got[:, :1].expand_as(got))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_rows_with_non_finite_elements_read_back_as_nan(kv, fmt):
    x = torch.randn(6, 2, 64, device="cuda")
    x[1, 0, 5], x[2, 1, 63], x[3, 0, 0] = float("nan"), float("inf"), float("-inf")
    table, pages = layout([6], 4, 1)
    cache = kv.PagedKVCache(pages, 2, 64, page_size=4, fmt=fmt)
    kv.kv_append(cache, x, x, table, _i32([6]), _i32([0, 6]))
    for y in kv.kv_gather(cache, table, _i32([6]), _i32([0, 6]), tokens=6, dtype=torch.float32):
        bad = torch.zeros(6, 2, dtype=torch.bool, device="cuda")
        bad[1, 0] = bad[2, 1] = bad[3, 0] = True
        assert torch.equal(y.isnan().all(-1), bad) and torch.equal(y.isnan().any(-1), bad)


def test_decode_form_inactive_sequences_and_untouched_neighbours(kv):
    table, pages = layout([5, 9, 3], 4, 2)
    cache = kv.PagedKVCache(pages, 2, 64, page_size=4, fmt="int8")
    k = torch.randn(3, 2, 64, device="cuda").bfloat16()
    kv.kv_append(cache, k, k, table, _i32([5, 0, 3]))            # sequence 1 has ended
    got, _ = kv.kv_gather(cache, table, _i32([5, 0, 3]), dtype=torch.float32)
    assert not got[1].any() and got[0].any() and got[2].any()
    assert int((cache.k != 0).any(-1).sum()) <= 4                # two tokens x two heads


def test_bad_indices_are_skipped_and_recorded(kv):
    from inspark_proper_format_b200 import _lib
    cache = kv.PagedKVCache(3, 1, 64, page_size=4, fmt="bf16")
    k = torch.ones(2, 1, 64, device="cuda").bfloat16()
    _lib.read_device_error(clear=True)
    kv.kv_append(cache, k, k, _i32([[3, 0], [-1, 0]]), _i32([1, 1]))        # page ids outside the pool
    assert _lib.read_device_error(clear=True) == _lib.ISP_ERR_ARG
    kv.kv_append(cache, k, k, _i32([[0, 1], [1, 2]]), _i32([9, 10 ** 9]))   # beyond the page table
    assert _lib.read_device_error(clear=True) == _lib.ISP_ERR_ARG
    assert not cache.k.any() and not cache.v.any()
    kv.kv_append(cache, k, k, _i32([[0, 1], [1, 2]]), _i32([8, 1]))
    assert _lib.read_device_error(clear=True) == 0
    assert cache.k[1, 0, 3].all() and cache.k[1, 0, 0].all()


def test_refusals(kv):
    cache = kv.PagedKVCache(4, 2, 64, page_size=4, fmt="e4m3")
    table, lens = _i32([[0], [1]]), _i32([1, 1])
    ok = torch.zeros(2, 2, 64, device="cuda").bfloat16()
    with pytest.raises(ValueError):
        kv.kv_append(cache, ok[:, :1], ok[:, :1], table, lens)
    with pytest.raises(ValueError):
        kv.kv_append(cache, ok.to(torch.float64), ok.to(torch.float64), table, lens)
    with pytest.raises(ValueError):
        kv.kv_append(cache, ok, ok, table.long(), lens)
    with pytest.raises(ValueError):
        kv.kv_append(cache, ok, ok, table, lens[:1])
    with pytest.raises(ValueError):
        kv.kv_append(cache, ok[:1], ok[:1], table, lens)
    with pytest.raises(ValueError):
        kv.kv_append(cache, ok.cpu(), ok.cpu(), table, lens)
    with pytest.raises(ValueError):
        kv.kv_gather(cache, table, lens, _i32([0, 1, 2]))
    with pytest.raises(ValueError):
        kv.kv_gather(cache, table, lens, dtype=torch.float64)
    with pytest.raises(ValueError):
        kv.PagedKVCache(4, 2, 96)
    with pytest.raises(ValueError):
        kv.PagedKVCache(4, 2, 64, fmt="fp4")
    with pytest.raises(ValueError):
        kv.PagedKVCache.from_tensors(cache.k, cache.v)
    with pytest.raises(ValueError):
        kv.PagedKVCache.from_tensors(cache.k[:, :, :, :32], cache.v[:, :, :, :32], cache.k_scale, cache.v_scale)


def test_empty_calls(kv):
    cache = kv.PagedKVCache(1, 1, 64)
    none = torch.zeros(0, 1, 64, device="cuda").bfloat16()
    table, lens = torch.zeros(0, 1, dtype=torch.int32, device="cuda"), _i32([])
    kv.kv_append(cache, none, none, table, lens)
    got = kv.kv_gather(cache, table, lens)
    assert got[0].shape == (0, 1, 64)
    kv.kv_append(cache, none, none, _i32([[0]]), _i32([0]), _i32([0, 0]))


def test_offsets_beyond_32_bits(kv):
    """A pool whose element offsets pass 2^32 (4.6 GB of codes): the last pages are written where they lie."""
    pages, heads, page = 2300, 8, 1024
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GB")
    size = (pages, heads, page, 128)
    pools = [torch.empty(size, device="cuda", dtype=torch.int8) for _ in range(2)]
    scales = [torch.empty(size[:3], device="cuda") for _ in range(2)]
    assert pools[0].numel() > 2 ** 31
    cache = kv.PagedKVCache.from_tensors(*pools, *scales)
    table, lens, cu = _i32([[0, pages - 1], [pages - 2, 1]]), _i32([page + 5, page]), _i32([0, 5, 9])
    k = torch.randn(9, heads, 128, device="cuda").bfloat16()
    kv.kv_append(cache, k, -k, table, lens, cu)
    a, b = kv.kv_gather(cache, table, lens, cu, tokens=9, dtype=torch.float32)
    codes, s, values = quantise(k.float().cpu().numpy(), "int8")
    np.testing.assert_array_equal(a.cpu().numpy(), values)
    np.testing.assert_array_equal(b.cpu().numpy(), -values)
    np.testing.assert_array_equal(cache.k[pages - 1, :, :5].cpu().numpy(), codes[:5].transpose(1, 0, 2))
