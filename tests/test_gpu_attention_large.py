"""GPU: attention over operands whose element offsets pass 2^32, and over thousands of sequences."""
import numpy as np
import pytest
import torch

from attention_f64 import U, attend, check
from test_gpu_attention import _cu, _i32, _randn, check_decode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def at():
    from inspark_proper_format_b200 import attention
    return attention


@pytest.fixture(scope="module")
def kv():
    from inspark_proper_format_b200 import kv_cache
    return kv_cache


@pytest.fixture(autouse=True)
def no_device_error():
    from inspark_proper_format_b200 import _lib
    _lib.read_device_error(clear=True)
    yield
    assert _lib.read_device_error(clear=True) == 0


def needs(gigabytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip(f"needs {gigabytes} GB")


@pytest.mark.parametrize("fmt", ["int8", "bf16"])
def test_cache_of_more_than_2_to_the_32_elements(at, kv, fmt):
    """Sequences in the first and the last pages of a pool of 4.4e9 elements: written, read back, attended."""
    needs(24)
    pages, heads, page, dim = 4200, 8, 1024, 128
    size = (pages, heads, page, dim)
    pools = [torch.empty(size, device="cuda", dtype=kv.FORMATS[fmt]) for _ in range(2)]
    scales = [torch.empty(size[:3], device="cuda") for _ in range(2)] if fmt == "int8" else []
    assert pools[0].numel() > 2 ** 32
    cache = kv.PagedKVCache.from_tensors(*pools, *scales)
    lens = [page + 500, 2 * page, 77]
    table = _i32([[0, pages - 1], [pages - 2, 1], [pages - 3, pages]])
    k = _randn(sum(lens), heads, dim, seed=200, dtype=torch.bfloat16)
    v = _randn(sum(lens), heads, dim, seed=201, dtype=torch.bfloat16)
    kv.kv_append(cache, k, v, table, _i32(lens), _cu(lens))
    back = kv.kv_gather(cache, table, _i32(lens), _cu(lens), tokens=sum(lens), dtype=torch.float32)
    if fmt == "bf16":
        assert torch.equal(back[0], k.float()) and torch.equal(back[1], v.float())
    else:                                                       # half a step of each row, and FP32's rounding of the product
        for x, y in zip((k, v), back):
            assert bool(((x.float() - y).abs() <= x.float().abs().amax(-1, keepdim=True) / 253.9).all())
    q = _randn(3, 2 * heads, dim, seed=202, dtype=torch.bfloat16)
    check_decode(at.paged_decode_attention(q, cache, table, _i32(lens)), q, back, lens)


def test_prompt_rows_more_than_2_to_the_32_elements_apart(at):
    """q, k, v and out as columns of one matrix whose rows are 2^24 elements long, bit for bit as from compact rows;
    among the values one infinity in view of some rows."""
    needs(14)
    tokens, dim, stride = 300, 64, 1 << 24
    wide = torch.empty((tokens - 1) * stride + 4096, device="cuda", dtype=torch.bfloat16)
    assert wide.numel() > 2 ** 32

    def column(first, heads):
        return wide.as_strided((tokens, heads, dim), (stride, dim, 1), first)
    q, k, v, out = column(0, 4), column(256, 2), column(384, 2), column(512, 4)
    compact = [_randn(tokens, heads, dim, seed=210 + heads, dtype=torch.bfloat16) for heads in (4, 2, 2)]
    compact[2][290, 1, 7] = float("inf")
    for to, x in zip((q, k, v), compact):
        to.copy_(x)
    ref = at.prompt_attention(*compact, _cu([170, 130]))
    got = at.prompt_attention(q, k, v, _cu([170, 130]), out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got.nan_to_num(nan=7.0), ref.nan_to_num(nan=7.0))
    assert torch.isinf(ref[290:, 2:, 7]).all() and ref[:290].isfinite().all()


def test_prompt_thousands_of_sequences_of_mixed_lengths(at):
    """3000 sequences of 0 to 600 tokens: blocks of one, two and three steps among each other."""
    g = np.random.default_rng(220)
    lens = g.integers(0, 601, 3000)
    lens[[5, 1500, 2999]] = [600, 0, 513]
    t = int(lens.sum())
    q = _randn(t, 2, 64, seed=221, dtype=torch.bfloat16)
    k = _randn(t, 1, 64, seed=222, dtype=torch.bfloat16)
    v = _randn(t, 1, 64, seed=223, dtype=torch.bfloat16)
    out = torch.full_like(q, float("nan"))
    at.prompt_attention(q, k, v, _cu(lens.tolist()), out=out)
    first = np.concatenate([[0], np.cumsum(lens)])
    for b in [0, 5, 1499, 1500, 1501, 2998, 2999, *g.integers(0, 3000, 60).tolist()]:
        s = slice(int(first[b]), int(first[b + 1]))
        if lens[b]:
            check(out[s], attend(q[s], k[s], v[s], 0.125, True), q.dtype, 64, U[q.dtype])
    assert not out.isnan().any()
