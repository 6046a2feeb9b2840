"""GPU: views of tensors as operands of the cache and attention calls."""
import pytest
import torch

from test_gpu_attention import _i32, _randn, make_cache

pytestmark = pytest.mark.gpu


def test_sequences_that_share_one_expanded_page_table():
    """Three queries over prefixes of one context, its page table expanded to three rows."""
    from inspark_proper_format_b200 import attention, kv_cache
    cache, table, _ = make_cache(kv_cache, [200], 2, 64, 16, "e4m3", torch.bfloat16, 120)
    q = _randn(3, 4, 64, seed=123, dtype=torch.bfloat16)
    lengths, shared = _i32([200, 131, 7]), table.expand(3, table.shape[1])
    out = attention.paged_decode_attention(q, cache, shared, lengths)
    assert torch.equal(out, attention.paged_decode_attention(q, cache, shared.contiguous(), lengths))
    for got, want in zip(kv_cache.kv_gather(cache, shared, lengths), kv_cache.kv_gather(cache, shared.contiguous(), lengths)):
        assert torch.equal(got, want) and got.any(-1).all()
