"""CPU: host-side refusals of the cache and attention entry points (before any device work),
and the 64-bit definition the GPU tests compare with."""
import ctypes

import pytest
import torch

from attention_f64 import attend


@pytest.fixture(scope="module")
def lib():
    from inspark_proper_format_b200 import _lib, build
    build.build()
    return _lib.load()


def _cache(**kw):
    from inspark_proper_format_b200 import _lib
    d = dict(k=256, v=512, k_scale=1024, v_scale=2048, pages=4, dtype=_lib.E4M3, page_size=16, kv_heads=2, head_dim=64)
    d.update(kw)
    return _lib.KVCache(**d)


def _append(lib, cache, *, k=256, dtype=0, t=2, ks=128, hs=64, cu=None, table=64, stride=4, width=4, lengths=64, b=2):
    return lib.isp_kv_append(k, 256, dtype, t, ks, hs, 128, 64, cu, table, stride, width, lengths, b,
                             ctypes.byref(cache) if cache is not None else None, None)


def test_cache_refusals(lib):
    ok = _cache()
    assert _append(lib, None) == 7 and _append(lib, ok, k=None) == 7 and _append(lib, ok, table=None) == 7
    assert _append(lib, _cache(k=None)) == 7
    assert _append(lib, _cache(k_scale=None)) == 7                       # 8-bit rows need scales
    assert _append(lib, _cache(dtype=0)) == 7                            # 16-bit rows have none
    assert _append(lib, _cache(dtype=1)) == 3 and _append(lib, ok, dtype=3) == 3
    for kw in (dict(head_dim=96), dict(pages=0), dict(page_size=0), dict(kv_heads=0), dict(pages=2 ** 32)):
        assert _append(lib, _cache(**kw)) == 1
    assert _append(lib, ok, t=3) == 1 and _append(lib, ok, width=0) == 1 and _append(lib, ok, stride=3) == 1
    assert _append(lib, ok, t=-1, cu=64) == 1 and _append(lib, ok, ks=-64) == 1
    assert _append(lib, ok, ks=129) == 2 and _append(lib, ok, k=264) == 2 and _append(lib, _cache(v=520)) == 2


def test_attention_refusals(lib):
    def prompt(q=256, dtype=0, tq=4, b=1, heads=4, kv=2, dim=64, scale=1.0, causal=1, qs=256, cu=64):
        return lib.isp_prompt_attention(q, 256, 256, dtype, tq, 4, cu, cu, b, heads, kv, dim, qs, 64, 128, 64, 128, 64,
                                        scale, causal, 256, 256, 64, None)
    assert prompt(q=None) == 7 and prompt(cu=None) == 7 and prompt(causal=2) == 7
    assert prompt(scale=0.0) == 7 and prompt(scale=float("nan")) == 7 and prompt(scale=float("inf")) == 7
    assert prompt(dtype=1) == 3
    assert prompt(dim=80) == 1 and prompt(heads=3) == 1 and prompt(kv=0) == 1 and prompt(b=-1) == 1 and prompt(tq=-1) == 1
    assert prompt(q=258) == 2 and prompt(qs=257) == 2
    assert prompt(b=65537) == 1 and prompt(qs=0) == 1                    # too many sequences, overlapping rows

    def decode(cache=None, dtype=0, heads=4, scale=1.0, ws=256, size=1 << 30, qs=256):
        return lib.isp_paged_decode(256, dtype, qs, 64, ctypes.byref(cache or _cache()), 64, 4, 4, 64, 2, heads, scale,
                                    256, 256, 64, ws, size, None)
    assert decode(ws=None) == 7 and decode(scale=-1.0) == 7
    assert decode(dtype=1) == 3
    assert decode(_cache(dtype=2, k_scale=None, v_scale=None)) == 3      # FP16 rows, BF16 queries
    assert decode(heads=5) == 1 and decode(size=16) == 1
    assert decode(ws=272) == 2 and decode(qs=129) == 2
    size = ctypes.c_int64(0)
    assert lib.isp_paged_decode_workspace(None) == 7
    assert lib.isp_paged_decode_workspace(ctypes.byref(size)) == 0 and size.value > 0


def test_wrappers_refuse_host_tensors():
    from inspark_proper_format_b200 import attention, kv_cache
    cache = kv_cache.PagedKVCache(2, 1, 64, fmt="bf16", device="cpu")
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        kv_cache.kv_append(cache, x, x, i[None], i)
    with pytest.raises(ValueError):
        kv_cache.kv_gather(cache, i[None], i)
    with pytest.raises(ValueError):
        attention.prompt_attention(x, x, x, torch.tensor([0, 1], dtype=torch.int32))
    with pytest.raises(ValueError):
        attention.paged_decode_attention(x, cache, i[None], i)


def test_definition_by_hand():
    """Two keys with scores 0 and log 3: weights 1/4 and 3/4; the causal row of the first query sees one key."""
    q = torch.tensor([[[1.0]], [[1.0]]])
    k = torch.tensor([[[0.0]], [[1.0]]])
    v = torch.tensor([[[8.0]], [[-4.0]]])
    out, size, spread = attend(q, k, v, float(torch.log(torch.tensor(3.0, dtype=torch.float64))), True)
    torch.testing.assert_close(out[:, 0, 0], torch.tensor([8.0, -1.0], dtype=torch.float64))
    torch.testing.assert_close(size[:, 0, 0], torch.tensor([8.0, 5.0], dtype=torch.float64))
    assert not attend(q, k[:0], v[:0], 1.0, True)[0].any()
