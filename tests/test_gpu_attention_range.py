"""GPU: attention over rows of very different sizes, against the definition in 64 bits
(tests/attention_f64.py)."""
import numpy as np
import pytest
import torch

from attention_f64 import U, attend, bound
from test_gpu_attention import _cu, _i32, _randn, check_decode, make_cache
from test_gpu_kv_cache import layout

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


def cache_of(kv, k, v, lens, page, fmt, seed):
    """A cache that holds these rows, its page table, and (k, v) as it reads them back."""
    table, pages = layout(lens, page, seed)
    cache = kv.PagedKVCache(pages, k.shape[1], k.shape[2], page_size=page, fmt=fmt)
    kv.kv_append(cache, k, v, table, _i32(lens), _cu(lens))
    return cache, table, kv.kv_gather(cache, table, _i32(lens), _cu(lens), tokens=sum(lens), dtype=torch.float32)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,heads,kv_heads,page", [([9], 1, 1, 16), ([700, 40], 8, 2, 16), ([5000], 4, 4, 64)])
def test_decode_one_large_value_row(at, kv, lens, heads, kv_heads, page, dim, dtype, fmt):
    """One key's values are 2^up larger than the others' and its weight 2^-drop of theirs: it adds
    up to as much as they do, or nothing that counts, and takes nothing from what they add,
    wherever it stands in the sequence."""
    q = _randn(len(lens), heads, dim, seed=100, dtype=dtype, gain=0.5)
    q[..., 0] = 1.0
    k = _randn(sum(lens), kv_heads, dim, seed=101, dtype=torch.float32)
    k[..., 0] = 0.0
    v = _randn(sum(lens), kv_heads, dim, seed=102, dtype=torch.float32)
    first = np.concatenate([[0], np.cumsum(lens)[:-1]])
    for drop, up in ((80, 22), (80, 26), (80, 28), (80, 30), (80, 32), (80, 60), (30, 30), (80, 84)):
        for where in (0.0, 0.5, 1.0):
            kk, vv = k.clone(), v.clone()
            for a, n in zip(first, lens):
                row = int(a + where * (n - 1))
                kk[row] = 0.0
                kk[row, :, 0] = -drop * np.log(2.0) * dim ** 0.5       # the score is -drop log 2
                vv[row] *= 2.0 ** up
            cache, table, back = cache_of(kv, kk, vv, lens, page, fmt, 103)
            check_decode(at.paged_decode_attention(q, cache, table, _i32(lens)), q, back, lens)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
def test_decode_value_rows_over_32_octaves(at, kv, order, fmt):
    """V rows whose scales span 2^32, each at a score of its own."""
    lens, dim = [3000, 257], 64
    q = _randn(2, 8, dim, seed=110, dtype=torch.bfloat16, gain=2.0)
    k = _randn(sum(lens), 2, dim, seed=111, dtype=torch.float32)
    v = _randn(sum(lens), 2, dim, seed=112, dtype=torch.float32)
    octaves = torch.cat([torch.linspace(-16, 16, n) for n in lens])
    if order == "falling":
        octaves = -octaves
    elif order == "mixed":
        octaves = octaves[torch.randperm(sum(lens), generator=torch.Generator().manual_seed(113))]
    v *= torch.exp2(octaves.round())[:, None, None].cuda()
    cache, table, back = cache_of(kv, k, v, lens, 64, fmt, 114)
    check_decode(at.paged_decode_attention(q, cache, table, _i32(lens)), q, back, lens)


def fp16_rows(n, heads, kv_heads, dim, seed):
    """q, k, v of n tokens: key j's weight is about 2^-drop_j of the first key's, its values 2^drop_j
    of the first's, drop_j from 0 to 26, so all keys count alike."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    drop = torch.randint(0, 27, (n, kv_heads, 1), device="cuda", generator=g).float()
    drop[0] = 0
    q = _randn(n, heads, dim, seed=seed + 1, dtype=torch.float16, gain=0.1)
    q[..., 0] = 1.0
    k = _randn(n, kv_heads, dim, seed=seed + 2, dtype=torch.float16, gain=0.1)
    k[..., :1] = -drop * np.log(2.0) * dim ** 0.5
    v = (0.5 + 0.5 * torch.rand(n, kv_heads, dim, device="cuda", generator=g)) * torch.exp2(drop - 12)
    return q, k, v.half()


def check_fp16(got, q, k, v, causal):
    """The bound of attention_f64, and what FP16's smallest steps add: the largest weight of a row is
    at least 2^7 units, so rounding to multiples of 2^-24 units is off by at most 2^-32 of it."""
    n, heads, dim = q.shape
    out, size, spread = attend(q, k, v, dim ** -0.5, causal)
    group = heads // k.shape[1]
    s = torch.einsum("qhd,khd->hqk", q.double(), k.double().repeat_interleave(group, 1)) * dim ** -0.5
    seen = torch.ones_like(s, dtype=torch.bool)
    if causal:
        seen = seen.tril(k.shape[0] - n)
    s = s.masked_fill(~seen, -torch.inf)
    total = torch.exp(s - s.amax(-1, keepdim=True)).sum(-1).transpose(0, 1)[..., None]
    steps = torch.einsum("hqk,khd->qhd", seen.double(), v.double().abs().repeat_interleave(group, 1)) * 2.0 ** -32 / total
    err = (got.double() - out).abs()
    lim = bound(out, size, spread, torch.float16, dim, U[torch.float16]) + steps
    assert bool((err <= lim).all()), f"worst {float((err / lim).max()):.3g} x bound"


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [40, 700])
def test_prompt_fp16_small_weights_of_large_values(at, n, dim, causal):
    q, k, v = fp16_rows(n, 4, 2, dim, 130)
    check_fp16(at.prompt_attention(q, k, v, _cu([n]), causal=causal), q, k, v, causal)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [40, 5000])
def test_decode_fp16_small_weights_of_large_values(at, kv, n, dim):
    q, k, v = fp16_rows(n, 4, 2, dim, 140)
    cache, table, _ = cache_of(kv, k, v, [n], 16, "f16", 141)
    check_fp16(at.paged_decode_attention(q[-1:], cache, table, _i32([n])), q[-1:], k, v, False)


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [2, 300])
def test_decode_small_rows_where_the_large_are_zero(at, kv, n, dim, fmt):
    """Every other row is 2^up larger, and zero in the odd elements, which the small rows alone make."""
    q = _randn(3, 4, dim, seed=170, dtype=torch.bfloat16)
    k = _randn(n, 2, dim, seed=171, dtype=torch.float32)
    even = (torch.arange(dim, device="cuda") % 2 == 0).float()
    for up in (20, 32, 45, 58):
        v = _randn(n, 2, dim, seed=172, dtype=torch.float32)
        v[0::2] *= 2.0 ** up * even
        v[1::2] *= 1 - even
        cache, table, back = cache_of(kv, k, v, [n], 16, fmt, 173)
        for row in range(3):
            check_decode(at.paged_decode_attention(q[row:row + 1], cache, table, _i32([n])), q[row:row + 1], back, [n])


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "f16"])
@pytest.mark.parametrize("n", [2, 300])
def test_decode_fp16_small_weights_where_the_large_rows_are_zero(at, kv, n, fmt):
    """Every other key has 2^-drop of the weight, and the odd elements of V to itself."""
    dim = 64
    q = _randn(1, 4, dim, seed=180, dtype=torch.float16, gain=0.1)
    q[..., 0] = 1.0
    even = (torch.arange(dim, device="cuda") % 2 == 0).float()
    for drop in (26, 31, 34, 37):
        k = _randn(n, 2, dim, seed=181, dtype=torch.float32) * 0.1
        k[..., 0] = 0
        k[1::2, :, 0] = -drop * np.log(2.0) * dim ** 0.5
        v = 1.0 + torch.rand(n, 2, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(182))
        v[0::2] *= even
        v[1::2] *= (1 - even) * 2.0 ** 14
        cache, table, back = cache_of(kv, k.half(), v.half(), [n], 16, fmt, 183)
        check_decode(at.paged_decode_attention(q, cache, table, _i32([n])), q, back, [n])
