"""GPU: visible keys that make a score infinite.  A score of -inf is a weight of 0: the row is what the
other keys make it, and zeros where there is no other; a score of +inf makes the row NaN."""
import pytest
import torch

from attention_f64 import U, attend, check
from test_gpu_attention import _cu, _i32, _randn
from test_gpu_attention_range import cache_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def at():
    from inspark_proper_format_b200 import attention
    return attention


@pytest.fixture(scope="module")
def kv():
    from inspark_proper_format_b200 import kv_cache
    return kv_cache


def operands(n, dim, dtype, bad, hit):
    q, k, v = (_randn(n, 2, dim, seed=s, dtype=dtype) for s in (150, 151, 152))
    q[..., 3] = torch.where(q[..., 3] < 0, q[..., 3] - 0.5, q[..., 3] + 0.5)       # not 0: 0 inf is NaN
    k[hit, 0, 3] = bad
    return q, k, v


def check_rows(got, q, k, v, hit, bad, causal):
    """Head 0 of queries that see key `hit`: NaN or the attention without that key; head 1 as ever."""
    others = torch.arange(k.shape[0], device="cuda") != hit
    up = (q[:, 0, 3] * bad) > 0
    assert got[up, 0].isnan().all()
    ref = attend(q[:, :1], k[others, :1], v[others, :1], q.shape[2] ** -0.5, causal)
    check(got[~up, :1], [x[~up] for x in ref], q.dtype, q.shape[2], U[q.dtype])
    check(got[:, 1:], attend(q[:, 1:], k[:, 1:], v[:, 1:], q.shape[2] ** -0.5, causal), q.dtype, q.shape[2], U[q.dtype])


@pytest.mark.parametrize("bad", [float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,hit", [(300, 0), (300, 131), (300, 299), (2, 0)])
def test_prompt_keys_with_infinite_scores(at, n, hit, dim, dtype, bad):
    q, k, v = operands(n, dim, dtype, bad, hit)
    check_rows(at.prompt_attention(q, k, v, _cu([n]), causal=False), q, k, v, hit, bad, False)
    out = at.prompt_attention(q, k, v, _cu([n]))
    check_rows(out[hit:], q[hit:], k, v, hit, bad, True)      # the others do not see the key
    if hit:
        ref = attend(q[:hit], k[:hit], v[:hit], dim ** -0.5, True)
        check(out[:hit], ref, dtype, dim, U[dtype])


@pytest.mark.parametrize("bad", [float("inf"), float("-inf")])
@pytest.mark.parametrize("fmt,dtype", [("bf16", torch.bfloat16), ("f16", torch.float16)])
@pytest.mark.parametrize("n,hit", [(2000, 0), (2000, 777), (2000, 1999), (2, 1)])
def test_decode_keys_with_infinite_scores(at, kv, n, hit, fmt, dtype, bad):
    q, k, v = operands(n, 64, dtype, bad, hit)
    cache, table, _ = cache_of(kv, k, v, [n], 16, fmt, 153)
    q = q[:24]                                                # a sequence each, of the same pages
    b = q.shape[0]
    out = at.paged_decode_attention(q, cache, table.expand(b, table.shape[1]), _i32([n] * b))
    check_rows(out, q, k, v, hit, bad, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_whose_scores_are_all_minus_infinity_give_zeros(at, kv, dtype):
    n = 200
    q, k, v = (_randn(n, 2, 64, seed=s, dtype=dtype) for s in (160, 161, 162))
    q[..., 3] = q[..., 3].abs() + 0.5
    k[:, 0, 3] = float("-inf")
    for causal in (True, False):
        out = at.prompt_attention(q, k, v, _cu([n]), causal=causal)
        assert not out[:, 0].any()
        check(out[:, 1:], attend(q[:, 1:], k[:, 1:], v[:, 1:], 0.125, causal), dtype, 64, U[dtype])
    cache, table, _ = cache_of(kv, k, v, [n], 16, "bf16" if dtype == torch.bfloat16 else "f16", 163)
    out = at.paged_decode_attention(q[:1], cache, table, _i32([n]))
    assert not out[:, 0].any() and out[:, 1].any()
