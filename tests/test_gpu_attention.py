"""GPU: prompt attention and paged decode attention against the definition in 64 bits
(tests/attention_f64.py), with error bounds from the formats' unit roundoffs."""
import math

import numpy as np
import pytest
import torch

from attention_f64 import U, attend, check
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


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cu(lens):
    return _i32(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))


def _randn(*shape, seed, dtype, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * gain).to(dtype)


def check_prompt(out, q, k, v, lens, keys, causal, scale=None):
    a = b = 0
    dim = q.shape[2]
    for n, m in zip(lens, keys):
        ref = attend(q[a:a + n], k[b:b + m], v[b:b + m], scale or 1 / math.sqrt(dim), causal)
        check(out[a:a + n], ref, q.dtype, dim, U[q.dtype])
        a, b = a + n, b + m


PROMPTS = [
    ([1], [1], 1, 1),
    ([1, 2, 127, 128, 129, 255, 256, 257], None, 4, 2),
    ([300, 0, 17, 640], None, 5, 5),
    ([5, 130, 1, 400], [90, 130, 700, 513], 8, 1),               # behind cached prefixes
    ([200, 40], [100, 0], 6, 2),                                 # queries that see no key
    ([1100], None, 7, 1),
    ([64] * 40, None, 3, 3),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,keys,heads,kv_heads", PROMPTS)
def test_prompt_against_definition(at, lens, keys, heads, kv_heads, dim, dtype, causal):
    keys = keys or lens
    q = _randn(sum(lens), heads, dim, seed=1, dtype=dtype, gain=2.0)
    k = _randn(sum(keys), kv_heads, dim, seed=2, dtype=dtype)
    v = _randn(sum(keys), kv_heads, dim, seed=3, dtype=dtype)
    out = at.prompt_attention(q, k, v, _cu(lens), cu_seqlens_k=_cu(keys), causal=causal)
    check_prompt(out, q, k, v, lens, keys, causal)


@pytest.mark.parametrize("gain", [0.0, 8.0, 60.0])
def test_prompt_flat_and_peaked_rows(at, gain):
    """Scores all equal, and scores so large that one key takes the row; the maximum moves
    from tile to tile."""
    lens, dim = [517], 64
    q = _randn(517, 2, dim, seed=4, dtype=torch.bfloat16, gain=gain)
    k = _randn(517, 2, dim, seed=5, dtype=torch.bfloat16)
    k *= torch.linspace(0.1, 1.0, 517, device="cuda")[:, None, None].bfloat16()
    v = _randn(517, 2, dim, seed=6, dtype=torch.bfloat16)
    out = at.prompt_attention(q, k, v, _cu(lens))
    check_prompt(out, q, k, v, lens, lens, True)


def test_prompt_scale_and_negative_scores(at):
    lens, dim = [300], 128
    q = _randn(300, 2, dim, seed=7, dtype=torch.float16).abs()
    k = -_randn(300, 2, dim, seed=8, dtype=torch.float16).abs()       # every score far below zero
    v = _randn(300, 2, dim, seed=9, dtype=torch.float16)
    for scale in (0.3, 1.0):
        out = at.prompt_attention(q, k, v, _cu(lens), scale=scale)
        check_prompt(out, q, k, v, lens, lens, True, scale)


def test_prompt_operands_of_a_fused_projection_and_given_output(at):
    t, heads, dim = 333, 6, 64
    qkv = _randn(t, 3 * heads * dim, seed=10, dtype=torch.bfloat16)
    q, k, v = (qkv[:, i * heads * dim:(i + 1) * heads * dim].view(t, heads, dim) for i in range(3))
    lens = [100, 233]
    ref = at.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), _cu(lens))
    check_prompt(ref, q, k, v, lens, lens, True)
    assert torch.equal(at.prompt_attention(q, k, v, _cu(lens)), ref)
    wide = torch.full((t, heads + 2, dim + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    got = at.prompt_attention(q, k, v, _cu(lens), out=wide[:, 1:-1, :dim])
    assert torch.equal(got, ref) and got.data_ptr() == wide[:, 1:-1].data_ptr()
    assert bool((wide[:, 0] == 7).all() and (wide[:, -1] == 7).all() and (wide[..., dim:] == 7).all())
    # heads outermost, an unaligned base, a broadcast key head
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(t * heads * dim + 1, device="cuda", dtype=torch.bfloat16)[1:].view(t, heads, dim).copy_(k)
    assert torch.equal(at.prompt_attention(swapped, odd, v, _cu(lens)), ref)
    one = k[:, :1]
    assert torch.equal(at.prompt_attention(q, one.expand(t, heads, dim), v, _cu(lens)),
                       at.prompt_attention(q, one.expand(t, heads, dim).contiguous(), v, _cu(lens)))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_masked_places_do_not_matter(at, bad, dim):
    """Non-finite keys and values of later tokens and of the neighbouring sequences leave a
    row as it is; the rows that see a non-finite value show it."""
    lens, heads = [200, 130, 77], 2
    t = sum(lens)
    q = _randn(t, heads, dim, seed=11, dtype=torch.bfloat16)
    k = _randn(t, heads, dim, seed=12, dtype=torch.bfloat16)
    v = _randn(t, heads, dim, seed=13, dtype=torch.bfloat16)
    ref = at.prompt_attention(q, k, v, _cu(lens))
    for which in ("k", "v"):
        kk, vv = k.clone(), v.clone()
        hit = 200 + 97                                          # token 97 of the second sequence
        (kk if which == "k" else vv)[hit, 0, 3] = bad
        out = at.prompt_attention(q, kk, vv, _cu(lens))
        same = torch.ones(t, heads, dtype=torch.bool, device="cuda")
        same[hit:200 + 130, 0] = False
        assert torch.equal(out[same], ref[same])
        rows = out[hit:200 + 130, 0].float()
        if which == "v":
            assert torch.equal(rows[:, :3], ref[hit:200 + 130, 0, :3].float())
            if math.isnan(bad):
                assert rows[:, 3].isnan().all()
            else:
                assert (rows[:, 3] == bad).all()
        elif not math.isinf(bad):
            assert rows.isnan().all()
    # both signs of infinity in view cancel to NaN
    vv = v.clone()
    vv[0, 0, 1], vv[1, 0, 1] = float("inf"), float("-inf")
    out = at.prompt_attention(q, k, vv, _cu(lens))
    assert out[0, 0, 1] == float("inf") and out[1:200, 0, 1].isnan().all()
    assert torch.equal(out[200:], ref[200:]) and torch.equal(out[:, 1], ref[:, 1])


def test_prompt_lowest_values(at):
    """Operands at the type's largest magnitude: scores beyond FP16, products of both signs."""
    dim, n = 64, 140
    big = torch.finfo(torch.float16).max
    q = torch.zeros(n, 1, dim, device="cuda", dtype=torch.float16)
    q[:, :, 0] = big
    k = torch.zeros(n, 1, dim, device="cuda", dtype=torch.float16)
    k[::2, :, 0], k[1::2, :, 0] = -big, big
    v = _randn(n, 1, dim, seed=14, dtype=torch.float16)
    out = at.prompt_attention(q, k, v, _cu([n]))
    for i in range(n):
        seen = v[1:i + 1:2, 0] if i else v[:1, 0]
        torch.testing.assert_close(out[i, 0].float(), seen.float().mean(0), rtol=2e-3, atol=2e-3)


def test_prompt_unclaimed_rows_and_bad_bounds(at):
    from inspark_proper_format_b200 import _lib
    q = _randn(60, 1, 64, seed=15, dtype=torch.bfloat16)
    out = at.prompt_attention(q, q, q, _i32([0, 20, 40]))         # rows 40.. belong to no sequence
    check_prompt(out[:40], q, q, q, [20, 20], [20, 20], True)
    at.prompt_attention(q, q, q, _i32([0, 20, 60]), cu_seqlens_k=_i32([0, 20, 61]))
    assert _lib.read_device_error(clear=True) == _lib.ISP_ERR_ARG
    assert at.prompt_attention(q[:0], q, q, _i32([0]), cu_seqlens_k=_i32([0])).shape == (0, 1, 64)
    assert not at.prompt_attention(q, q[:0], q[:0], _i32([0, 60]), cu_seqlens_k=_i32([0, 0])).any()


def test_prompt_many_sequences(at):
    lens = [(i * 7) % 23 for i in range(700)]
    t = sum(lens)
    q = _randn(t, 2, 64, seed=16, dtype=torch.bfloat16)
    k = _randn(t, 1, 64, seed=17, dtype=torch.bfloat16)
    v = _randn(t, 1, 64, seed=18, dtype=torch.bfloat16)
    out = at.prompt_attention(q, k, v, _cu(lens))
    first = np.concatenate([[0], np.cumsum(lens)])
    for b in (0, 1, 2, 348, 349, 698, 699):
        s = slice(int(first[b]), int(first[b + 1]))
        check(out[s], attend(q[s], k[s], v[s], 0.125, True), q.dtype, 64, U[q.dtype])
    assert not out.isnan().any()


def test_prompt_repeats_bit_for_bit(at):
    q = _randn(3000, 4, 64, seed=19, dtype=torch.bfloat16)
    cu = _cu([1700, 1300])
    a = at.prompt_attention(q, q, q, cu)
    assert all(torch.equal(a, at.prompt_attention(q, q, q, cu)) for _ in range(5))


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
def make_cache(kv, lens, kv_heads, dim, page, fmt, dtype, seed, extra=2):
    """A cache that holds random rows of these sequences, and (k, v) as it reads them back."""
    table, pages = layout(lens, page, seed, extra)
    cache = kv.PagedKVCache(pages, kv_heads, dim, page_size=page, fmt=fmt)
    t = sum(lens)
    k = _randn(t, kv_heads, dim, seed=seed + 1, dtype=dtype)
    v = _randn(t, kv_heads, dim, seed=seed + 2, dtype=dtype)
    kv.kv_append(cache, k, v, table, _i32(lens), _cu(lens))
    back = kv.kv_gather(cache, table, _i32(lens), _cu(lens), tokens=t, dtype=torch.float32)
    return cache, table, back


def check_decode(out, q, back, lens, scale=None):
    a = 0
    for b, n in enumerate(lens):
        k, v = back[0][a:a + n], back[1][a:a + n]
        check(out[b:b + 1], attend(q[b:b + 1], k, v, scale or 1 / math.sqrt(q.shape[2]), False), q.dtype, q.shape[2],
              U[q.dtype])
        a += n


DECODES = [
    ([1], 1, 1, 16),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129], 20, 20, 16),
    ([700, 0, 3000, 5], 8, 2, 48),
    ([257, 1031], 7, 1, 64),
    ([100, 37], 64, 2, 7),                                      # 32 queries to a key head
    ([5000], 12, 1, 1),                                         # one token per page
    ([900] * 50, 4, 4, 128),
]


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "16"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,heads,kv_heads,page", DECODES)
def test_decode_against_definition(at, kv, lens, heads, kv_heads, page, dim, dtype, fmt):
    fmt = fmt if fmt != "16" else ("bf16" if dtype == torch.bfloat16 else "f16")
    cache, table, back = make_cache(kv, lens, kv_heads, dim, page, fmt, dtype, 20)
    q = _randn(len(lens), heads, dim, seed=23, dtype=dtype, gain=2.0)
    ws = at.DecodeWorkspace()
    out = at.paged_decode_attention(q, cache, table, _i32(lens), workspace=ws)
    check_decode(out, q, back, lens)
    for _ in range(3):                                          # the workspace is ready again, the result the same
        assert torch.equal(out, at.paged_decode_attention(q, cache, table, _i32(lens), workspace=ws))
    assert torch.equal(out, at.paged_decode_attention(q, cache, table, _i32(lens)))


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "bf16"])
def test_decode_one_long_context(at, kv, fmt):
    lens = [70001]
    cache, table, back = make_cache(kv, lens, 2, 128, 64, fmt, torch.bfloat16, 30)
    q = _randn(1, 8, 128, seed=33, dtype=torch.bfloat16, gain=3.0)
    out = at.paged_decode_attention(q, cache, table, _i32(lens))
    check_decode(out, q, back, lens)


def test_decode_strides_scale_and_given_output(at, kv):
    lens, heads, dim = [90, 300, 0], 8, 64
    cache, table, back = make_cache(kv, lens, 4, dim, 16, "e4m3", torch.bfloat16, 40)
    qkv = _randn(3, 3 * heads * dim, seed=43, dtype=torch.bfloat16)
    q = qkv[:, heads * dim:2 * heads * dim].view(3, heads, dim)
    out = at.paged_decode_attention(q, cache, table, _i32(lens), scale=0.5)
    check_decode(out, q, back, lens, 0.5)
    wide = torch.full((3, heads + 1, dim + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    got = at.paged_decode_attention(q, cache, table, _i32(lens), scale=0.5, out=wide[:, 1:, 8:])
    assert torch.equal(got, out)
    assert bool((wide[:, 0] == 7).all() and (wide[..., :8] == 7).all())
    wider = torch.cat([table, table], 1)                        # a page table that is a view of a larger one
    assert torch.equal(at.paged_decode_attention(q, cache, wider[:, :table.shape[1]], _i32(lens), scale=0.5), out)


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "bf16"])
def test_decode_stale_rows_do_not_matter(at, kv, fmt):
    """What the last page holds behind the sequence's end, and what other pages hold, is not read into it."""
    lens = [50, 7]
    cache, table, back = make_cache(kv, lens, 2, 64, 16, fmt, torch.bfloat16, 50, extra=3)
    q = _randn(2, 4, 64, seed=53, dtype=torch.bfloat16)
    ref = at.paged_decode_attention(q, cache, table, _i32(lens))
    mine = torch.zeros(cache.pages, 16, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        for p in range(n):
            mine[table[b, p // 16].long(), p % 16] = True
    stale = ~mine[:, None].expand(cache.pages, 2, 16)
    if cache.k_scale is not None:
        cache.k_scale[stale], cache.v_scale[stale] = float("nan"), float("inf")
        cache.k.view(torch.uint8)[stale] = 0x7F
        cache.v.view(torch.uint8)[stale] = 0xFF
    else:
        cache.k[stale], cache.v[stale] = float("nan"), float("inf")
    assert torch.equal(at.paged_decode_attention(q, cache, table, _i32(lens)), ref)


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "bf16"])
def test_decode_non_finite_rows_show(at, kv, fmt):
    lens = [130, 40]
    cache, table, _ = make_cache(kv, lens, 2, 64, 16, fmt, torch.bfloat16, 60)
    q = _randn(2, 4, 64, seed=63, dtype=torch.bfloat16)
    ref = at.paged_decode_attention(q, cache, table, _i32(lens))
    row = torch.randn(2, 2, 64, device="cuda").bfloat16()
    row[0, 0, 9] = float("nan")
    fine = torch.randn(2, 2, 64, device="cuda").bfloat16()
    kv.kv_append(cache, fine, row, table, _i32([130, 0]))       # the last row of sequence 0, head 0: a NaN value
    out = at.paged_decode_attention(q, cache, table, _i32(lens))
    assert torch.equal(out[1], ref[1]) and not out[0, 2:].isnan().any()
    assert out[0, :2, 9].isnan().all()
    kv.kv_append(cache, row, fine, table, _i32([130, 0]))       # and as a key
    out = at.paged_decode_attention(q, cache, table, _i32(lens))
    assert out[0, :2].isnan().all() and not out[0, 2:].isnan().any() and torch.equal(out[1], ref[1])


def test_decode_bad_pages_are_recorded(at, kv):
    from inspark_proper_format_b200 import _lib
    cache = kv.PagedKVCache(4, 1, 64, page_size=16, fmt="bf16")
    q = _randn(1, 1, 64, seed=70, dtype=torch.bfloat16)
    for table, n in ((_i32([[0, 4]]), 20), (_i32([[-1, 1]]), 3), (_i32([[0, 1]]), 33)):
        out = at.paged_decode_attention(q, cache, table, _i32([n]))
        assert _lib.read_device_error(clear=True) == _lib.ISP_ERR_ARG
        assert not out.isnan().any()


def test_decode_agrees_with_prompt_attention(at, kv):
    """The last query of a causal prompt is a decode step over the same rows."""
    lens = [200, 513, 1]
    cache, table, back = make_cache(kv, lens, 2, 128, 32, "bf16", torch.bfloat16, 80)
    k, v = back[0].bfloat16(), back[1].bfloat16()
    q = _randn(sum(lens), 8, 128, seed=83, dtype=torch.bfloat16)
    full = at.prompt_attention(q, k, v, _cu(lens))
    last = np.cumsum(lens) - 1
    out = at.paged_decode_attention(q[last], cache, table, _i32(lens))
    check_decode(out, q[last], back, lens)
    check_decode(full[last], q[last], back, lens)


def test_another_stream_and_graph_capture(at, kv):
    lens = [300, 41]
    cache, table, back = make_cache(kv, lens, 4, 64, 16, "e4m3", torch.bfloat16, 90)
    q = _randn(2, 8, 64, seed=93, dtype=torch.bfloat16)
    lengths, ws = _i32(lens), at.DecodeWorkspace()
    ref = at.paged_decode_attention(q, cache, table, lengths, workspace=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = at.paged_decode_attention(q, cache, table, lengths, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
    k = _randn(2, 4, 64, seed=94, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kv.kv_append(cache, k, k, table, lengths)
        at.paged_decode_attention(q, cache, table, lengths, workspace=ws, out=out)
    for step in range(3):                                       # lengths move on the device between replays
        lengths.copy_(_i32([300 + step, 41 + step]))
        graph.replay()
        k2, v2 = kv.kv_gather(cache, table, lengths, _cu([300 + step, 41 + step]), tokens=341 + 2 * step,
                              dtype=torch.float32)
        check_decode(out, q, (k2, v2), [300 + step, 41 + step])


def test_refusals(at, kv):
    q = torch.zeros(4, 4, 64, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    cu = _i32([0, 4])
    bad = [
        lambda: at.prompt_attention(q.float(), k.float(), k.float(), cu),
        lambda: at.prompt_attention(q, k.half(), k.half(), cu),
        lambda: at.prompt_attention(q[:, :3], k, k, cu),
        lambda: at.prompt_attention(q[..., :32], k[..., :32], k[..., :32], cu),
        lambda: at.prompt_attention(q, k, k[:2], cu),
        lambda: at.prompt_attention(q, k[:2], k[:2], cu),
        lambda: at.prompt_attention(q, k, k, cu.long()),
        lambda: at.prompt_attention(q, k, k, cu.cpu()),
        lambda: at.prompt_attention(q, k, k, cu, cu_seqlens_k=_i32([0, 2, 4])),
        lambda: at.prompt_attention(q, k, k, cu, scale=0.0),
        lambda: at.prompt_attention(q, k, k, cu, scale=float("inf")),
        lambda: at.prompt_attention(q, k, k, cu, out=torch.empty_like(q).half()),
        lambda: at.prompt_attention(q.cpu(), k.cpu(), k.cpu(), cu),
    ]
    cache = kv.PagedKVCache(4, 2, 64, page_size=4, fmt="bf16")
    table, lens = _i32([[0]] * 4), _i32([1] * 4)
    bad += [
        lambda: at.paged_decode_attention(q.half(), cache, table, lens),
        lambda: at.paged_decode_attention(q[:, :3], cache, table, lens),
        lambda: at.paged_decode_attention(q[:3], cache, table, lens),
        lambda: at.paged_decode_attention(q, cache, table, lens.long()),
        lambda: at.paged_decode_attention(q, cache, table[:, :0], lens),
        lambda: at.paged_decode_attention(q, cache, table, lens, scale=-1.0),
        lambda: at.paged_decode_attention(q.float(), cache, table, lens),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
