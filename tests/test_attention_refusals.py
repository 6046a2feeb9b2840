"""CPU: refusals of the attention entries that hang on several arguments at once.  Every call has a
misaligned query pointer, so that the last check refuses (2) what the others let through."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from inspark_proper_format_b200 import _lib, build
    build.build()
    return _lib.load()


def _prompt(lib, tokens=4, heads=4, dim=64, out=(256, 64), scale=1.0):
    return lib.isp_prompt_attention(264, 256, 256, 0, tokens, 4, 64, 64, 1, heads, 2, dim, 1 << 20, dim, 1 << 20, dim,
                                    1 << 20, dim, scale, 1, 256, *out, None)


def _decode(lib, tokens=4, heads=4, dim=64, out=(256, 64), scale=1.0):
    from inspark_proper_format_b200 import _lib
    cache = _lib.KVCache(256, 512, 1024, 2048, 4, _lib.E4M3, 16, 2, dim)
    return lib.isp_paged_decode(264, 0, 1 << 20, dim, ctypes.byref(cache), 64, 4, 4, 64, tokens, heads, scale, 256, *out,
                                256, 1 << 30, None)


def _overlap(tokens, heads, dim, token_stride, head_stride):
    taken = set()
    for t in range(tokens):
        for h in range(heads):
            row = range(t * token_stride + h * head_stride, t * token_stride + h * head_stride + dim)
            if not taken.isdisjoint(row):
                return True
            taken.update(row)
    return False


@pytest.mark.parametrize("entry", [_prompt, _decode])
@pytest.mark.parametrize("tokens,heads", [(1, 4), (4, 2), (3, 6), (2, 2), (7, 4)])
def test_output_rows_that_overlap_are_refused(lib, entry, tokens, heads):
    """Every pair of strides up to a few rows: refused (1) exactly where two rows share an element."""
    for dim in (64, 128):
        for token_stride in range(0, 8 * dim, 32):
            for head_stride in range(0, 8 * dim, 32):
                status = entry(lib, tokens, heads, dim, (token_stride, head_stride))
                want = 1 if _overlap(tokens, heads, dim, token_stride, head_stride) else 2
                assert status == want, (token_stride, head_stride)


@pytest.mark.parametrize("entry", [_prompt, _decode])
def test_scales_that_overflow_in_base_2_are_refused(lib, entry):
    """The kernels take scale * log2(e), which is infinite from FP32's largest value / 1.4427 on."""
    for scale in (2.4e38, 3.4e38, float("inf"), 0.0, -1.0, float("nan")):
        assert entry(lib, scale=scale) == 7, scale
    for scale in (2.3e38, 1e-40, 1.0):
        assert entry(lib, scale=scale) == 2, scale
