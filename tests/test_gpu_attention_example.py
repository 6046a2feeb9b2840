"""GPU: the serving example end to end (prompts, a chunk behind a cached prefix, graph-replayed
decode steps) against one prompt over all tokens."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location(
        "ar_attention", Path(__file__).resolve().parent.parent / "examples" / "ar_attention.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_example_runs_the_operators_together(example):
    """With a BF16 cache both computations see the same keys and values.  Each is off by at most
    u |o| + (u + 2^-12) A, u = 2^-8: the output's rounding and that of the weights p (and FP32
    sums), where A is the row's attention over |v|, known here to a factor 1 + 2^-6."""
    got, ref, spread = example.main(dim=256, heads=4, prompts=(70, 33, 1, 128), steps=3, page_size=16, fmt="bf16")
    u = 2.0 ** -8
    assert bool(((got - ref).abs() <= 2 * (1 + 2.0 ** -5) * (u * ref.abs() + (u + 2.0 ** -12) * spread)).all())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_example_with_a_quantised_cache(example, fmt):
    from inspark_proper_format_b200 import _lib
    got, ref, _ = example.main(dim=256, heads=4, prompts=(70, 33, 1, 128), steps=3, page_size=16, fmt=fmt)
    assert got.isfinite().all() and ref.isfinite().all() and _lib.read_device_error(clear=True) == 0
