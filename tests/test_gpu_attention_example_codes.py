"""GPU: the serving example over 8-bit caches, row by row against the definition in 64 bits over what the
cache holds."""
import numpy as np
import pytest
import torch

from attention_f64 import U, attend, check
from test_gpu_attention_example import example  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_rows_of_the_example_against_the_definition(example, fmt, monkeypatch):  # noqa: F811
    """The decode steps read codes and scales as they are; the chunk behind the cached prefix reads them
    rounded to BF16.  (The first prompts' rows come from unquantised keys and values.)"""
    from inspark_proper_format_b200 import kv_cache
    queries, gathers = [], []

    def prompt_attention(q, *args, _call=example.prompt_attention, **kw):
        queries.append(q)
        return _call(q, *args, **kw)

    def kv_gather(cache, table, lengths, cu, _call=example.kv_gather, **kw):
        gathers.append((cache, table.clone(), lengths.clone(), cu))
        return _call(cache, table, lengths, cu, **kw)
    monkeypatch.setattr(example, "prompt_attention", prompt_attention)
    monkeypatch.setattr(example, "kv_gather", kv_gather)
    prompts, steps, heads, dim = (70, 33, 1, 128), 3, 4, 64
    got, _, _ = example.main(dim=heads * dim, heads=heads, prompts=prompts, steps=steps, page_size=16, fmt=fmt)
    cache, table, lengths, cu = gathers[-1]
    lens = [prompts[0] + 40 + steps] + [n + steps for n in prompts[1:]]
    assert lengths.tolist() == lens
    first = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q = queries[-1]                                             # of every token
    k, v = kv_cache.kv_gather(cache, table, lengths, cu, tokens=sum(lens), dtype=torch.float32)

    def row(i, b, n, dtype):
        """Row i of the results is token n of sequence b."""
        s = slice(first[b], first[b] + n + 1)
        ref = attend(q[first[b] + n:first[b] + n + 1], k[s].to(dtype), v[s].to(dtype), dim ** -0.5, True)
        check(got[i].view(1, heads, dim), ref, torch.bfloat16, dim, U[torch.bfloat16])
    row(len(prompts), 0, prompts[0] + 39, torch.bfloat16)
    for step in range(steps):
        for b in range(len(prompts)):
            row(len(prompts) + 1 + step * len(prompts) + b, b, lens[b] - steps + step, torch.float32)
    assert got.shape[0] == len(prompts) + 1 + steps * len(prompts)
