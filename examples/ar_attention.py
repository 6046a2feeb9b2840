"""One causal self-attention block of the AR model (dim 1280, 20 heads) served from a paged,
quantised key-value cache: prompts of different lengths at once, one more chunk of one
conversation behind its cached prefix, then decode steps replayed as one CUDA graph.

    python examples/ar_attention.py

The projections are the INT8 SmoothQuant GEMMs; between them ``kv_append``,
``prompt_attention``, ``kv_gather`` and ``paged_decode_attention``.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from inspark_proper_format_b200.attention import DecodeWorkspace, paged_decode_attention, prompt_attention  # noqa: E402
from inspark_proper_format_b200.gemm import Int8SmoothQuantLinear, scaled_gemm  # noqa: E402
from inspark_proper_format_b200.kv_cache import PagedKVCache, kv_append, kv_gather  # noqa: E402
from inspark_proper_format_b200.norm_quant import norm_quant  # noqa: E402


def quantised(linear: torch.nn.Linear, sample: torch.Tensor) -> Int8SmoothQuantLinear:
    """SmoothQuant (alpha 1) of a linear layer from a sample of its inputs."""
    smooth = (sample.float().abs().amax(0) / 127).clamp_min(1e-5)
    weight = (linear.weight.detach().float() * smooth).abs().amax(1) / 127
    return Int8SmoothQuantLinear(linear, dict(smooth_scale=smooth, input_scale=1.0, weight_scale=weight.clamp_min(1e-12)))


class CausalAttention:
    """x [tokens, dim] BF16 -> (heads' outputs, projected output), both [tokens, dim] BF16; keys and
    values are cached on the way."""

    def __init__(self, dim: int, heads: int, qkv: Int8SmoothQuantLinear, out: Int8SmoothQuantLinear,
                 cache: PagedKVCache):
        self.dim, self.heads, self.qkv, self.out, self.cache = dim, heads, qkv, out, cache
        self.workspace = DecodeWorkspace(cache.device)

    def _project(self, linear, x):
        codes, _ = norm_quant(x, kind="none", fmt="int8", scale=linear.input_scale, smooth=linear.smooth_scale)
        return scaled_gemm(codes, linear.weight_q, a_scale=linear.input_scale, w_scale=linear.weight_scale,
                           bias=linear.bias, out_dtype=torch.bfloat16)

    def _project_out(self, o):
        o = o.flatten(1)
        return o, self._project(self.out, o)

    def _rows(self, x):
        rows = self._project(self.qkv, x).view(x.shape[0], 3, self.heads, self.dim // self.heads)
        return rows[:, 0], rows[:, 1], rows[:, 2]               # views: the kernels take the strides

    def prompt(self, x, cu_seqlens, page_table, lengths):
        """New sequences: their tokens see each other."""
        q, k, v = self._rows(x)
        kv_append(self.cache, k, v, page_table, lengths, cu_seqlens)
        return self._project_out(prompt_attention(q, k, v, cu_seqlens))

    def extend(self, x, cu_seqlens, page_table, lengths, cu_seqlens_k, keys: int):
        """More tokens of sequences that have a cached prefix: they see it as the cache holds it."""
        q, k, v = self._rows(x)
        kv_append(self.cache, k, v, page_table, lengths, cu_seqlens)
        k, v = kv_gather(self.cache, page_table, lengths, cu_seqlens_k, tokens=keys, dtype=q.dtype)
        return self._project_out(prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k=cu_seqlens_k))

    def step(self, x, page_table, lengths):
        """One token of each sequence; nothing here reads the lengths on the host."""
        q, k, v = self._rows(x)
        kv_append(self.cache, k, v, page_table, lengths)
        return self._project_out(paged_decode_attention(q, self.cache, page_table, lengths, workspace=self.workspace))


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def cumulative(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def main(dim=1280, heads=20, prompts=(256, 190, 77, 256, 31, 1, 128, 200), steps=8, page_size=64, fmt="e4m3"):
    torch.manual_seed(0)
    batch, most = len(prompts), max(prompts) + 64 + steps
    width = (most + page_size - 1) // page_size
    tokens = torch.randn(batch, most, dim, device="cuda").bfloat16()         # every sequence's inputs
    linears = [torch.nn.Linear(dim, n, device="cuda") for n in (3 * dim, dim)]
    qkv = quantised(linears[0], tokens.flatten(0, 1))
    out = quantised(linears[1], torch.randn(256, dim, device="cuda"))
    cache = PagedKVCache(batch * width, heads, dim // heads, page_size=page_size, fmt=fmt)
    table = torch.randperm(batch * width, device="cuda").int().view(batch, width)
    block = CausalAttention(dim, heads, qkv, out, cache)

    lens = list(prompts)
    lengths, cu = i32(lens), i32(cumulative(lens))
    results = {}                                                             # (sequence, position) -> heads' outputs
    o, _ = block.prompt(torch.cat([tokens[b, :n] for b, n in enumerate(lens)]), cu, table, lengths)
    at = cumulative(lens)
    for b, n in enumerate(lens):
        results[b, n - 1] = o[at[b + 1] - 1]

    # 40 more tokens of the first sequence behind its prefix
    lens[0] += 40
    lengths = i32(lens)
    o, _ = block.extend(tokens[0, lens[0] - 40:lens[0]], i32([0, 40]), table[:1], lengths[:1], i32([0, lens[0]]), lens[0])
    results[0, lens[0] - 1] = o[-1]

    # decode: one graph, its inputs and lengths moved on the device between replays
    x = torch.empty(batch, dim, device="cuda", dtype=torch.bfloat16)
    pick = torch.arange(batch, device="cuda")
    keep = lengths.clone()
    block.step(x.zero_(), table, keep + 1)                                   # warm up; the rows are written again below
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.copy_(tokens[pick, lengths.long()])
        lengths.add_(1)
        o, y = block.step(x, table, lengths)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for _ in range(steps):
        graph.replay()
        lens = [n + 1 for n in lens]
        for b, n in enumerate(lens):
            results[b, n - 1] = o[b].clone()
    end.record()
    torch.cuda.synchronize()

    # the same rows from one prompt over everything, keys and values as the cache holds them
    cu = i32(cumulative(lens))
    full = torch.cat([tokens[b, :n] for b, n in enumerate(lens)])
    q, _, _ = block._rows(full)
    k, v = kv_gather(cache, table, lengths, cu, tokens=full.shape[0], dtype=torch.bfloat16)
    at = cumulative(lens)
    where = torch.tensor([at[b] + n for b, n in results], device="cuda")
    got, ref = torch.stack(list(results.values())).float(), prompt_attention(q, k, v, cu).flatten(1)[where].float()
    print(f"{batch} sequences, {sum(lens)} cached tokens ({fmt}), {steps} decode steps: "
          f"{start.elapsed_time(end) / steps * 1e3:.0f} us a step, relative difference of {len(results)} rows to one "
          f"prompt over all tokens {float((got - ref).norm() / ref.norm()):.1e}, last output finite: {bool(y.isfinite().all())}")
    return got, ref, prompt_attention(q, k, v.abs(), cu).flatten(1)[where].float()


if __name__ == "__main__":
    main()
