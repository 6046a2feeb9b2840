"""Attention by its definition in 64 bits (torch, any device), with the quantities that
bound a kernel's rounding errors.  Only visible keys enter a row's sums, so what masked
places hold cannot matter."""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # unit roundoffs


def attend(q, k, v, scale, causal):
    """One sequence: q [n, H, D], k, v [m, Hk, D] (64-bit values).  Returns (out, A, B), each
    [n, H, ...]: A = sum p |v| / sum p, B = max over visible keys of scale * sum |q_d k_d|."""
    n, heads, dim = q.shape
    m, kv_heads = k.shape[0], k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    k = k.repeat_interleave(heads // kv_heads, 1)
    v = v.repeat_interleave(heads // kv_heads, 1)
    out = torch.zeros_like(q)
    size = torch.zeros_like(q)
    spread = torch.zeros(n, heads, 1, dtype=torch.float64, device=q.device)
    step = max(1, (1 << 26) // max(1, n * m))
    for h in range(0, heads, step):
        hs = slice(h, min(heads, h + step))
        s = torch.einsum("qhd,khd->hqk", q[:, hs], k[:, hs]) * scale
        b = torch.einsum("qhd,khd->hqk", q[:, hs].abs(), k[:, hs].abs()) * scale
        if causal:
            hidden = torch.arange(m, device=q.device)[None] > torch.arange(n, device=q.device)[:, None] + (m - n)
            s = s.masked_fill(hidden, -torch.inf)
            b = b.masked_fill(hidden, 0.0)
        if m == 0:
            continue
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -torch.inf, torch.zeros_like(top), top))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total == 0, torch.ones_like(total), total)
        out[:, hs] = torch.einsum("hqk,khd->qhd", p, v[:, hs])
        size[:, hs] = torch.einsum("hqk,khd->qhd", p, v[:, hs].abs())
        spread[:, hs] = b.amax(-1).transpose(0, 1)[..., None]
    return out, size, spread


def bound(out, size, spread, dtype, dim, p_unit):
    """Elementwise error bound of a result rounded once to `dtype` whose weights p are rounded
    to `p_unit` and whose scores, sums and exponentials are FP32: a score of D products is
    off by at most (D + 4) * 2^-24 of its absolute sum B (at most half of that counted for
    the running sum of keys, which adds 2^-24 per tile), exp by 2^-21 of its value."""
    u32 = 2.0 ** -24
    inner = (p_unit + 2 * (dim + 4) * u32 * spread + 2.0 ** -20 + 4096 * u32) * size
    return U[dtype] * (out.abs() + inner) + inner + 2.0 ** -24


def check(got, ref, dtype, dim, p_unit):
    out, size, spread = ref
    err = (got.double() - out).abs()
    lim = bound(out, size, spread, dtype, dim, p_unit)
    bad = ~(err <= lim)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / lim).nan_to_num(1e9).max()):.3g} x bound"
