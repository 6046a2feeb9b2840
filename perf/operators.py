"""Serving attention over packed prompts and a paged, quantised key-value cache: what is timed.

Three operators, each in its plain form (elementary torch operations in 32 bits) and as the
framework's calls:

* ``kv``: K and V rows of packed sequences are written into the pages of a cache, quantised per
  (token, head) row, and the written rows are read back (``kv_append`` then ``kv_gather``);
* ``prompt``: attention over packed sequences of different lengths with grouped heads
  (``prompt_attention``), causal from the end of the keys, or over all keys;
* ``decode``: attention of one new token of each sequence over the paged cache
  (``paged_decode_attention``).

A case is a dict of plain values; the lengths of its sequences follow from the case alone, every
tensor from the seed.
"""
import math
import random

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_QMAX = {"e4m3": 448.0, "int8": 127.0}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decode step of the 20-head AR model at batch 64: 64 new rows per head go to the cache
        dict(name="kv_step_e4m3", op="kv", batch=64, lo=1, hi=1, past=900, mix=1, kv_heads=20, dim=64, page=64,
             fmt="e4m3", dtype="bf16"),
        # the same model's prompts, 64 x 256 tokens, written at once
        dict(name="kv_prompt_int8", op="kv", batch=64, lo=256, hi=256, past=0, mix=2, kv_heads=20, dim=64, page=64,
             fmt="int8", dtype="bf16"),
        # long ragged prompts of a grouped-head model, odd page size, appended to cached prefixes
        dict(name="kv_ragged_e4m3", op="kv", batch=13, lo=301, hi=12000, past=777, mix=3, kv_heads=8, dim=128, page=48,
             fmt="e4m3", dtype="f16"),
        # a few short prompts: latency
        dict(name="prompt_few_short", op="prompt", batch=4, lo=1, hi=131, past=0, mix=4, heads=20, kv_heads=20, dim=64,
             dtype="bf16", causal=True),
        # AR prefill, 64 x 256 tokens, 20 heads
        dict(name="prompt_b64_t256", op="prompt", batch=64, lo=256, hi=256, past=0, mix=5, heads=20, kv_heads=20,
             dim=64, dtype="bf16", causal=True),
        # flow-matching frames, 64 x 760, hidden 512, every frame sees every frame
        dict(name="prompt_frames_b64_t760", op="prompt", batch=64, lo=760, hi=760, past=0, mix=6, heads=8, kv_heads=8,
             dim=64, dtype="f16", causal=False),
        # ragged packed prompts with grouped heads, each behind a prefix that is cached already
        dict(name="prompt_ragged_prefix", op="prompt", batch=11, lo=33, hi=5003, past=500, mix=7, heads=32, kv_heads=8,
             dim=128, dtype="bf16", causal=True),
        # one long document
        dict(name="prompt_long", op="prompt", batch=1, lo=16384, hi=16384, past=0, mix=8, heads=32, kv_heads=8,
             dim=128, dtype="bf16", causal=True),
        # one user, a short context: latency of a single token
        dict(name="decode_one_short", op="decode", batch=1, lo=300, hi=300, mix=9, heads=20, kv_heads=20, dim=64,
             page=64, fmt="bf16", dtype="bf16"),
        # the AR model's decode step at batch 64, ragged contexts
        dict(name="decode_b64_e4m3", op="decode", batch=64, lo=256, hi=2048, mix=10, heads=20, kv_heads=20, dim=64,
             page=64, fmt="e4m3", dtype="bf16"),
        # grouped heads, 16-bit cache, odd pages, among them sequences that have ended (length 0)
        dict(name="decode_grouped_f16", op="decode", batch=37, lo=0, hi=6000, mix=11, heads=32, kv_heads=8, dim=128,
             page=48, fmt="f16", dtype="f16"),
        # two very long contexts: the cache's length is split over the whole card
        dict(name="decode_long_int8", op="decode", batch=2, lo=90001, hi=131072, mix=12, heads=32, kv_heads=8, dim=128,
             page=64, fmt="int8", dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        case = _draw(rng)
        cost = work(case)
        if cost["bytes"] <= 500e6 and cost["flops"] <= 2e12:
            return case


def _draw(rng):
    op = rng.choice(["kv", "prompt", "decode"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 5, 8, 20])
    group = rng.choice([1, 2, 4, 7, 8]) if kv_heads <= 8 else 1
    mix = rng.randrange(1 << 20)
    if op == "kv":
        tokens = _log_int(rng, 1, 60000)
        batch = _log_int(rng, 1, min(tokens, 128))
        per = max(1, tokens // batch)
        return dict(op=op, batch=batch, lo=rng.choice([1, per]), hi=per, past=rng.choice([0, 5, 1000]), mix=mix,
                    kv_heads=kv_heads, dim=dim, page=rng.choice([16, 48, 64, 128]),
                    fmt=rng.choice(["e4m3", "int8", "bf16"]), dtype=rng.choice(["bf16", "f16", "f32"]))
    if op == "prompt":
        hi = _log_int(rng, 1, 12000)
        batch = _log_int(rng, 1, max(1, min(96, 40000 // hi)))
        return dict(op=op, batch=batch, lo=rng.choice([1, hi]), hi=hi, past=rng.choice([0, 0, 129, 1000]), mix=mix,
                    heads=kv_heads * group, kv_heads=kv_heads, dim=dim, dtype=rng.choice(["bf16", "f16"]),
                    causal=rng.random() < 0.8)
    hi = _log_int(rng, 1, 130000)
    batch = _log_int(rng, 1, max(1, min(192, 200000 // hi)))
    fmt = rng.choice(["e4m3", "int8", "16"])
    dtype = rng.choice(["bf16", "f16"])
    return dict(op=op, batch=batch, lo=rng.choice([0, 1, hi]), hi=hi, mix=mix, heads=kv_heads * group,
                kv_heads=kv_heads, dim=dim, page=rng.choice([16, 48, 64, 128]), fmt=dtype if fmt == "16" else fmt,
                dtype=dtype)


def _lengths(case):
    """One length per sequence, spread over the logarithm of [lo, hi]; lo = 0 makes every fifth sequence empty."""
    rng = random.Random(case["mix"])
    lo, hi = case["lo"], case["hi"]
    out = []
    for i in range(case["batch"]):
        n = hi if lo == hi or i == case["batch"] // 2 else _log_int(rng, max(lo, 1), max(hi, 1))
        out.append(0 if lo == 0 and i % 5 == 4 else n)
    return out


def _pasts(case):
    """Cached tokens before the new ones of each sequence."""
    rng = random.Random(case["mix"] + 1)
    return [rng.randint(0, case["past"]) if case["past"] else 0 for _ in range(case["batch"])]


def work(case):
    lens, dim = _lengths(case), case["dim"]
    if case["op"] == "kv":
        rows = 2 * sum(lens) * case["kv_heads"]                  # K and V rows
        item = _DTYPE[case["dtype"]].itemsize
        code = 1 if case["fmt"] in _QMAX else 2
        scale = 4 if case["fmt"] in _QMAX else 0
        # the rows are read, their codes and scales written, read back and written out in the input's type
        return {"bytes": rows * (2 * dim * item + 2 * (dim * code + scale)), "flops": rows * dim * 4}
    if case["op"] == "prompt":
        seen = 0
        for n, past in zip(lens, _pasts(case)):
            seen += n * past + (n * (n + 1) // 2 if case["causal"] else n * n)
        rows = sum(lens)
        keys = rows + sum(_pasts(case))
        return {"bytes": 2 * dim * (2 * rows * case["heads"] + 2 * keys * case["kv_heads"]),
                "flops": 4 * dim * case["heads"] * seen}
    keys = sum(lens)
    per = 2 * dim * (1 if case["fmt"] in _QMAX else 2) + (8 if case["fmt"] in _QMAX else 0)
    return {"bytes": keys * case["kv_heads"] * per + 4 * dim * case["heads"] * case["batch"],
            "flops": 4 * dim * case["heads"] * keys}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=_device())


def _cumulative(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _pages_for(totals, page, mix):
    """A page table whose pages lie in the pool in random order, and the pool's number of pages."""
    need = [(n + page - 1) // page for n in totals]
    width = max(1, max(need))
    order = list(range(sum(need) + 1))
    random.Random(mix + 2).shuffle(order)
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (width - n))
        at += n
    return _ints(table), sum(need) + 1


def _codes(x, fmt):
    """Per-row codes of x [..., dim] and their FP32 scales, in elementary operations."""
    x = x.float()
    top = x.abs().amax(-1)
    scale = torch.clamp(top / torch.full_like(top, _QMAX[fmt]), min=1e-12)   # a quotient, not a product with 1 / max
    y = x / scale[..., None]
    if fmt == "int8":
        return torch.clamp(torch.round(y), -127, 127).to(torch.int8), scale
    return torch.clamp(y, -448, 448).to(torch.float8_e4m3fn), scale


def _inputs(case, seed):
    device = _device()
    g = torch.Generator(device=device).manual_seed(seed)
    lens, dim = _lengths(case), case["dim"]
    dtype = _DTYPE[case["dtype"]]

    def rows(n, heads, gain=1.0):
        # a few channels are larger than the rest, as the keys and values of trained models have them
        x = torch.randn(n, heads, dim, device=device, generator=g)
        x *= gain * (1.0 + 3.0 * (torch.rand(heads, dim, device=device, generator=g) < 0.04))
        return x.to(dtype)

    if case["op"] == "kv":
        totals = [a + b for a, b in zip(lens, _pasts(case))]
        table, pages = _pages_for(totals, case["page"], case["mix"])
        return dict(case=case, k=rows(sum(lens), case["kv_heads"]), v=rows(sum(lens), case["kv_heads"]), table=table,
                    pages=pages, lengths=_ints(totals), cu=_ints(_cumulative(lens)), lens=lens, totals=totals)
    if case["op"] == "prompt":
        keys = [a + b for a, b in zip(lens, _pasts(case))]
        return dict(case=case, q=rows(sum(lens), case["heads"], 1.5), k=rows(sum(keys), case["kv_heads"]),
                    v=rows(sum(keys), case["kv_heads"]), cu=_ints(_cumulative(lens)), cu_k=_ints(_cumulative(keys)),
                    lens=lens, keys=keys)
    table, pages = _pages_for(lens, case["page"], case["mix"])
    q = rows(case["batch"], case["heads"], 1.5)
    shape = (pages, case["kv_heads"], case["page"], dim)
    pool = {}
    for name in ("k", "v"):
        x = torch.randn(shape, device=device, generator=g)
        x *= 1.0 + 3.0 * (torch.rand(case["kv_heads"], 1, dim, device=device, generator=g) < 0.04)
        if case["fmt"] in _QMAX:
            pool[name], pool[name + "_scale"] = _codes(x, case["fmt"])
        else:
            pool[name], pool[name + "_scale"] = x.to(_DTYPE[case["fmt"]]), None
    return dict(case=case, q=q, table=table, pages=pages, lengths=_ints(lens), lens=lens, **pool)


def prepare(case, seed):
    state = _inputs(case, seed)
    if case["op"] == "kv":
        shape = (state["pages"], case["kv_heads"], case["page"], case["dim"])
        if case["fmt"] in _QMAX:
            code = torch.int8 if case["fmt"] == "int8" else torch.float8_e4m3fn
            for name in ("k_pool", "v_pool"):
                state[name] = torch.zeros(shape, device=_device(), dtype=torch.uint8).view(code)
                state[name + "_scale"] = torch.zeros(shape[:3], device=_device())
        else:
            for name in ("k_pool", "v_pool"):
                state[name] = torch.zeros(shape, device=_device(), dtype=_DTYPE[case["fmt"]])
                state[name + "_scale"] = None
    if own and case["op"] != "prompt":
        from inspark_proper_format_b200 import attention, kv_cache
        if case["op"] == "kv":
            state["cache"] = kv_cache.PagedKVCache.from_tensors(state["k_pool"], state["v_pool"],
                                                                state["k_pool_scale"], state["v_pool_scale"])
        else:
            state["cache"] = kv_cache.PagedKVCache.from_tensors(state["k"], state["v"], state["k_scale"],
                                                                state["v_scale"])
            state["workspace"] = attention.DecodeWorkspace(state["q"].device)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        from inspark_proper_format_b200 import attention, kv_cache
        if case["op"] == "kv":
            kv_cache.kv_append(state["cache"], state["k"], state["v"], state["table"], state["lengths"], state["cu"])
            return kv_cache.kv_gather(state["cache"], state["table"], state["lengths"], state["cu"],
                                      tokens=state["k"].shape[0], dtype=state["k"].dtype)
        if case["op"] == "prompt":
            return attention.prompt_attention(state["q"], state["k"], state["v"], state["cu"],
                                              cu_seqlens_k=state["cu_k"], causal=case["causal"])
        return attention.paged_decode_attention(state["q"], state["cache"], state["table"], state["lengths"],
                                                workspace=state["workspace"])
    return {"kv": _plain_kv, "prompt": _plain_prompt, "decode": _plain_decode}[case["op"]](state)


def _plain_kv(state):
    """Positions, pages and rows by indexing; codes as the values they stand for when read back."""
    case = state["case"]
    cu, lengths, page = state["cu"].long(), state["lengths"].long(), case["page"]
    token = torch.arange(state["k"].shape[0], device=cu.device)
    seq = torch.searchsorted(cu[1:], token, right=True)
    pos = token - cu[seq] + lengths[seq] - (cu[seq + 1] - cu[seq])
    slot, off = state["table"].long()[seq, pos // page], pos % page
    out = []
    for name in ("k", "v"):
        pool, scales = state[name + "_pool"], state[name + "_pool_scale"]
        if scales is None:
            pool[slot, :, off] = state[name].to(pool.dtype)
            back = pool[slot, :, off].float()
        else:
            codes, s = _codes(state[name], case["fmt"])
            pool.view(torch.uint8)[slot, :, off] = codes.view(torch.uint8)
            scales[slot, :, off] = s
            back = pool.view(torch.uint8)[slot, :, off].view(pool.dtype).float() * scales[slot, :, off][..., None]
        out.append(back.to(state[name].dtype))
    return tuple(out)


def _plain_softmax_product(scores, v):
    """Rows of scores (masked places hold -inf) times v; a row without a visible key gives zeros."""
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_prompt(state):
    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    group = case["heads"] // case["kv_heads"]
    out = torch.empty_like(q)
    a = b = 0
    for n, m in zip(state["lens"], state["keys"]):
        hidden = None
        if case["causal"]:
            hidden = torch.arange(m, device=q.device)[None, :] > torch.arange(n, device=q.device)[:, None] + (m - n)
        step = max(1, (1 << 29) // max(1, group * n * m))        # key-value heads at once
        for h in range(0, case["kv_heads"], step):
            e = min(case["kv_heads"], h + step)
            qs = q[a:a + n, h * group:e * group].float().transpose(0, 1).reshape(e - h, group, n, -1)
            ks = k[b:b + m, h:e].float().transpose(0, 1)[:, None]
            vs = v[b:b + m, h:e].float().transpose(0, 1)[:, None]
            scores = torch.matmul(qs, ks.transpose(-1, -2)) * (1.0 / math.sqrt(case["dim"]))
            if hidden is not None:
                scores = scores.masked_fill_(hidden, -math.inf)
            o = _plain_softmax_product(scores, vs)
            out[a:a + n, h * group:e * group] = o.reshape((e - h) * group, n, -1).transpose(0, 1).to(q.dtype)
        a, b = a + n, b + m
    return out


def _plain_decode(state):
    case = state["case"]
    q, page = state["q"], case["page"]
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros_like(q)
    for b, n in enumerate(state["lens"]):
        if n == 0:
            continue
        ids = state["table"][b, :(n + page - 1) // page].long()
        kv = []
        for name in ("k", "v"):
            pool = state[name]
            x = pool.view(torch.uint8)[ids].view(pool.dtype) if pool.element_size() == 1 else pool[ids]
            x = x.float()
            if state[name + "_scale"] is not None:
                x = x * state[name + "_scale"][ids][..., None]
            kv.append(x.transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :n])
        qs = q[b].float().reshape(case["kv_heads"], group, -1)
        scores = torch.matmul(qs, kv[0].transpose(-1, -2)) * (1.0 / math.sqrt(case["dim"]))
        out[b] = _plain_softmax_product(scores, kv[1]).reshape(case["heads"], -1).to(q.dtype)
    return out


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    state = _inputs(case, seed)
    if case["op"] == "kv":
        return tuple(_exact_read_back(state[name].double(), case["fmt"]) for name in ("k", "v"))
    heads = [h // (case["heads"] // case["kv_heads"]) for h in range(case["heads"])]
    q = state["q"].double() / case["dim"] ** 0.5
    out = torch.zeros_like(q)
    if case["op"] == "prompt":
        first_q, first_k = _cumulative(state["lens"]), _cumulative(state["keys"])
        for i, (n, m) in enumerate(zip(state["lens"], state["keys"])):
            at_once = max(1, (1 << 28) // max(1, n * m))
            for j in range(0, case["heads"], at_once):
                hs = list(range(j, min(case["heads"], j + at_once)))
                x = q[first_q[i]:first_q[i + 1], hs]
                kk = state["k"][first_k[i]:first_k[i + 1]][:, [heads[h] for h in hs]].double()
                vv = state["v"][first_k[i]:first_k[i + 1]][:, [heads[h] for h in hs]].double()
                s = torch.einsum("qhd,khd->hqk", x, kk)
                if case["causal"]:
                    s += torch.full((n, m), -math.inf, device=s.device, dtype=s.dtype).triu(m - n + 1)
                out[first_q[i]:first_q[i + 1], hs] = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), vv)
        return out
    page = case["page"]
    for b, n in enumerate(state["lens"]):
        if n == 0:
            continue
        pos = torch.arange(n, device=q.device)
        ids, off = state["table"][b].long()[pos // page], pos % page
        k, v = (_stands_for(state[name], state[name + "_scale"], ids, off) for name in ("k", "v"))   # [n, kv_heads, dim]
        for h in range(case["kv_heads"]):
            mine = [j for j in range(case["heads"]) if heads[j] == h]
            w = torch.softmax(q[b, mine] @ k[:, h].T, -1)
            out[b, mine] = w @ v[:, h]
    return out


def _stands_for(pool, scale, ids, off):
    if scale is None:
        return pool[ids, :, off].double()
    raw = pool.view(torch.uint8)[ids, :, off].long()
    if pool.dtype == torch.int8:
        value = torch.where(raw > 127, raw - 256, raw).double()
    else:
        exponent, mantissa = (raw >> 3) & 15, (raw & 7).double()
        size = torch.where(exponent == 0, mantissa / 8 * 2.0 ** -6,
                           (1 + mantissa / 8) * torch.exp2((exponent - 7).double()))
        value = torch.where(raw > 127, -size, size)
    return value * scale[ids, :, off].double()[..., None]


def _exact_read_back(x, fmt):
    """The value that the code of each element stands for; scale and quotient are FP32 numbers by definition."""
    if fmt not in _QMAX:
        return x.to(_DTYPE[fmt]).double()
    scale = (x.abs().amax(-1, keepdim=True) / _QMAX[fmt]).clamp_min(1e-12).float().double()
    y = (x / scale).float().double()
    if fmt == "int8":
        return y.round().clamp(-127, 127) * scale
    # 3 bits behind the leading one, exponents from -6 up, ties to even, at most 448
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return ((y / step).round() * step).clamp(-448, 448) * scale
