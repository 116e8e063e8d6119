"""Timed cases of the paged-cache serving operators: a cache of pages with the attention that reads it, and the attention
of packed prompts that fills it.

Three operators, each with its plain form (elementary torch operations in 32 bits, rounded once at the end), the
framework's kernels (``own``) and its definition in 64 bits (``exact``):

* ``append``  RoPE of new tokens' q and k, their k and v written into the cache's pages (bf16 / fp32 pages, or 8-bit
  floating-point codes with one power-of-two scale per token and head), and the pages read back as packed rows;
* ``paged``   attention of each sequence's newest token(s) over its pages;
* ``packed``  causal attention of packed prompts of different lengths (or new chunks of prompts whose earlier keys
  are given too), grouped heads.

The 8-bit form of a vector x (one token of one head): e = the smallest integer with max|x| <= 448 * 2^e, held to
[-40, 40]; the codes are x * 2^-e rounded to e4m3, the scale byte is e + 127.
"""

import random

import torch

own = False

MAX_COST = 1.1e12  # flops of the largest listed case: a drawn one costs no more
MAX_PLAIN = 2.3e9  # scores the plain form of a drawn packed case may hold at once


# ----------------------------------------------------------------------------------------------------------------
# cases

def listed():
    return [
        # One stream's speculative step: a draft of 4 tokens and the newest, 32 heads x 128, about 700 keys (latency).
        {"name": "paged_verify_one", "op": "paged", "rows": 1, "tokens": 5, "heads": 32, "kv_heads": 32, "dim": 128,
         "page": 64, "lo": 700, "hi": 700, "dtype": "bf16", "cache": "bf16"},
        # A serving batch's decode step with grouped heads, prompts and answers of all lengths.
        {"name": "paged_batch", "op": "paged", "rows": 48, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "lo": 61, "hi": 4093, "dtype": "bf16", "cache": "bf16"},
        # The shipped decoder's head geometry, a full batch on 30 s of audio each, 8-bit cache.
        {"name": "paged_wide_fp8", "op": "paged", "rows": 32, "tokens": 1, "heads": 8, "kv_heads": 8, "dim": 512,
         "page": 64, "lo": 1400, "hi": 1600, "dtype": "bf16", "cache": "fp8"},
        # A few very long contexts, 8-bit cache: the cache is all that counts.
        {"name": "paged_long_fp8", "op": "paged", "rows": 4, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "lo": 60001, "hi": 131072, "dtype": "bf16", "cache": "fp8"},
        # An fp32 model's short prompts, odd lengths, small heads.
        {"name": "packed_small_f32", "op": "packed", "seqs": 3, "heads": 8, "kv_heads": 4, "dim": 64, "lo": 17, "hi": 131,
         "past_lo": 0, "past_hi": 0, "dtype": "f32"},
        # A batch of prompts as they come.
        {"name": "packed_ragged", "op": "packed", "seqs": 12, "heads": 32, "kv_heads": 8, "dim": 128, "lo": 60, "hi": 2047,
         "past_lo": 0, "past_hi": 0, "dtype": "bf16"},
        # The shipped decoder's prefill: 8 prefixes of about 1500 positions, 8 heads x 512.
        {"name": "packed_wide", "op": "packed", "seqs": 8, "heads": 8, "kv_heads": 8, "dim": 512, "lo": 1400, "hi": 1500,
         "past_lo": 0, "past_hi": 0, "dtype": "bf16"},
        # A chunk of a long prompt against the keys of the chunks before it.
        {"name": "packed_chunk", "op": "packed", "seqs": 1, "heads": 32, "kv_heads": 8, "dim": 128, "lo": 2048, "hi": 2048,
         "past_lo": 29700, "past_hi": 29700, "dtype": "bf16"},
        # A decode step's append into a plain cache, one token of each of 64 sequences; their newest pages read back.
        {"name": "append_step", "op": "append", "seqs": 64, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "lo": 1, "hi": 1,
         "past_lo": 0, "past_hi": 2000, "dtype": "bf16", "cache": "bf16", "back": "page"},
        # The same into an 8-bit cache at the shipped geometry.
        {"name": "append_step_fp8", "op": "append", "seqs": 32, "heads": 8, "kv_heads": 8, "dim": 512, "page": 64, "lo": 1, "hi": 1,
         "past_lo": 1400, "past_hi": 1600, "dtype": "bf16", "cache": "fp8", "back": "page"},
        # A prompt chunk written to an 8-bit cache, and the whole context read back for the chunk's attention.
        {"name": "append_chunk_fp8", "op": "append", "seqs": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "lo": 2048,
         "hi": 2048, "past_lo": 29700, "past_hi": 29700, "dtype": "bf16", "cache": "fp8", "back": "all"},
        # A batch of prompts written to an 8-bit cache.
        {"name": "append_prompts_fp8", "op": "append", "seqs": 12, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "lo": 60,
         "hi": 2047, "past_lo": 0, "past_hi": 0, "dtype": "bf16", "cache": "fp8", "back": "all"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], its logarithm spread evenly."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _heads(rng, dim):
    kv = rng.choice([1, 2, 4, 8]) if dim >= 256 else rng.choice([1, 2, 4, 8, 16, 32])
    group = rng.choice([1, 1, 2, 3, 4, 8]) if kv <= 8 else rng.choice([1, 2])
    return kv * group, kv


def draw(rng):
    op = rng.choice(["paged", "packed", "append"])
    while True:
        dtype = "f32" if rng.random() < 0.15 else "bf16"
        dim = rng.choice([16, 32, 64, 128, 256]) if dtype == "f32" else rng.choice([64, 128, 128, 128, 128, 256, 512, 512])
        heads, kv = _heads(rng, dim)
        c = {"op": op, "heads": heads, "kv_heads": kv, "dim": dim, "dtype": dtype}
        if op == "paged":
            hi = _log(rng, 1, 131072)
            c |= {"rows": _log(rng, 1, 256), "tokens": rng.choice([1, 1, 1, 1, 2, 5, 8]), "page": rng.choice([8, 16, 16, 32, 64, 128]),
                  "lo": rng.randint(0, hi), "hi": hi, "cache": rng.choice([dtype, "fp8"])}
            keys = sum(_spread(c["lo"], c["hi"], c["rows"]))
            if c["rows"] * c["hi"] * kv * dim > 1.0e9 or keys * heads * c["tokens"] > 2e8:
                continue  # the plain form holds every key in 32 bits
            if dtype == "f32" and keys * kv * dim > 6e7:
                continue
        else:
            past = op == "append" or rng.random() < 0.4
            hi = _log(rng, 1, 8192)
            c |= {"seqs": _log(rng, 1, 64), "lo": rng.randint(1, hi), "hi": hi, "past_hi": _log(rng, 1, 30000) if past else 0}
            c["past_lo"] = rng.randint(0, c["past_hi"])
            if op == "append":
                c |= {"page": rng.choice([8, 16, 16, 32, 64, 128]), "cache": rng.choice([dtype, "fp8"]),
                      "back": rng.choice(["page", "all"]) if c["seqs"] * c["hi"] < 2048 else "all"}
                if c["seqs"] * ((c["hi"] + c["past_hi"]) * kv + c["hi"] * heads) * dim > 2.5e8:
                    continue
            else:
                if c["seqs"] * heads * c["hi"] * (c["hi"] + c["past_hi"]) > MAX_PLAIN or work(c)["flops"] > MAX_COST:
                    continue
                if dtype == "f32" and work(c)["flops"] > 3e10:
                    continue
        return c


def _spread(lo, hi, n):
    """n lengths of [lo, hi], the ends among them, in no order."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * 7 + 3) % n) // (n - 1) if n % 7 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(case, seed):
    """(new, past) lengths per sequence: the case's, in an order of the seed."""
    r = random.Random("%s lengths" % seed)
    new = _spread(case["lo"], case["hi"], case["seqs"])
    past = _spread(case["past_lo"], case["past_hi"], case["seqs"])
    both = list(zip(new, past))
    r.shuffle(both)
    return [n for n, _ in both], [p for _, p in both]


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "paged":
        t = case["tokens"]
        lens = _spread(case["lo"], case["hi"], case["rows"])
        read = sum(n + t - 1 for n in lens if n + t - 1 > 0)
        pairs = sum(max(0, n + i) for n in lens for i in range(t))
        vec = d + 1 if case["cache"] == "fp8" else d * e
        return {"bytes": read * kv * vec * 2 + 2 * case["rows"] * t * h * d * e + 4 * sum(-(-n // case["page"]) for n in lens),
                "flops": 4 * pairs * h * d}
    new, past = _lengths(case, 0)
    if case["op"] == "packed":
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
        return {"bytes": (2 * sum(new) * h + 2 * (sum(new) + sum(past)) * kv) * d * e, "flops": 4 * pairs * h * d}
    vec = d + 1 if case["cache"] == "fp8" else d * e
    back = sum(_back(case, n, p) for n, p in zip(new, past))
    return {"bytes": sum(new) * ((2 * h + 2 * kv) * d * e + 4 * d + 2 * kv * vec) + 2 * back * kv * (vec + d * e),
            "flops": 6 * sum(new) * (h + kv) * d}


def _back(case, new, past):
    """Tokens read back of a sequence: all, or those of its newest page."""
    n = new + past
    return n if case["back"] == "all" else (n - 1) % case["page"] + 1


# ----------------------------------------------------------------------------------------------------------------
# inputs

_TORCH = {"bf16": torch.bfloat16, "f32": torch.float32}


def _quantise(x):
    """(codes, scale bytes) of the vectors x [..., dim] (fp32)."""
    m, k = torch.frexp(x.abs().amax(-1))
    e = torch.where(m <= 0.875, k - 9, k - 8).clamp(-40, 40)
    codes = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _values(codes, scale):
    return torch.ldexp(codes.float(), scale[..., None].int() - 127)


def _randn(gen, shape, dtype, dim):
    """Normal values with channels of different sizes, as projections have them."""
    size = torch.exp(0.4 * torch.randn(dim, generator=gen, device="cuda"))
    return (torch.randn(*shape, dim, generator=gen, device="cuda") * size).to(dtype)


def _pool(case, gen, pages):
    """K and V pages [pages, kv_heads, page, dim] (and their scale bytes)."""
    out = []
    for _ in range(2):
        x = _randn(gen, (pages, case["kv_heads"], case["page"]), _TORCH[case["dtype"]], case["dim"])
        if case["cache"] == "fp8":
            out.append(_quantise(x.float()))
        else:
            out.append((x, None))
    return out


def _table(counts, gen, spare):
    """A page table for sequences of `counts` pages, the pages in any order in a pool with `spare` more."""
    total = sum(counts) + spare
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    width = max(1, max(counts))
    start = torch.tensor([sum(counts[:i]) for i in range(len(counts))], device="cuda")
    count = torch.tensor(counts, device="cuda")
    i = torch.arange(width, device="cuda")
    at = (start[:, None] + i).clamp(max=total - 1)
    return torch.where(i < count[:, None], order[at], torch.zeros_like(order[at])), total


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 60))
    h, kv, d, dtype = case["heads"], case["kv_heads"], case["dim"], _TORCH[case["dtype"]]
    s = {"case": case, "scale": d**-0.5}
    if case["op"] == "paged":
        lens = _spread(case["lo"], case["hi"], case["rows"])
        random.Random("%s lengths" % seed).shuffle(lens)
        t = case["tokens"]
        counts = [-(-(n + t - 1) // case["page"]) for n in lens]
        s["table"], pages = _table(counts, gen, 3)
        (s["k"], s["k_scale"]), (s["v"], s["v_scale"]) = _pool(case, gen, pages)
        s["lengths"] = torch.tensor(lens, device="cuda")
        s["q"] = _randn(gen, (case["rows"] * t, h), dtype, d)
        return s
    new, past = _lengths(case, seed)
    offsets = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], device="cuda")  # noqa: E731
    s["q_offsets"] = offsets(new)
    if case["op"] == "packed":
        both = [n + p for n, p in zip(new, past)]
        s["k_offsets"] = offsets(both)
        s["most"] = (max(new), max(both))
        s["q"] = _randn(gen, (sum(new), h), dtype, d)
        s["k"] = _randn(gen, (sum(both), kv), dtype, d)
        s["v"] = _randn(gen, (sum(both), kv), dtype, d)
        return s
    page = case["page"]
    counts = [-(-(n + p) // page) for n, p in zip(new, past)]
    table, pages = _table(counts, gen, 3)
    (s["k"], s["k_scale"]), (s["v"], s["v_scale"]) = _pool(case, gen, pages)
    s["qkv"] = _randn(gen, (sum(new), h + 2 * kv), dtype, d).reshape(sum(new), -1)
    pos = torch.cat([torch.arange(p, n + p, device="cuda") for n, p in zip(new, past)])
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
    s["pos"] = pos
    s["slots"] = table[seq, pos // page].long() * page + pos % page
    freq = 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    angle = torch.arange(max(n + p for n, p in zip(new, past)), device="cuda", dtype=torch.float64)[:, None] * freq
    s["cs"] = torch.stack([angle.cos(), angle.sin()], -1).float()
    s["table"] = table if case["back"] == "all" else table.gather(1, torch.tensor(counts, device="cuda")[:, None] - 1)
    back = [_back(case, n, p) for n, p in zip(new, past)]
    s["back"], s["back_tokens"] = offsets(back), sum(back)
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ----------------------------------------------------------------------------------------------------------------
# one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"paged": _own_paged, "packed": _own_packed, "append": _own_append}[op](state)
    return {"paged": _plain_paged, "packed": _plain_packed, "append": _plain_append}[op](state)


_kernels = None


def _own():
    """The framework's kernel module."""
    global _kernels
    if _kernels is None:
        import os
        import sys

        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "omniasr-trt_b200"))
        from omniasr_b200 import kernels

        _kernels = kernels
    return _kernels


def _own_paged(s):
    return _own().paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["scale"],
                                  tokens=s["case"]["tokens"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_packed(s):
    return _own().packed_attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], s["scale"])


def _own_append(s):
    k = _own()
    q = k.paged_rope_kv(s["qkv"], s["cs"], s["pos"], s["k"], s["v"], s["slots"], s["case"]["heads"],
                        s["case"]["kv_heads"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    back = k.paged_kv_read(s["k"], s["v"], s["table"], s["back"], s["back_tokens"], k_scale=s["k_scale"],
                           v_scale=s["v_scale"], dtype=s["qkv"].dtype)
    return q, back[0], back[1]


def _masked_softmax(x, seen):
    """Softmax over the last axis of the scores that are seen; a row that sees none gives zeros."""
    x = x.masked_fill(~seen, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _gathered(pages, scale, table):
    """A table's pages as rows [rows, kv_heads, keys, dim] in 32 bits."""
    x = pages.view(torch.uint8)[table.long()].view(pages.dtype) if scale is not None else pages[table.long()]
    x = x.float() if scale is None else _values(x, scale[table.long()])
    b, w, kv, page, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, kv, w * page, d)


def _plain_paged(s):
    c = s["case"]
    t, kv, d = c["tokens"], c["kv_heads"], c["dim"]
    g = c["heads"] // kv
    k, v = _gathered(s["k"], s["k_scale"], s["table"]), _gathered(s["v"], s["v_scale"], s["table"])
    b, keys = k.size(0), k.size(2)
    q = s["q"].float().view(b, t, kv, g, d).permute(0, 2, 1, 3, 4).reshape(b, kv, t * g, d)
    x = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    limit = s["lengths"][:, None] + torch.arange(t, device=q.device)  # keys each query sees
    seen = torch.arange(keys, device=q.device) < limit[:, :, None, None]
    p = _masked_softmax(x, seen.expand(b, t, g, keys).reshape(b, 1, t * g, keys))
    o = torch.matmul(p, v)
    return o.view(b, kv, t, g, d).permute(0, 2, 1, 3, 4).reshape(b * t, c["heads"], d).to(s["q"].dtype)


def _plain_packed(s):
    c = s["case"]
    kv, d = c["kv_heads"], c["dim"]
    g = c["heads"] // kv
    nq, nk = s["most"]
    qo, ko = s["q_offsets"], s["k_offsets"]
    lq, lk = qo.diff(), ko.diff()
    n = lq.numel()
    qi, ki = torch.arange(nq, device=qo.device), torch.arange(nk, device=qo.device)
    q_at = (qo[:-1, None] + qi).clamp(max=s["q"].size(0) - 1)
    k_at = (ko[:-1, None] + ki).clamp(max=s["k"].size(0) - 1)
    q = s["q"].float()[q_at].view(n, nq, kv, g, d).permute(0, 2, 3, 1, 4).reshape(n, kv, g * nq, d)
    k = s["k"].float()[k_at].permute(0, 2, 1, 3)
    v = s["v"].float()[k_at].permute(0, 2, 1, 3)
    x = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).view(n, kv, g, nq, nk)
    limit = (lk - lq)[:, None] + qi + 1  # keys each query sees
    p = _masked_softmax(x, (ki < limit[:, :, None])[:, None, None])
    o = torch.matmul(p.view(n, kv, g * nq, nk), v).view(n, kv, g, nq, d)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, nq, c["heads"], d)
    return o[qi < lq[:, None]].to(s["q"].dtype)


def _rotate(x, cs):
    """Interleaved pairs of x [tokens, heads, dim] turned by cs [tokens, dim / 2, 2]."""
    re, im = x[..., 0::2], x[..., 1::2]
    co, si = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.stack([re * co - im * si, re * si + im * co], -1).flatten(-2)


def _plain_append(s):
    c = s["case"]
    h, kv, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    dtype = s["qkv"].dtype
    n = s["qkv"].size(0)
    x = s["qkv"].view(n, h + 2 * kv, d)
    turned = _rotate(x[:, : h + kv].float(), s["cs"][s["pos"]]).to(dtype)
    at, off = s["slots"] // page, s["slots"] % page
    out = []
    for pages, scale, rows in ((s["k"], s["k_scale"], turned[:, h:]), (s["v"], s["v_scale"], x[:, h + kv:])):
        if scale is None:
            pages[at, :, off] = rows
        else:
            codes, e = _quantise(rows.float())
            pages.view(torch.uint8)[at, :, off] = codes.view(torch.uint8)
            scale[at, :, off] = e
        i = torch.arange(s["back_tokens"], device=at.device)
        seq = torch.searchsorted(s["back"], i, right=True) - 1
        j = i - s["back"][seq]
        src, o = s["table"][seq, j // page].long(), j % page
        if scale is None:
            out.append(pages[src, :, o])
        else:
            out.append(_values(pages.view(torch.uint8)[src, :, o].view(pages.dtype), scale[src, :, o]).to(dtype))
    return turned[:, :h].contiguous(), out[0], out[1]


# ----------------------------------------------------------------------------------------------------------------
# the definition in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    g = h // kv
    if case["op"] == "append":
        return _exact_append(s)
    q = s["q"].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    if case["op"] == "packed":
        qo, ko = s["q_offsets"].tolist(), s["k_offsets"].tolist()
        for a, b, u, w in zip(qo, qo[1:], ko, ko[1:]):
            for j in range(kv):
                k, v = s["k"][u:w, j].double(), s["v"][u:w, j].double()
                limit = torch.arange(b - a, device=q.device) + (w - u) - (b - a) + 1
                for i in range(g):
                    out[a:b, j * g + i] = _exact_rows(q[a:b, j * g + i], k, v, limit, s["scale"])
        return out
    t = case["tokens"]
    for r, n in enumerate(s["lengths"].tolist()):
        n += t - 1
        ids = s["table"][r, : -(-n // case["page"])].long()
        limit = n - t + 1 + torch.arange(t, device=q.device)
        for j in range(kv):
            k, v = (_exact_cache(s, name, ids, j)[:n] for name in ("k", "v"))
            for i in range(g):
                out[r * t:(r + 1) * t, j * g + i] = _exact_rows(q[r * t:(r + 1) * t, j * g + i], k, v, limit, s["scale"])
    return out


def _exact_rows(q, k, v, limit, scale):
    """Attention of rows q over the first limit[i] of the keys k."""
    if not k.size(0):
        return torch.zeros_like(q)
    x = q @ k.t() * scale
    hidden = torch.arange(k.size(0), device=q.device) >= limit[:, None]
    x[hidden] = float("-inf")
    p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
    return p @ v


def _exact_cache(s, name, ids, head):
    """One head's rows of the pages `ids`, as the numbers they stand for."""
    x, e = s[name], s[name + "_scale"]
    if e is None:
        return x[ids, head].double().flatten(0, 1)
    codes = x.view(torch.uint8)[ids, head].view(x.dtype).float().double()
    return (codes * 2.0 ** (e[ids, head].double() - 127.0)[..., None]).flatten(0, 1)


def _exact_append(s):
    """q and the cache's rows as they are before any rounding: the new tokens' own numbers, the earlier tokens' as the
    cache held them."""
    c = s["case"]
    h, kv, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    x = s["qkv"].double().view(-1, h + 2 * kv, d)
    z = torch.view_as_complex(x[:, : h + kv].unflatten(-1, (d // 2, 2)).contiguous())
    turn = torch.view_as_complex(s["cs"].double()[s["pos"]])
    turned = torch.view_as_real(z * turn[:, None]).flatten(-2)
    out = [turned[:, :h]]
    for name, rows in (("k", turned[:, h:]), ("v", x[:, h + kv:])):
        rest = s[name].double() if s[name + "_scale"] is None else \
            s[name].float().double() * 2.0 ** (s[name + "_scale"].double() - 127.0)[..., None]
        flat = rest.permute(0, 2, 1, 3).reshape(-1, kv, d)
        flat[s["slots"]] = rows
        ends = s["back"].tolist()
        parts = []
        for i, (a, b) in enumerate(zip(ends, ends[1:])):
            j = torch.arange(b - a, device=flat.device)
            parts.append(flat[s["table"][i].long()[j // page] * page + j % page])
        out.append(torch.cat(parts))
    return tuple(out)
