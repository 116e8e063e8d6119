"""Timed cases of a serving step in four bits: a paged cache whose keys and values take four bits, weights that do, queries and
keys normed per head before they are rotated, and page tables that are built on the GPU.

Five operators, each with its plain form (elementary torch operations in 32 bits, rounded once at the end), the framework's
kernels (``own``) and its definition in 64 bits (``exact``):

* ``attend``  attention of each sequence's newest token(s) over its 4-bit pages;
* ``append``  RoPE of new tokens' q and k, their k and v written into 4-bit pages, and the pages read back as packed rows;
* ``norm``    q and k normed per head, rotated, and k and v appended to the pages, in one pass;
* ``plan``    a step's positions, slots, block tables, lengths and offsets from the requests' lengths, with the pages that it takes
              from a stack of free ones, and the pages given back when the step is undone;
* ``gemm``    a few tokens times 4-bit weights with group scales.

The 4-bit form of 32 numbers x (a group of a vector's consecutive dims, as the model's type holds them): m the one of largest
magnitude (the negative one of two), s = -m / 8 rounded to bf16, the codes c = x / s rounded to a whole number of [-8, 7] plus
8 (8 where s is 0); the value is s (c - 8). A weight's group is longer and its scale is given.

Where a vector's codes lie, two to a byte, the low four bits first: with quads u = dim / 4, blocks of 32 quads, NG = the groups of
a block, group = u % 32 / 8 and i = u % 8, a quad of K lies at quad (i / 2 * NG + group) * 2 + i % 2 of its block, one of V at
i * NG + group.
"""

import random

import torch

own = False

MAX_KEYS = 5.4e8  # rows x longest x kv_heads x dim of the largest listed cache
MAX_BYTES, MAX_FLOPS = 4.4e8, 6.2e9  # of the largest listed case
MAX_NEW = 1.6e8  # numbers of the largest listed append


# ----------------------------------------------------------------------------------------------------------------
# cases

def listed():
    return [
        # One stream's speculative step: the newest token and a draft of 4, about 700 keys (latency).
        {"name": "attend_verify_one", "op": "attend", "rows": 1, "tokens": 5, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "lo": 700, "hi": 700, "dtype": "bf16"},
        # A serving batch's decode step with grouped heads, prompts and answers of all lengths.
        {"name": "attend_batch", "op": "attend", "rows": 48, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "lo": 61, "hi": 4093, "dtype": "bf16"},
        # The shipped decoder's head geometry, a full batch on 30 s of audio each.
        {"name": "attend_wide", "op": "attend", "rows": 32, "tokens": 1, "heads": 8, "kv_heads": 8, "dim": 512, "page": 64,
         "lo": 1400, "hi": 1600, "dtype": "bf16"},
        # A few very long contexts: the cache is all that counts.
        {"name": "attend_long", "op": "attend", "rows": 4, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "lo": 60001, "hi": 131072, "dtype": "bf16"},
        # A decode step's append at the shipped geometry, one token of each of 32 sequences; their newest pages read back.
        {"name": "append_step", "op": "append", "seqs": 32, "heads": 8, "kv_heads": 8, "dim": 512, "page": 64, "lo": 1, "hi": 1,
         "past_lo": 1400, "past_hi": 1600, "dtype": "bf16", "back": "page"},
        # A prompt chunk written, and the whole context read back for the chunk's attention.
        {"name": "append_chunk", "op": "append", "seqs": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "lo": 2048,
         "hi": 2048, "past_lo": 29700, "past_hi": 29700, "dtype": "bf16", "back": "all"},
        # A decode step of 64 sequences of a model that norms its queries and keys.
        {"name": "norm_step", "op": "norm", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "past": 2000,
         "dtype": "bf16"},
        # The prompts of a batch, together as many tokens.
        {"name": "norm_prompts", "op": "norm", "tokens": 12643, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "past": 0,
         "dtype": "bf16"},
        # A decode step's tables: one token of each of 64 sequences.
        {"name": "plan_step", "op": "plan", "requests": 64, "new_lo": 1, "new_hi": 1, "past_lo": 61, "past_hi": 4093, "page": 16,
         "spare": 200},
        # A step that mixes decode tokens and chunks of prompts, in pages of 64.
        {"name": "plan_mixed", "op": "plan", "requests": 256, "new_lo": 0, "new_hi": 512, "past_lo": 0, "past_hi": 8000,
         "page": 64, "spare": 3000},
        # One token through a square projection with the residual stream added (latency).
        {"name": "gemm_one", "op": "gemm", "rows": 1, "n": 4096, "k": 4096, "group": 128, "mode": "residual"},
        # Eight tokens through a feed-forward block's gate and inner product.
        {"name": "gemm_gate", "op": "gemm", "rows": 8, "n": 11008, "k": 4096, "group": 128, "mode": "swiglu"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], its logarithm spread evenly."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _heads(rng, dim):
    kv = rng.choice([1, 2, 4, 8]) if dim >= 256 else rng.choice([1, 2, 4, 8, 16, 32])
    group = rng.choice([1, 1, 2, 3, 4, 8]) if kv <= 8 else rng.choice([1, 2])
    return kv * group, kv


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "norm", "plan", "gemm"])
    while True:
        if op == "gemm":
            c = {"op": op, "rows": _log(rng, 1, 64), "n": _log(rng, 5, 11008), "k": 32 * _log(rng, 1, 344),
                 "group": rng.choice([32, 64, 128, 128]), "mode": rng.choice(["store", "residual", "swiglu"])}
            if c["rows"] * c["n"] * c["k"] * (2 if c["mode"] == "swiglu" else 1) > 8 * 2 * 11008 * 4096:
                continue
            return c
        if op == "plan":
            hi = _log(rng, 1, 512)
            c = {"op": op, "requests": _log(rng, 1, 256), "new_lo": rng.randint(0, hi), "new_hi": hi, "past_lo": 0,
                 "past_hi": _log(rng, 1, 8000), "page": rng.choice([8, 16, 16, 24, 32, 64, 128])}
            c["past_lo"] = rng.randint(0, c["past_hi"])
            # Some steps find fewer free pages than they want: the requests that do not fit are told so.
            c["spare"] = int(c["requests"] * (hi / c["page"] + 1) * rng.choice([0.2, 0.6, 1.0, 1.5])) + 1
            return c
        dtype = "f32" if rng.random() < 0.12 else "bf16"
        dim = rng.choice([32, 64, 128, 256]) if dtype == "f32" else rng.choice([64, 128, 128, 128, 256, 512, 512])
        heads, kv = _heads(rng, dim)
        c = {"op": op, "heads": heads, "kv_heads": kv, "dim": dim, "page": rng.choice([8, 16, 16, 32, 64, 128]), "dtype": dtype}
        if op == "attend":
            hi = _log(rng, 1, 131072)
            c |= {"rows": _log(rng, 1, 256), "tokens": rng.choice([1, 1, 1, 1, 2, 5, 8]), "lo": rng.randint(0, hi), "hi": hi}
            keys = sum(_spread(c["lo"], c["hi"], c["rows"]))
            if c["rows"] * hi * kv * dim > MAX_KEYS or work(c)["bytes"] > MAX_BYTES or work(c)["flops"] > MAX_FLOPS:
                continue  # the plain form holds every key in 32 bits
            if dtype == "f32" and keys * kv * dim > 6e7:
                continue
        elif op == "append":
            hi = _log(rng, 1, 8192)
            c |= {"seqs": _log(rng, 1, 64), "lo": rng.randint(1, hi), "hi": hi, "past_hi": _log(rng, 1, 30000)}
            c["past_lo"] = rng.randint(0, c["past_hi"])
            c["back"] = rng.choice(["page", "all"]) if c["seqs"] * hi < 2048 else "all"
            if c["seqs"] * ((hi + c["past_hi"]) * kv + hi * heads) * dim > MAX_NEW / 2:
                continue
        else:
            c |= {"tokens": _log(rng, 1, 12643), "past": _log(rng, 1, 8000)}
            if c["tokens"] * (heads + 2 * kv) * dim > 7.7e7:
                continue
        return c


def _spread(lo, hi, n):
    """n numbers of [lo, hi], the ends among them, in no order."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * ((i * 7 + 3) % n) // (n - 1) if n % 7 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(case, seed):
    """(new, past) lengths per sequence: the case's, in an order of the seed."""
    r = random.Random("%s lengths" % seed)
    both = list(zip(_spread(case["lo"], case["hi"], case["seqs"]), _spread(case["past_lo"], case["past_hi"], case["seqs"])))
    r.shuffle(both)
    return [n for n, _ in both], [p for _, p in both]


def _requests(case, seed):
    """(new, past) per request, each in an order of the seed."""
    r = random.Random("%s requests" % seed)
    new = _spread(case["new_lo"], case["new_hi"], case["requests"])
    past = _spread(case["past_lo"], case["past_hi"], case["requests"])
    r.shuffle(new)
    r.shuffle(past)
    return new, past


def _back(case, new, past):
    """Tokens read back of a sequence: all, or those of its newest page."""
    n = new + past
    return n if case["back"] == "all" else (n - 1) % case["page"] + 1


def work(case):
    if case["op"] == "gemm":
        n = case["n"] * (2 if case["mode"] == "swiglu" else 1)
        m, k = case["rows"], case["k"]
        res = m * case["n"] * 2 if case["mode"] == "residual" else 0
        return {"bytes": n * k // 2 + n * -(-k // case["group"]) * 2 + m * k * 2 + m * case["n"] * 2 + res, "flops": 2 * m * n * k}
    if case["op"] == "plan":
        new, past = _requests(case, 0)
        pages = sum(-(-(n + p) // case["page"]) for n, p in zip(new, past))
        take = sum(-(-(n + p) // case["page"]) - -(-p // case["page"]) for n, p in zip(new, past))
        # positions, slots and the batch's table written, its page numbers read, the pages taken and given back, each request's
        # numbers (number, new, past, kept, offsets, lengths)
        return {"bytes": 16 * sum(new) + 8 * pages + 16 * take + 72 * case["requests"], "flops": 4 * sum(new) + 8 * pages}
    e = 4 if case["dtype"] == "f32" else 2
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    four = d // 2 + d // 16  # a vector's codes and scales
    if case["op"] == "attend":
        t = case["tokens"]
        lens = _spread(case["lo"], case["hi"], case["rows"])
        read = sum(n + t - 1 for n in lens if n + t - 1 > 0)
        pairs = sum(max(0, n + i) for n in lens for i in range(t))
        return {"bytes": read * kv * four * 2 + 2 * case["rows"] * t * h * d * e + 4 * sum(-(-n // case["page"]) for n in lens),
                "flops": 4 * pairs * h * d}
    if case["op"] == "norm":
        n = case["tokens"]
        return {"bytes": n * ((2 * h + 4 * kv) * d * e + 4 * d + 16) + 2 * d * e, "flops": 10 * n * (h + kv) * d}
    new, past = _lengths(case, 0)
    back = sum(_back(case, n, p) for n, p in zip(new, past))
    return {"bytes": sum(new) * ((2 * h + 2 * kv) * d * e + 4 * d + 2 * kv * four) + 2 * back * kv * (four + d * e),
            "flops": 6 * sum(new) * (h + kv) * d + 4 * back * kv * d}


# ----------------------------------------------------------------------------------------------------------------
# inputs

_TORCH = {"bf16": torch.bfloat16, "f32": torch.float32}


def _randn(gen, shape, dtype, dim):
    """Normal values with channels of different sizes, as projections have them."""
    size = torch.exp(0.4 * torch.randn(dim, generator=gen, device="cuda"))
    return (torch.randn(*shape, dim, generator=gen, device="cuda") * size).to(dtype)


def _order(dim, keys):
    """Where dim d's code lies among a vector's."""
    d = torch.arange(dim, device="cuda")
    u = d // 4
    groups = min(4, dim // 32)
    group, i = u % 32 // 8, u % 8
    quad = (i // 2 * groups + group) * 2 + i % 2 if keys else i * groups + group
    return (u // 32 * 32 + quad) * 4 + d % 4


def _pool(case, gen, pages):
    """K and V pages [pages, kv_heads, page, dim / 2] of random codes, and their scales [pages, kv_heads, page, dim / 32]."""
    out = []
    for _ in range(2):
        shape = (pages, case["kv_heads"], case["page"])
        size = torch.exp(0.4 * torch.randn(case["dim"] // 32, generator=gen, device="cuda"))
        # a group's codes: a normal vector's, the largest at an end of the range
        codes = torch.randn(*shape, case["dim"], generator=gen, device="cuda").mul_(3.6).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
        scale = torch.rand(*shape, case["dim"] // 32, generator=gen, device="cuda").mul_(0.12).add_(0.22).mul_(size)
        sign = torch.rand(scale.shape, generator=gen, device="cuda") < 0.5
        out.append((codes[..., 0::2] | codes[..., 1::2] << 4, torch.where(sign, -scale, scale).bfloat16()))
        del codes
    return out


def _table(counts, gen, spare):
    """A page table for sequences of `counts` pages, the pages in any order in a pool with `spare` more."""
    total = sum(counts) + spare
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    width = max(1, max(counts))
    count = torch.tensor(counts, device="cuda")
    start = count.cumsum(0) - count
    i = torch.arange(width, device="cuda")
    at = (start[:, None] + i).clamp(max=total - 1)
    return torch.where(i < count[:, None], order[at], torch.zeros_like(order[at])), total


def _rope_table(dim, positions):
    freq = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def _offsets(v):
    return torch.tensor([0] + v, device="cuda").cumsum(0)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 60))
    s = {"case": case}
    if case["op"] == "gemm":
        n = case["n"] * (2 if case["mode"] == "swiglu" else 1)
        m, k, group = case["rows"], case["k"], case["group"]
        s["codes"] = torch.randn(n, k, generator=gen, device="cuda").mul_(3.0).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
        s["scales"] = (torch.rand(n, -(-k // group), generator=gen, device="cuda") * 0.006 + 0.004).bfloat16()
        s["x"] = _randn(gen, (m,), torch.bfloat16, k)
        s["residual"] = torch.randn(m, n, generator=gen, device="cuda").bfloat16() if case["mode"] == "residual" else None
        return s
    if case["op"] == "plan":
        new, past = _requests(case, seed)
        page, b = case["page"], case["requests"]
        held = [-(-p // page) for p in past]
        width = -(-(case["new_hi"] + case["past_hi"]) // page)
        order = torch.randperm(b + 5, generator=gen, device="cuda")[:b]  # the requests' sequences of b + 5
        small, total = _table(held, gen, case["spare"])
        table = torch.zeros(b + 5, width, dtype=torch.int32, device="cuda")
        table[order, : small.size(1)] = small
        length = torch.zeros(b + 5, dtype=torch.int64, device="cuda")
        length[order] = torch.tensor(past, device="cuda")
        taken = torch.zeros(total, dtype=torch.bool, device="cuda")
        inside = torch.arange(small.size(1), device="cuda") < torch.tensor(held, device="cuda")[:, None]
        taken[small[inside].long()] = True
        rest = (~taken).nonzero()[:, 0]
        free = torch.zeros(total, dtype=torch.int32, device="cuda")
        free[: rest.numel()] = rest[torch.randperm(rest.numel(), generator=gen, device="cuda")].to(torch.int32)
        s |= {"rows": order, "new": torch.tensor(new, device="cuda"), "tokens": sum(new), "length": length, "table": table,
              "free": free, "free_count": torch.tensor([rest.numel()], device="cuda"), "keep": torch.tensor(past, device="cuda")}
        return s
    h, kv, d, dtype = case["heads"], case["kv_heads"], case["dim"], _TORCH[case["dtype"]]
    page = case["page"]
    if case["op"] == "norm":
        n = case["tokens"]
        pages = -(-n // page) + 3
        s["qkv"] = _randn(gen, (n, h + 2 * kv), dtype, d).reshape(n, -1)
        s["k"], s["v"] = (_randn(gen, (pages, kv, page), dtype, d) for _ in range(2))
        s["q_norm"], s["k_norm"] = ((1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dtype) for _ in range(2))
        s["eps"] = 1e-6
        s["pos"] = torch.randint(0, case["past"] + 1, (n,), generator=gen, device="cuda") if case["past"] else torch.arange(n, device="cuda")
        s["slots"] = torch.randperm(pages, generator=gen, device="cuda").repeat_interleave(page)[:n] * page + \
            torch.arange(n, device="cuda") % page
        s["cs"] = _rope_table(d, max(case["past"] + 1, n))
        return s
    if case["op"] == "attend":
        lens = _spread(case["lo"], case["hi"], case["rows"])
        random.Random("%s lengths" % seed).shuffle(lens)
        t = case["tokens"]
        counts = [-(-(n + t - 1) // page) for n in lens]
        s["table"], pages = _table(counts, gen, 3)
        (s["k"], s["k_scale"]), (s["v"], s["v_scale"]) = _pool(case, gen, pages)
        s["lengths"] = torch.tensor(lens, device="cuda")
        s["q"] = _randn(gen, (case["rows"] * t, h), dtype, d)
        s["scale"] = d**-0.5
        return s
    new, past = _lengths(case, seed)
    counts = [-(-(n + p) // page) for n, p in zip(new, past)]
    table, pages = _table(counts, gen, 3)
    (s["k"], s["k_scale"]), (s["v"], s["v_scale"]) = _pool(case, gen, pages)
    s["qkv"] = _randn(gen, (sum(new), h + 2 * kv), dtype, d).reshape(sum(new), -1)
    s["pos"] = torch.cat([torch.arange(p, n + p, device="cuda") for n, p in zip(new, past)])
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"))
    s["slots"] = table[seq, s["pos"] // page].long() * page + s["pos"] % page
    s["cs"] = _rope_table(d, max(n + p for n, p in zip(new, past)))
    s["table"] = table if case["back"] == "all" else table.gather(1, torch.tensor(counts, device="cuda")[:, None] - 1)
    back = [_back(case, n, p) for n, p in zip(new, past)]
    s["back"], s["back_tokens"] = _offsets(back), sum(back)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] in ("attend", "append"):
        s["k_order"], s["v_order"] = _order(case["dim"], True), _order(case["dim"], False)
    if own and case["op"] == "gemm":  # the weights as the kernels read them, laid out once when a model is loaded
        s["weights"] = _own().int4_weights(s["codes"], s["scales"], case["group"])
    return s


# ----------------------------------------------------------------------------------------------------------------
# one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"attend": _own_attend, "append": _own_append, "norm": _own_norm, "plan": _own_plan, "gemm": _own_gemm}[op](state)
    return {"attend": _plain_attend, "append": _plain_append, "norm": _plain_norm, "plan": _plain_plan, "gemm": _plain_gemm}[op](state)


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


def _own_attend(s):
    return _own().paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["scale"], tokens=s["case"]["tokens"],
                                  k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_append(s):
    k = _own()
    q = k.paged_rope_kv(s["qkv"], s["cs"], s["pos"], s["k"], s["v"], s["slots"], s["case"]["heads"], s["case"]["kv_heads"],
                        k_scale=s["k_scale"], v_scale=s["v_scale"])
    back = k.paged_kv_read(s["k"], s["v"], s["table"], s["back"], s["back_tokens"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                           dtype=s["qkv"].dtype)
    return q, back[0], back[1]


def _own_norm(s):
    q = _own().paged_norm_rope_kv(s["qkv"], s["q_norm"], s["k_norm"], s["cs"], s["pos"], s["k"], s["v"], s["slots"],
                                  s["case"]["heads"], s["case"]["kv_heads"], eps=s["eps"])
    return q, s["k"], s["v"]


def _own_plan(s):
    k = _own()
    state = (s["length"], s["table"], s["free"], s["free_count"])
    out = k.paged_plan(s["rows"], s["new"], s["tokens"], s["case"]["page"], *state)
    k.paged_trim(s["rows"], s["keep"], s["case"]["page"], *state)
    return (*out, *state)


def _own_gemm(s):
    return _own().decode_gemm_int4(s["x"], s["weights"], s["case"]["mode"], residual=s["residual"])


def _unpacked(codes, scale, order):
    """4-bit vectors as the numbers they stand for."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., order].float() - 8.0
    return (c.unflatten(-1, (-1, 32)) * scale.float()[..., None]).flatten(-2)


def _plain_attend(s):
    c = s["case"]
    t, kv, d = c["tokens"], c["kv_heads"], c["dim"]
    g = c["heads"] // kv
    at = s["table"].long()
    b, keys = at.size(0), at.size(1) * c["page"]
    k, v = (_unpacked(s[x][at], s[x + "_scale"][at], s[x + "_order"]).permute(0, 2, 1, 3, 4).reshape(b, kv, keys, d) for x in "kv")
    q = s["q"].float().view(b, t, kv, g, d).permute(0, 2, 1, 3, 4).reshape(b, kv, t * g, d)
    x = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    limit = s["lengths"][:, None] + torch.arange(t, device=q.device)  # keys each query sees
    seen = (torch.arange(keys, device=q.device) < limit[:, :, None, None]).expand(b, t, g, keys).reshape(b, 1, t * g, keys)
    x = x.masked_fill(~seen, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))  # a query that sees no key: zeros
    o = torch.matmul(p, v)
    return o.view(b, kv, t, g, d).permute(0, 2, 1, 3, 4).reshape(b * t, c["heads"], d).to(s["q"].dtype)


def _rotate(x, cs):
    """Interleaved pairs of x [tokens, heads, dim] turned by cs [tokens, dim / 2, 2]."""
    re, im = x[..., 0::2], x[..., 1::2]
    co, si = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.stack([re * co - im * si, re * si + im * co], -1).flatten(-2)


def _packed(x, order):
    """(bytes, scales) of the vectors x [..., dim] (32 bits)."""
    g = x.unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = (torch.where(hi > -lo, hi, lo) * -0.125).bfloat16()
    f = scale.float()[..., None]
    c = torch.where(f == 0, torch.zeros_like(g), g / f).round().clamp(-8, 7).add(8).to(torch.uint8).flatten(-2)
    stored = torch.empty_like(c)
    stored[..., order] = c
    return stored[..., 0::2] | stored[..., 1::2] << 4, scale


def _plain_append(s):
    c = s["case"]
    h, kv, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    dtype = s["qkv"].dtype
    x = s["qkv"].view(-1, h + 2 * kv, d)
    turned = _rotate(x[:, : h + kv].float(), s["cs"][s["pos"]]).to(dtype)
    at, off = s["slots"] // page, s["slots"] % page
    out = []
    for name, rows in (("k", turned[:, h:]), ("v", x[:, h + kv:])):
        codes, scale = _packed(rows.float(), s[name + "_order"])
        s[name][at, :, off] = codes
        s[name + "_scale"][at, :, off] = scale
        i = torch.arange(s["back_tokens"], device=at.device)
        seq = torch.searchsorted(s["back"], i, right=True) - 1
        j = i - s["back"][seq]
        src, o = s["table"][seq, j // page].long(), j % page
        out.append(_unpacked(s[name][src, :, o], s[name + "_scale"][src, :, o], s[name + "_order"]).to(dtype))
    return turned[:, :h].contiguous(), out[0], out[1]


def _plain_norm(s):
    c = s["case"]
    h, kv, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    dtype = s["qkv"].dtype
    x = s["qkv"].view(-1, h + 2 * kv, d)
    y = x[:, : h + kv].float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + s["eps"])
    y = torch.cat([y[:, :h] * s["q_norm"].float(), y[:, h:] * s["k_norm"].float()], 1)
    y = _rotate(y, s["cs"][s["pos"]]).to(dtype)
    at, off = s["slots"] // page, s["slots"] % page
    s["k"][at, :, off] = y[:, h:]
    s["v"][at, :, off] = x[:, h + kv:]
    return y[:, :h].contiguous(), s["k"], s["v"]


def _plain_plan(s):
    """The requests in order: one that needs pages gets them if those before it and its own are free."""
    page = s["case"]["page"]
    rows, new, tokens = s["rows"], s["new"], s["tokens"]
    length, table, free, count = s["length"], s["table"], s["free"], s["free_count"]
    width = table.size(1)
    past = length[rows]
    held, want = (past + page - 1) // page, (past + new + page - 1) // page
    need = want - held
    upto = need.cumsum(0)
    taken = (need == 0) | (upto <= count)
    got = torch.where(taken, need, torch.zeros_like(need))
    # the pages: the k-th that a request takes is so far below the stack's top
    j = torch.arange(width, device=rows.device)
    fresh = taken[:, None] & (j >= held[:, None]) & (j < want[:, None])
    depth = (upto - need)[:, None] + j - held[:, None]
    here = table[rows]
    here = torch.where(fresh, free[(count - 1 - depth).clamp(0, free.numel() - 1)], here)
    table[rows] = here
    now = past + torch.where(taken, new, torch.zeros_like(new))
    length[rows] = now
    count -= got.sum()
    inside = j < ((now + page - 1) // page)[:, None]
    batch_table = torch.where(inside, here, torch.zeros_like(here))
    q_offsets = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    k_offsets = torch.cat([torch.zeros_like(now[:1]), now.cumsum(0)])
    i = torch.arange(tokens, device=rows.device)
    seq = torch.searchsorted(q_offsets, i, right=True) - 1
    pos = past[seq] + i - q_offsets[seq]
    slots = torch.where(taken[seq], batch_table[seq, (pos // page).clamp(max=width - 1)].long() * page + pos % page,
                        torch.full_like(pos, -1))
    lengths = torch.where(taken, past + 1, torch.zeros_like(past))
    # the step undone: the pages past the kept positions go back, the last request's first, each request's last page first
    keep = s["keep"]
    left = (keep + page - 1) // page
    back = (now + page - 1) // page - left
    before = back.sum() - back.cumsum(0)  # pages given back before this request's
    give = (j >= left[:, None]) & (j < (left + back)[:, None])
    place = count + before[:, None] + (left + back)[:, None] - 1 - j
    free[place[give]] = here[give]
    count += back.sum()
    length[rows] = keep
    return pos, slots, batch_table, lengths, q_offsets, k_offsets, taken, length, table, free, count


def _plain_gemm(s):
    c = s["case"]
    scale = s["scales"].float().repeat_interleave(c["group"], 1)[:, : c["k"]]
    y = s["x"].float() @ ((s["codes"].float() - 8.0) * scale).t()
    if c["mode"] == "residual":
        y = y + s["residual"].float()
    elif c["mode"] == "swiglu":
        gate, inner = y.chunk(2, -1)
        y = inner * gate / (1 + torch.exp(-gate))
    return y.bfloat16()


# ----------------------------------------------------------------------------------------------------------------
# the definition in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "norm": _exact_norm, "plan": lambda s: None, "gemm": _exact_gemm}[case["op"]](s)


def _exact_values(s, name, ids, head):
    """One head's rows of the pages `ids`, as the numbers they stand for: dim by dim from its nibble."""
    d = s["case"]["dim"]
    codes = s[name][ids, head].flatten(0, 1).long()
    scale = s[name + "_scale"][ids, head].flatten(0, 1).double()
    groups = min(4, d // 32)
    cols = []
    for dim in range(d):
        block, rest = divmod(dim, 128)
        group, i, n = rest // 32, rest % 32 // 4, rest % 4
        quad = 32 * block + ((i // 2 * groups + group) * 2 + i % 2 if name == "k" else i * groups + group)
        cols.append(4 * quad + n)
    cols = torch.tensor(cols, device=codes.device)
    c = codes[:, cols // 2] // torch.where(cols % 2 == 1, 16, 1) % 16 - 8
    return c.double() * scale[:, torch.arange(d, device=codes.device) // 32]


def _exact_attend(s):
    case = s["case"]
    kv, t, page = case["kv_heads"], case["tokens"], case["page"]
    g = case["heads"] // kv
    q = s["q"].double()
    out = torch.zeros_like(q)
    for r, n in enumerate(s["lengths"].tolist()):
        most = n + t - 1
        if most <= 0:
            continue
        ids = s["table"][r, : -(-most // page)].long()
        for j in range(kv):
            k, v = (_exact_values(s, x, ids, j)[:most] for x in ("k", "v"))
            rows = q[r * t:(r + 1) * t, j * g:(j + 1) * g]
            x = torch.einsum("tgd,nd->tgn", rows, k) * s["scale"]
            for i in range(t):
                if n + i > 0:
                    out[r * t + i, j * g:(j + 1) * g] = torch.softmax(x[i, :, : n + i], -1) @ v[: n + i]
    return out


def _turned(x, cs):
    z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous())
    return torch.view_as_real(z * torch.view_as_complex(cs.double())[:, None]).flatten(-2)


def _exact_append(s):
    """The cache's rows as four bits hold the vectors of the model's type."""
    c = s["case"]
    h, kv, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    dtype = s["qkv"].dtype
    x = s["qkv"].double().view(-1, h + 2 * kv, d)
    turned = _turned(x[:, : h + kv], s["cs"][s["pos"]])
    out = [turned[:, :h]]
    every = torch.arange(s["k"].size(0), device=x.device)
    for name, rows in (("k", turned[:, h:].to(dtype)), ("v", x[:, h + kv:])):
        flat = torch.stack([_exact_values(s, name, every, j) for j in range(kv)], 1)
        g = rows.double().reshape(-1, kv, d // 32, 32)
        ends = torch.sort(g, -1).values[..., [0, -1]]
        m = torch.where(ends.sum(-1) > 0, ends[..., 1], ends[..., 0])  # (the negative one, where two are as large)
        step = (-m / 8).to(torch.bfloat16).double()[..., None]
        c4 = torch.where(step == 0, torch.zeros_like(g), (g / step).round().clamp(-8, 7))
        flat[s["slots"]] = (c4 * step).flatten(-2)
        ends = s["back"].tolist()
        parts = []
        for i, (a, b) in enumerate(zip(ends, ends[1:])):
            j = torch.arange(b - a, device=flat.device)
            parts.append(flat[s["table"][i].long()[j // page] * page + j % page])
        out.append(torch.cat(parts))
    return tuple(out)


def _exact_norm(s):
    c = s["case"]
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].double().view(-1, h + 2 * kv, d)
    rms = (x[:, : h + kv].pow(2).sum(-1, keepdim=True) / d + s["eps"]).sqrt()
    weight = torch.cat([s["q_norm"].double().expand(h, d), s["k_norm"].double().expand(kv, d)])
    y = _turned(x[:, : h + kv] / rms * weight, s["cs"][s["pos"]])
    out = [y[:, :h]]
    for name, rows in (("k", y[:, h:]), ("v", x[:, h + kv:])):
        pool = s[name].double()
        flat = pool.transpose(1, 2).reshape(-1, kv, d)
        flat[s["slots"]] = rows
        out.append(flat.view(pool.size(0), -1, kv, d).transpose(1, 2))
    return tuple(out)


def _exact_gemm(s):
    c = s["case"]
    k = torch.arange(c["k"], device=s["x"].device)
    w = (s["codes"].double() - 8) * s["scales"].double()[:, k // c["group"]]
    y = s["x"].double() @ w.t()
    if c["mode"] == "residual":
        return s["residual"].double() + y
    if c["mode"] == "swiglu":
        return y[:, c["n"]:] * y[:, : c["n"]] * torch.sigmoid(y[:, : c["n"]])
    return y
