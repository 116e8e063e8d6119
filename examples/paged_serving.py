"""Serving a small decoder from a paged cache: prompts of different lengths prefilled together, long ones in chunks, then
decoded together. Random weights, grouped heads, greedy tokens; the cache in the model's type or in 8 bits.

    python examples/paged_serving.py [--fp8] [--steps 16]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "omniasr-trt_b200"))

from omniasr_b200 import kernels  # noqa: E402
from omniasr_b200.paged import PagedCache  # noqa: E402


class Decoder:
    """A pre-norm decoder with rotary positions, grouped heads and a SwiGLU block, on random weights."""

    def __init__(self, layers=2, heads=8, kv_heads=2, dim=128, width=512, vocab=1000, positions=4096, seed=0):
        g = torch.Generator().manual_seed(seed)
        w = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).to(torch.bfloat16).cuda()  # noqa: E731
        self.heads, self.kv_heads, self.dim, self.layers = heads, kv_heads, dim, layers
        self.embed, self.head = w(vocab, width), w(vocab, width)
        self.blocks = [(w((heads + 2 * kv_heads) * dim, width), w(width, heads * dim), w(4 * width, width), w(width, 2 * width))
                       for _ in range(layers)]
        freq = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
        self.cs = torch.stack([angle.cos(), angle.sin()], -1).float().cuda()

    def norm(self, x):
        return F.rms_norm(x, (x.size(-1),))

    def step(self, tokens: torch.Tensor, attend) -> torch.Tensor:
        """Hidden states of the tokens [N]; ``attend(layer, qkv)`` is the attention [N, heads, D]."""
        h = self.embed[tokens]
        for i, (qkv_w, out_w, in_w, down_w) in enumerate(self.blocks):
            o = attend(i, self.norm(h) @ qkv_w.t())
            h = torch.addmm(h, o.reshape(len(tokens), -1), out_w.t())
            gate, inner = (self.norm(h) @ in_w.t()).chunk(2, -1)
            h = torch.addmm(h, F.silu(gate) * inner, down_w.t())
        return self.norm(h)

    def next(self, h: torch.Tensor) -> torch.Tensor:
        return (h @ self.head.t()).float().argmax(-1)


def serve(model: Decoder, prompts: list[list[int]], steps: int, kind: torch.dtype, page: int = 16, chunk: int = 64) -> list[list[int]]:
    """Greedy continuations of the prompts. Prompts past ``chunk`` tokens are prefilled in chunks, beside the others."""
    need = sum(-(-(len(p) + steps + 1) // page) for p in prompts) + 4
    cache = PagedCache(model.layers, need, page, model.kv_heads, model.dim, kind=kind)
    seqs = [cache.add() for _ in prompts]
    left = [list(p) for p in prompts]
    out: list[list[int]] = [[] for _ in prompts]
    while any(left):  # rounds of at most `chunk` tokens of each prompt that still has some
        live = [i for i, p in enumerate(left) if p]
        parts = [left[i][:chunk] for i in live]
        batch = cache.extend([seqs[i] for i in live], [len(p) for p in parts])
        tokens = torch.tensor([t for p in parts for t in p], device="cuda")
        h = model.step(tokens, lambda i, qkv: cache.prefill(i, qkv, model.cs, batch, model.heads))
        last = model.next(h[batch.q_offsets[1:] - 1])
        for i, token in zip(live, last.tolist()):
            left[i] = left[i][chunk:]
            if not left[i]:
                out[i].append(token)
    for _ in range(steps):
        batch = cache.extend(seqs, [1] * len(seqs))
        tokens = torch.tensor([o[-1] for o in out], device="cuda")
        h = model.step(tokens, lambda i, qkv: cache.decode(i, qkv, model.cs, batch, model.heads))
        for o, token in zip(out, model.next(h).tolist()):
            o.append(token)
    for s in seqs:
        cache.free(s)
    assert cache.free_pages == need
    return out


def dense(model: Decoder, prompt: list[int], tokens_out: list[int]) -> list[tuple[int, float]]:
    """Without a cache, attention in float32 over everything so far: for each token of a continuation, the token this form
    prefers there and by how much (in logits) over the one that was taken."""
    tokens = list(prompt)
    got = []
    for taken in tokens_out:
        n = len(tokens)
        cs = model.cs[:n]

        def attend(_, qkv):
            x = qkv.float().view(n, -1, model.dim)
            q, k, v = x.split([model.heads, model.kv_heads, model.kv_heads], 1)
            turn = lambda t: torch.stack([t[..., 0::2] * cs[:, None, :, 0] - t[..., 1::2] * cs[:, None, :, 1],  # noqa: E731
                                          t[..., 0::2] * cs[:, None, :, 1] + t[..., 1::2] * cs[:, None, :, 0]], -1).flatten(-2)
            q, k = turn(q).to(torch.bfloat16).float(), turn(k).to(torch.bfloat16).float()
            g = model.heads // model.kv_heads
            k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
            s = torch.einsum("ihd,jhd->hij", q, k) * model.dim**-0.5
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
            return torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).to(torch.bfloat16)

        h = model.step(torch.tensor(tokens, device="cuda"), attend)
        logits = (h[-1:] @ model.head.t()).float()[0]
        got.append((int(logits.argmax()), float(logits.max() - logits[taken])))
        tokens.append(taken)
    return got


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--fp8", action="store_true", help="8-bit cache")
    ap.add_argument("--steps", type=int, default=16)
    args = ap.parse_args()
    assert kernels.available(torch.device("cuda")), "needs a B200"
    model = Decoder()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (5, 200, 1, 63, 64)]
    for p, o in zip(prompts, serve(model, prompts, args.steps, torch.float8_e4m3fn if args.fp8 else torch.bfloat16)):
        print(f"{len(p):4d} tokens ->", *o)
    assert kernels.read_status() == 0


if __name__ == "__main__":
    main()
