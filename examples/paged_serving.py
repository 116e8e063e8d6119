"""Serving a small decoder from a paged cache: prompts of different lengths prefilled together, long ones in chunks, then
decoded together. Random weights, grouped heads, greedy tokens; the cache in the model's type, in 8 bits or in 4, the weights of
the decode steps in 4 bits, queries and keys normed per head, and the decode loop as a CUDA graph that keeps its own tables.

    python examples/paged_serving.py [--fp8 | --int4] [--int4-weights] [--norms] [--graph] [--steps 16]
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

    def __init__(self, layers=2, heads=8, kv_heads=2, dim=128, width=512, vocab=1000, positions=4096, seed=0, norms=False,
                 int4=False):
        g = torch.Generator().manual_seed(seed)
        w = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).to(torch.bfloat16).cuda()  # noqa: E731
        self.heads, self.kv_heads, self.dim, self.layers = heads, kv_heads, dim, layers
        self.embed, self.head = w(vocab, width), w(vocab, width)
        self.blocks = [(w((heads + 2 * kv_heads) * dim, width), w(width, heads * dim), w(4 * width, width), w(width, 2 * width))
                       for _ in range(layers)]
        self.norms = [None] * layers  # of queries and keys: weights and epsilon
        if norms:
            ones = lambda: 1 + 0.1 * w(dim) * dim**0.5  # noqa: E731
            self.norms = [(ones(), ones(), 1e-6) for _ in range(layers)]
        self.blocks4 = None  # the same weights in 4 bits, for steps of few tokens
        if int4:
            self.blocks4 = [[kernels.int4_quantise(m) for m in block] for block in self.blocks]
            self.blocks = [tuple(m.values().to(torch.bfloat16) for m in block) for block in self.blocks4]
        freq = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
        angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
        self.cs = torch.stack([angle.cos(), angle.sin()], -1).float().cuda()

    def norm(self, x):
        return F.rms_norm(x, (x.size(-1),))

    def step(self, tokens: torch.Tensor, attend) -> torch.Tensor:
        """Hidden states of the tokens [N]; ``attend(layer, qkv)`` is the attention [N, heads, D]."""
        h = self.embed[tokens]
        if self.blocks4 is not None and len(tokens) <= 64:
            return self.step4(h, attend)
        for i, (qkv_w, out_w, in_w, down_w) in enumerate(self.blocks):
            o = attend(i, self.norm(h) @ qkv_w.t())
            h = torch.addmm(h, o.reshape(len(tokens), -1), out_w.t())
            gate, inner = (self.norm(h) @ in_w.t()).chunk(2, -1)
            h = torch.addmm(h, F.silu(gate) * inner, down_w.t())
        return self.norm(h)

    def step4(self, h: torch.Tensor, attend) -> torch.Tensor:
        gemm = kernels.decode_gemm_int4
        for i, (qkv_w, out_w, in_w, down_w) in enumerate(self.blocks4):
            o = attend(i, gemm(self.norm(h), qkv_w))
            h = gemm(o.reshape(len(h), -1), out_w, "residual", residual=h)
            h = gemm(gemm(self.norm(h), in_w, "swiglu"), down_w, "residual", residual=h)
        return self.norm(h)

    def next(self, h: torch.Tensor) -> torch.Tensor:
        return (h @ self.head.t()).float().argmax(-1)


def serve(model: Decoder, prompts: list[list[int]], steps: int, kind: torch.dtype, page: int = 16, chunk: int = 64,
          graph: bool = False) -> list[list[int]]:
    """Greedy continuations of the prompts. Prompts past ``chunk`` tokens are prefilled in chunks, beside the others."""
    if graph:
        return serve_graph(model, prompts, steps, kind, page)
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
        h = model.step(tokens, lambda i, qkv: cache.prefill(i, qkv, model.cs, batch, model.heads, norms=model.norms[i]))
        last = model.next(h[batch.q_offsets[1:] - 1])
        for i, token in zip(live, last.tolist()):
            left[i] = left[i][chunk:]
            if not left[i]:
                out[i].append(token)
    for _ in range(steps):
        batch = cache.extend(seqs, [1] * len(seqs))
        tokens = torch.tensor([o[-1] for o in out], device="cuda")
        h = model.step(tokens, lambda i, qkv: cache.decode(i, qkv, model.cs, batch, model.heads, norms=model.norms[i]))
        for o, token in zip(out, model.next(h).tolist()):
            o.append(token)
    for s in seqs:
        cache.free(s)
    assert cache.free_pages == need
    return out


def serve_graph(model: Decoder, prompts: list[list[int]], steps: int, kind: torch.dtype, page: int = 16) -> list[list[int]]:
    """The same with the tables on the GPU: the prompts in one step, the decode loop as one graph that is replayed, each replay
    taking its pages, writing, attending and choosing the next tokens from the ones before."""
    n = len(prompts)
    width = max(-(-(len(p) + steps + 1) // page) for p in prompts)
    cache = PagedCache(model.layers, sum(-(-(len(p) + steps + 1) // page) for p in prompts) + 4, page, model.kv_heads, model.dim, kind=kind)
    tables = cache.device_tables(n, width)
    rows = torch.arange(n, device="cuda")
    tokens = torch.tensor([t for p in prompts for t in p], device="cuda")
    batch = tables.plan(rows, torch.tensor([len(p) for p in prompts], device="cuda"), len(tokens), total=len(tokens))
    h = model.step(tokens, lambda i, qkv: cache.prefill(i, qkv, model.cs, batch, model.heads, norms=model.norms[i]))
    current = model.next(h[batch.q_offsets[1:] - 1])
    out = [current.tolist()]

    def step():
        batch = tables.plan(rows, 1)
        h = model.step(current, lambda i, qkv: cache.decode(i, qkv, model.cs, batch, model.heads, norms=model.norms[i]))
        current.copy_(model.next(h))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        if steps > 0:
            step()  # (eager once: what is set up at first use is)
            out.append(current.tolist())
        if steps > 1:
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured, stream=stream):
                step()
            for _ in range(steps - 1):
                captured.replay()
                out.append(current.tolist())
        tables.trim(rows, torch.zeros_like(rows))
    torch.cuda.current_stream().wait_stream(stream)
    free = cache.free_pages
    cache.take_back(tables)
    assert free == 0 and cache.free_pages == tables.free.numel()
    return [list(o) for o in zip(*out)]


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
    ap.add_argument("--int4", action="store_true", help="4-bit cache")
    ap.add_argument("--int4-weights", action="store_true", help="4-bit weights")
    ap.add_argument("--norms", action="store_true", help="queries and keys normed per head")
    ap.add_argument("--graph", action="store_true", help="tables on the GPU, decode steps as a CUDA graph")
    ap.add_argument("--steps", type=int, default=16)
    args = ap.parse_args()
    assert kernels.available(torch.device("cuda")), "needs a B200"
    model = Decoder(norms=args.norms, int4=args.int4_weights)
    kind = torch.uint8 if args.int4 else torch.float8_e4m3fn if args.fp8 else torch.bfloat16
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (5, 200, 1, 63, 64)]
    for p, o in zip(prompts, serve(model, prompts, args.steps, kind, graph=args.graph)):
        print(f"{len(p):4d} tokens ->", *o)
    assert kernels.read_status() == 0


if __name__ == "__main__":
    main()
