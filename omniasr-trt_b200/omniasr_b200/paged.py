"""A paged key-value cache for serving: pages handed out to sequences on the host, written and read by the kernels of
:mod:`omniasr_b200.kernels` (``paged_rope_kv``, ``paged_attention``, ``paged_kv_read``, ``packed_attention``).

A sequence holds whole pages of every layer; its positions lie in them in order. :class:`PagedCache` keeps which pages a
sequence has and gives the kernels' index tensors for a batch; :meth:`PagedCache.prefill` and :meth:`PagedCache.decode` are
one layer's attention of a batch of prompts (or chunks of them) and of one new token (or a draft) per sequence.
:class:`DeviceTables` is the same bookkeeping on the GPU (``paged_plan``, ``paged_trim``), for decode loops that the host does
not steer step by step, in a CUDA graph for instance.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import kernels


@dataclass
class Batch:
    """A step's index tensors (device): which sequences, where their new tokens go, and what they see."""

    tokens: int  # new tokens in all
    new: list[int] | None  # new tokens per sequence (None: the GPU alone knows)
    total: int | None  # keys in all, the new tokens' among them (None: the GPU alone knows)
    pos: torch.Tensor  # [tokens] position of each new token
    slots: torch.Tensor  # [tokens] page number * page + offset
    table: torch.Tensor  # [sequences, width] int32
    lengths: torch.Tensor  # [sequences] keys before the new tokens, plus one
    q_offsets: torch.Tensor  # [sequences + 1]
    k_offsets: torch.Tensor  # [sequences + 1]
    fresh: bool  # no sequence had keys before this step (False where the GPU alone knows)
    taken: torch.Tensor | None = None  # DeviceTables: [sequences] which requests got their pages


class PagedCache:
    """``layers`` caches of ``pages`` pages of ``page`` positions, ``kv_heads`` heads of ``dim``; ``kind`` is the element type:
    the model's dtype, ``torch.float8_e4m3fn`` (codes with one power-of-two scale byte per position and head), or ``torch.uint8``
    (4-bit codes with a bfloat16 scale per 32 dims, ``dim`` 32 and more: 4.5 bits a value)."""

    def __init__(self, layers: int, pages: int, page: int, kv_heads: int, dim: int, dtype: torch.dtype = torch.bfloat16,
                 kind: torch.dtype | None = None, device: torch.device | str = "cuda"):
        self.page, self.kv_heads, self.dim, self.dtype = page, kv_heads, dim, dtype
        self.device = torch.device(device)
        kind = dtype if kind is None else kind
        if kind == torch.uint8 and dim % 32:
            raise ValueError(f"PagedCache: 4-bit codes of head_dim {dim} (a multiple of 32)")
        shape = (layers, pages, kv_heads, page, dim // 2 if kind == torch.uint8 else dim)
        self.k = torch.zeros(shape, dtype=kind, device=self.device)
        self.v = torch.zeros(shape, dtype=kind, device=self.device)
        self.k_scale = self.v_scale = None
        if kind == torch.float8_e4m3fn:
            self.k_scale = torch.full(shape[:-1], 127, dtype=torch.uint8, device=self.device)
            self.v_scale = torch.full(shape[:-1], 127, dtype=torch.uint8, device=self.device)
        if kind == torch.uint8:
            self.k_scale = torch.zeros(*shape[:-1], dim // 32, dtype=torch.bfloat16, device=self.device)
            self.v_scale = torch.zeros_like(self.k_scale)
        self._free = list(range(pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._length: dict[int, int] = {}
        self._next = 0

    def add(self) -> int:
        """A new sequence without keys."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._length[seq] = [], 0
        return seq

    def free(self, seq: int) -> None:
        """Gives the sequence's pages back."""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._length[seq]

    def trim(self, seq: int, length: int) -> None:
        """Keeps the sequence's first ``length`` positions (drops drafts that were not accepted) and gives back the pages past
        them."""
        if not 0 <= length <= self._length[seq]:
            raise ValueError(f"trim: {length} of {self._length[seq]} positions")
        keep = -(-length // self.page)
        self._free.extend(reversed(self._pages[seq][keep:]))
        del self._pages[seq][keep:]
        self._length[seq] = length

    def length(self, seq: int) -> int:
        return self._length[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def extend(self, seqs: list[int], new: list[int]) -> Batch:
        """Room for ``new[i]`` tokens of ``seqs[i]`` each (at most once per sequence), which count as the sequence's from now
        on. Raises, with nothing changed, when the pages do not suffice."""
        if len(set(seqs)) != len(seqs) or len(new) != len(seqs) or any(n < 0 for n in new):
            raise ValueError("extend: one count of new tokens for each of different sequences")
        past = [self._length[s] for s in seqs]
        need = [-(-(p + n) // self.page) - len(self._pages[s]) for s, p, n in zip(seqs, past, new)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"the cache is full: {sum(need)} pages needed, {len(self._free)} free")
        for s, n, k in zip(seqs, new, need):
            self._pages[s].extend(self._free.pop() for _ in range(k))
            self._length[s] += n
        width = max([1] + [len(self._pages[s]) for s in seqs])
        table = torch.tensor([self._pages[s] + [0] * (width - len(self._pages[s])) for s in seqs], dtype=torch.int32)
        table = table.reshape(len(seqs), width)
        pos = torch.tensor([j for p, n in zip(past, new) for j in range(p, p + n)], dtype=torch.int64)
        slots = torch.tensor([self._pages[s][j // self.page] * self.page + j % self.page
                              for s, p, n in zip(seqs, past, new) for j in range(p, p + n)], dtype=torch.int64)
        offsets = lambda v: torch.tensor([0] + v, dtype=torch.int64).cumsum(0)  # noqa: E731
        both = [p + n for p, n in zip(past, new)]
        up = lambda t: t.to(self.device)  # noqa: E731
        return Batch(sum(new), list(new), sum(both), up(pos), up(slots), up(table),
                     up(torch.tensor([p + 1 for p in past], dtype=torch.int64)), up(offsets(list(new))), up(offsets(both)),
                     not any(past))

    def device_tables(self, seqs: int, width: int, pages: int | None = None) -> DeviceTables:
        """Tables on the GPU for ``seqs`` sequences of at most ``width`` pages, which take ``pages`` of the free pages (all of them
        by default) over: this object's own sequences no longer get those until :meth:`take_back`."""
        count = len(self._free) if pages is None else pages
        if not 0 <= count <= len(self._free):
            raise ValueError(f"device_tables: {count} pages of {len(self._free)} free")
        taken = [self._free.pop() for _ in range(count)]
        return DeviceTables(seqs, width, self.page, taken[::-1], self.device)

    def take_back(self, tables: DeviceTables) -> None:
        """Takes the pages of :meth:`device_tables` back, once all of the tables' sequences are freed (``trim`` to 0). Waits for the
        GPU. The tables have no pages from then on, in graphs that captured their steps too."""
        pages = tables.free.tolist()
        if int(tables.free_count) != len(pages):
            raise ValueError(f"take_back: {len(pages) - int(tables.free_count)} of {len(pages)} pages are still in use")
        mine = set(self._free).union(*self._pages.values())
        if tables.page != self.page or len(set(pages)) != len(pages) or any(p in mine or not 0 <= p < self.k.size(1) for p in pages):
            raise ValueError("take_back: tables of another cache, or taken back before")
        tables.free_count.zero_()
        self._free.extend(pages)

    def _layer(self, layer: int) -> tuple:
        scales = (None, None) if self.k_scale is None else (self.k_scale[layer], self.v_scale[layer])
        return self.k[layer], self.v[layer], scales

    def write(self, layer: int, qkv: torch.Tensor, cs: torch.Tensor, batch: Batch, heads: int,
              norms: tuple[torch.Tensor, torch.Tensor, float] | None = None) -> torch.Tensor:
        """RoPE of the new tokens' q and k, their k and v into the layer's pages; returns q [tokens, heads, D]. ``norms`` (q's
        weights [D], k's, epsilon): q and k are normed per head before."""
        k, v, (ks, vs) = self._layer(layer)
        if norms is None:
            return kernels.paged_rope_kv(qkv, cs, batch.pos, k, v, batch.slots, heads, self.kv_heads, k_scale=ks, v_scale=vs)
        return kernels.paged_norm_rope_kv(qkv, norms[0], norms[1], cs, batch.pos, k, v, batch.slots, heads, self.kv_heads,
                                          eps=norms[2], k_scale=ks, v_scale=vs)

    def prefill(self, layer: int, qkv: torch.Tensor, cs: torch.Tensor, batch: Batch, heads: int, scale: float | None = None,
                norms: tuple[torch.Tensor, torch.Tensor, float] | None = None) -> torch.Tensor:
        """One layer's causal attention of a batch of prompts, or of chunks whose earlier keys the cache holds: writes the new
        keys and reads all of them back as packed rows (what a later step sees, an 8-bit or 4-bit cache's rounding included)."""
        if batch.total is None:
            raise ValueError("prefill: a batch of tables on the GPU needs its number of keys (DeviceTables.plan's total)")
        q = self.write(layer, qkv, cs, batch, heads, norms)
        k, v, (ks, vs) = self._layer(layer)
        kk, vv = kernels.paged_kv_read(k, v, batch.table, batch.k_offsets, batch.total, k_scale=ks, v_scale=vs, dtype=self.dtype)
        return kernels.packed_attention(q, kk, vv, batch.q_offsets, batch.k_offsets, scale)

    def decode(self, layer: int, qkv: torch.Tensor, cs: torch.Tensor, batch: Batch, heads: int, scale: float | None = None,
               norms: tuple[torch.Tensor, torch.Tensor, float] | None = None) -> torch.Tensor:
        """One layer's attention of the same number of new tokens (one, or a draft) of every sequence, straight over the
        pages."""
        if batch.new is None or len(set(batch.new)) > 1:
            raise ValueError("decode: the same number of new tokens for every sequence (prefill takes others)")
        q = self.write(layer, qkv, cs, batch, heads, norms)
        if not any(batch.new):
            return q  # no queries
        k, v, (ks, vs) = self._layer(layer)
        return kernels.paged_attention(q, k, v, batch.table, batch.lengths, self.dim**-0.5 if scale is None else scale,
                                       tokens=batch.new[0], k_scale=ks, v_scale=vs)


class DeviceTables:
    """Which pages ``seqs`` sequences have, on the GPU: lengths, a table of at most ``width`` page numbers a sequence, and the free
    pages as a stack (``free``: their numbers, the last is taken first). Sequences are numbered from 0 and begin without keys."""

    def __init__(self, seqs: int, width: int, page: int, free: list[int], device: torch.device | str = "cuda"):
        device = torch.device(device)
        self.page, self.width = page, width
        self.length = torch.zeros(seqs, dtype=torch.int64, device=device)
        self.table = torch.zeros(seqs, width, dtype=torch.int32, device=device)
        self.free = torch.tensor(free, dtype=torch.int32).to(device)
        self.free_count = torch.tensor([len(free)], dtype=torch.int64).to(device)

    def _state(self) -> tuple:
        return self.length, self.table, self.free, self.free_count

    def plan(self, rows: torch.Tensor, new: int | torch.Tensor, tokens: int | None = None, total: int | None = None,
             width: int | None = None) -> Batch:
        """Room for new tokens of the sequences ``rows`` [B] (int64, on the GPU), ``new`` of each or ``new[i]`` of the i-th ([B], then
        with ``tokens``, a number that the host knows, at least their sum). ``total`` (for :meth:`PagedCache.prefill`): at least the
        keys of all these sequences after the step. ``width``: pages a sequence that the step's table has room for. Nothing waits
        for the GPU: whether the pages sufficed is in the batch's ``taken``, as :func:`kernels.paged_plan` describes it."""
        b = rows.numel()
        each = None
        if isinstance(new, int):
            each, new, tokens = new, torch.full((b,), new, dtype=torch.int64, device=rows.device), b * new
        if tokens is None:
            raise ValueError("plan: new tokens per request on the GPU need their number (tokens)")
        # (A refused request may ask for positions past the tables; a rope table need not reach there.)
        pos, slots, table, lengths, q_offsets, k_offsets, taken = kernels.paged_plan(rows, new, tokens, self.page, *self._state(), width=width,
                                                                                     positions=max(1, self.width * self.page))
        return Batch(tokens, None if each is None else [each] * b, total, pos, slots, table, lengths, q_offsets,
                     k_offsets, False, taken)

    def trim(self, rows: torch.Tensor, keep: torch.Tensor) -> None:
        """The sequences ``rows`` keep their first ``keep`` positions (both int64 on the GPU; 0 frees a sequence)."""
        kernels.paged_trim(rows, keep, self.page, *self._state())
