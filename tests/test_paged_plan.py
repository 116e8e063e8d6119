"""Tables, slots and offsets built on the GPU (paged_plan, paged_trim) against the same rules in plain Python, and against what
PagedCache does on the host. Whole numbers: everything is equal."""

import random

import pytest
import torch

from omniasr_b200 import kernels
from omniasr_b200.paged import PagedCache

DEV = "cuda"


class Host:
    """The state and its rules in plain Python."""

    def __init__(self, seqs, width, pages, page, r):
        self.page, self.width = page, width
        self.length = [0] * seqs
        self.table = [[0] * width for _ in range(seqs)]
        self.free = list(range(pages))
        r.shuffle(self.free)
        self.pages = pages

    def held(self, n):
        return -(-n // self.page)

    def plan(self, rows, new, tokens, width=None):
        width = self.width if width is None else width
        pos, slots = [0] * tokens, [-1] * tokens
        q, k, lengths, taken, batch = [0], [0], [], [], []
        top, sum_need, status, seen, writes = len(self.free), 0, 0, set(), []
        end = 0
        for r, n in zip(rows, new):
            ok = 0 <= r < len(self.length) and r not in seen
            inside = 0 <= r < len(self.length)
            if not ok:
                status = 1
            if inside:
                seen.add(r)
            past = self.length[r] if inside else 0
            fresh = max(0, n)
            end += fresh
            if n < 0 or end > tokens:
                ok, status = False, 1
            if ok and past + fresh > width * self.page:
                ok = False
            need = self.held(past + fresh) - self.held(past) if ok else 0
            if need > 0:
                sum_need += need
                ok = sum_need <= top
            first = q[-1]
            q.append(min(end, tokens))
            got = [self.free[top - 1 - (sum_need - need) - i] for i in range(need)] if ok else []
            pages = self.table[r][: self.held(past)] + got if inside else []
            for i in range(q[-1] - first):
                p = past + i
                pos[first + i] = p
                if ok:
                    slots[first + i] = pages[p // self.page] * self.page + p % self.page
            lengths.append(past + 1 if ok else 0)
            taken.append(ok)
            k.append(k[-1] + past + (fresh if ok else 0))
            batch.append((pages + [0] * width)[:width])
            if ok:
                writes.append((r, past, past + fresh, got))
        used = 0
        for r, past, now, got in writes:
            self.length[r] = now
            self.table[r][self.held(past):self.held(past) + len(got)] = got
            used += len(got)
        del self.free[len(self.free) - used:]
        return pos, slots, batch, lengths, q, k, taken, status

    def trim(self, rows, keep):
        status, seen, back = 0, set(), []
        for r, n in zip(rows, keep):
            ok = 0 <= r < len(self.length) and r not in seen
            seen.add(r)
            if not ok or not 0 <= n <= self.length[r]:
                status = 1
                continue
            back.append((r, n))
        total = sum(self.held(self.length[r]) - self.held(n) for r, n in back)
        if len(self.free) + total > self.pages:
            return 1
        for r, n in reversed(back):
            self.free += reversed(self.table[r][self.held(n):self.held(self.length[r])])
        for r, n in back:
            self.length[r] = n
        return status

    def tensors(self, device):
        free = torch.zeros(self.pages, dtype=torch.int32)
        free[: len(self.free)] = torch.tensor(self.free, dtype=torch.int32)
        state = (torch.tensor(self.length), torch.tensor(self.table, dtype=torch.int32).reshape(len(self.length), self.width), free,
                 torch.tensor([len(self.free)]))
        return tuple(t.to(device) for t in state)


def same_state(host, state):
    length, table, free, count = (t.cpu() for t in state)
    assert length.tolist() == host.length
    assert int(count) == len(host.free) and free[: len(host.free)].tolist() == host.free
    for r, n in enumerate(host.length):
        assert table[r, : host.held(n)].tolist() == host.table[r][: host.held(n)]


def same_plan(got, want):
    pos, slots, batch, lengths, q, k, taken, _ = want
    for g, w in zip(got, (pos, slots, batch, lengths, q, k, taken)):
        assert g.cpu().tolist() == w


def test_host_rules_agree_with_the_cache():
    """The plain rules give the pages and slots that PagedCache gives."""
    r = random.Random(0)
    cache = PagedCache(1, 40, 8, 1, 16, device="cpu")
    seqs = [cache.add() for _ in range(4)]
    host = Host(4, 12, 40, 8, r)
    host.free = list(cache._free)
    for new in ([5, 0, 17, 8], [1, 1, 1, 1], [3, 9, 0, 40]):
        batch = cache.extend(seqs, new)
        pos, slots, table, lengths, q, k, taken, status = host.plan(range(4), new, sum(new))
        assert status == 0 and all(taken)
        assert batch.pos.tolist() == pos and batch.slots.tolist() == slots and batch.lengths.tolist() == lengths
        assert batch.q_offsets.tolist() == q and batch.k_offsets.tolist() == k
        assert [row[: batch.table.size(1)] for row in table] == batch.table.tolist()
        assert host.free == cache._free
    before = list(host.free)
    host.plan(range(4), [6, 6, 0, 6], 18)
    host.trim(range(4), [n - d for n, d in zip(host.length, [6, 6, 0, 6])])
    assert host.free == before


def test_refusals():
    rows = torch.zeros(2, dtype=torch.int64)
    state = (torch.zeros(3, dtype=torch.int64), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(5, dtype=torch.int32), torch.zeros(1, dtype=torch.int64))
    plan = lambda rows=rows, new=rows, tokens=4, page=8, state=state, **kw: kernels.paged_plan(rows, new, tokens, page, *state, **kw)  # noqa: E731
    bad = lambda i, t: state[:i] + (t,) + state[i + 1:]  # noqa: E731
    for kw, match in ((dict(new=rows[:1]), "requests"), (dict(rows=rows[None]), "requests"), (dict(state=bad(0, state[0].int())), "length"),
                      (dict(state=bad(1, state[1].long())), "table"), (dict(state=bad(1, state[1][:2])), "table"),
                      (dict(state=bad(1, state[1].t().contiguous().t())), "table"), (dict(state=bad(2, state[2].long())), "free"),
                      (dict(state=bad(3, state[0])), "free_count"), (dict(page=0), "positions")):
        with pytest.raises(ValueError, match=match):
            plan(**kw)
        if "new" not in kw:
            kw = dict(kw)
            with pytest.raises(ValueError, match=match):
                kernels.paged_trim(kw.get("rows", rows), kw.get("rows", rows), kw.get("page", 8), *kw.get("state", state))
    with pytest.raises(ValueError, match="CUDA"):
        plan()


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,width,pages,page,requests,most,seed", [
    (1, 4, 3, 16, 1, 20, 0), (5, 6, 14, 8, 4, 20, 1), (40, 9, 200, 16, 40, 30, 2), (70, 30, 900, 7, 64, 50, 3), (600, 5, 1500, 16, 600, 9, 4),
    (3000, 12, 9000, 4, 2500, 12, 5), (8192, 3, 20000, 8, 8192, 5, 6), (33, 200, 3000, 1, 33, 60, 7), (3, 2, 0, 8, 3, 4, 8)])
def test_plan_and_trim_follow_the_rules(seqs, width, pages, page, requests, most, seed):
    r = random.Random(seed)
    host = Host(seqs, width, pages, page, r)
    state = host.tensors(DEV)
    for step in range(6):
        rows = r.sample(range(seqs), requests)
        new = [r.choice([0, 1, 1, r.randint(0, most)]) for _ in rows]
        spare = r.choice([0, 3])
        w = r.choice([width, max(1, width - 1)])
        want = host.plan(rows, new, sum(new) + spare, w)
        got = kernels.paged_plan(torch.tensor(rows, device=DEV), torch.tensor(new, device=DEV), sum(new) + spare, page, *state, width=w)
        same_plan(got, want)
        same_state(host, state)
        assert kernels.read_status() == want[-1] == 0
        rows = r.sample(range(seqs), requests)
        keep = [r.choice([0, n, r.randint(0, n)]) for n in (host.length[i] for i in rows)]
        assert host.trim(rows, keep) == 0
        kernels.paged_trim(torch.tensor(rows, device=DEV), torch.tensor(keep, device=DEV), page, *state)
        same_state(host, state)
        assert kernels.read_status() == 0


@pytest.mark.gpu
def test_bad_requests_are_refused_alone():
    r = random.Random(3)
    host = Host(6, 5, 30, 8, r)
    state = host.tensors(DEV)
    dev = lambda v: torch.tensor(v, device=DEV)  # noqa: E731
    for rows, new, tokens in (([0, 1, 2], [9, 20, 3], 32), ([0, 6, 1, -1], [1, 2, 3, 4], 10), ([3, 3, 4, 3], [5, 6, 7, 8], 26), ([0, 1], [2, -3], 4),
                              ([1, 2, 5], [4, 6, 2], 9), ([4, 4], [0, 0], 0), ([], [], 3), ([5, 0], [2**40, 1], 4), ([2, 0], [100, 1], 101)):
        want = host.plan(rows, new, tokens)
        got = kernels.paged_plan(dev(rows).long(), dev(new).long(), tokens, 8, *state)
        same_plan(got, want)
        same_state(host, state)
        assert kernels.read_status() == want[-1]
    for rows, keep in (([0, 0], [0, 1]), ([1, 9, -2], [3, 0, 0]), ([1, 2], [-1, 1]), ([3, 1], [2**50, 0]), ([4, 5, 3], [1, 0, 2])):
        status = host.trim(rows, keep)
        kernels.paged_trim(dev(rows), dev(keep), 8, *state)
        same_state(host, state)
        assert kernels.read_status() == status
    # more pages than the stack has room for (a sequence without any gives none back), and a stack that says it holds more than
    # there are
    state[3].fill_(30)
    before = [t.clone() for t in state]
    full = max(range(6), key=lambda i: host.length[i])
    assert host.length[0] == 0 and host.length[full] > 0
    kernels.paged_trim(dev([0]), dev([0]), 8, *state)
    assert kernels.read_status() == 0 and all(torch.equal(a, b) for a, b in zip(before, state))
    kernels.paged_trim(dev([0, full]), dev([0, 0]), 8, *state)
    assert kernels.read_status() == 1 and all(torch.equal(a, b) for a, b in zip(before, state))
    state[3].fill_(31)
    got = kernels.paged_plan(dev([5]), dev([9]), 9, 8, *state)
    assert kernels.read_status() == 1 and not bool(got[-1].any())


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    state = tuple(t.to(DEV) for t in (torch.zeros(3, dtype=torch.int64), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(5, dtype=torch.int32),
                                      torch.zeros(1, dtype=torch.int64)))
    rows = torch.zeros(2, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="tokens"):
        kernels.paged_plan(rows, rows, -1, 8, *state)
    with pytest.raises(ValueError, match="width"):
        kernels.paged_plan(rows, rows, 4, 8, *state, width=5)
    with pytest.raises(ValueError, match="at most 8192"):
        kernels.paged_plan(rows.new_zeros(8193), rows.new_zeros(8193), 4, 8, *state)
    with pytest.raises(ValueError, match="positions"):
        kernels.paged_plan(rows, rows, 4, 2**30, *state)
    with pytest.raises(ValueError, match="one device"):
        kernels.paged_plan(rows.cpu(), rows, 4, 8, *state)


@pytest.mark.gpu
def test_captured_steps():
    """A step's plan in a graph, replayed: every replay goes on from the state that it finds."""
    r = random.Random(4)
    host = Host(16, 20, 200, 8, r)
    state = host.tensors(DEV)
    rows, ones = torch.arange(16, device=DEV), torch.ones(16, dtype=torch.int64, device=DEV)
    kernels.paged_plan(rows, ones * 5, 80, 8, *state)
    host.plan(range(16), [5] * 16, 80)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = kernels.paged_plan(rows, ones, 16, 8, *state)
    for _ in range(9):
        graph.replay()
        torch.cuda.synchronize()
        same_plan(out, host.plan(range(16), [1] * 16, 16))
        same_state(host, state)
    assert kernels.read_status() == 0
