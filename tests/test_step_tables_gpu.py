"""Step tables on a B200, against the page pool's own bookkeeping on lists (whole numbers: equal)."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
PAGE = 16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Pool:
    """A free list and page lists of B requests, and their copies on the GPU."""

    def __init__(self, B, width, pages, seed, page=PAGE):
        self.rng, self.B, self.width, self.page = random.Random(seed), B, width, page
        ids = list(range(pages))
        self.rng.shuffle(ids)
        self.free, self.capacity, self.rows = ids, pages, [[] for _ in range(B)]
        self.table = torch.full((B, width), -7, dtype=torch.int32, device="cuda")
        self.held = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.stack = ints(ids) if ids else torch.zeros(0, dtype=torch.int32, device="cuda")
        self.top = ints([pages])
        self.entries = [[-7] * width for _ in range(B)]

    def step(self, kept, new, tokens):
        """The host's way."""
        need = [-(-(k + n) // self.page) for k, n in zip(kept, new)]
        for row, m in zip(self.rows, need):
            while len(row) > m:
                self.free.append(row.pop())
        for row, m, e in zip(self.rows, need, self.entries):
            while len(row) < m:
                e[len(row)] = self.free[-1]
                row.append(self.free.pop())
        indptr = [0]
        for n in new:
            indptr.append(indptr[-1] + n)
        pos = [k + i for k, n in zip(kept, new) for i in range(n)]
        slots = [row[(k + i) // self.page] * self.page + (k + i) % self.page for row, k, n in zip(self.rows, kept, new) for i in range(n)]
        pad = tokens - len(pos)
        return ([k + n for k, n in zip(kept, new)], indptr, pos + [0] * pad, slots + [-1] * pad,
                [e - 1 if n else -1 for e, n in zip(indptr[1:], new)])

    def call(self, kept, new, tokens=None, out=None):
        from msgl import ops
        return ops.step_tables(ints(kept), ints(new), self.table, self.held, self.stack, self.top, tokens, self.page, out=out)

    def check(self, kept, new, tokens):
        got = self.call(kept, new, tokens)
        want = self.step(kept, new, tokens)
        for g, w in zip(got, want):
            assert g.tolist() == w
        assert int(self.top) == len(self.free) and self.stack[:len(self.free)].tolist() == self.free
        assert self.held.tolist() == [len(r) for r in self.rows] and self.table.tolist() == self.entries
        return got


@pytest.mark.parametrize("B", [1, 2, 31, 64, 300, 1024, 1025, 2500])
def test_a_life_of_requests(cuda, B):
    """Prompts, drafted rows, rejections, requests that end and others in their place."""
    from msgl import ops
    p = Pool(B, 12, B * 12 + 3, seed=B)
    kept = [0] * B
    for step in range(8):
        new = []
        for r in range(B):
            if kept[r] and p.rng.random() < 0.15:
                kept[r] = 0  # finished; a new prompt, or nothing, takes its place
            room = 12 * PAGE - kept[r]
            new.append(min(room, p.rng.choice([0, 1, 1, 5, p.rng.randint(0, 60)])))
        p.check(kept, new, sum(new) + (step % 3) * 7)
        kept = [k + p.rng.randint(0, n) for k, n in zip(kept, new)]
    p.check([0] * B, [0] * B, 0)
    assert sorted(p.free) == list(range(p.capacity)) and ops.device_error() == (0, 0)


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("kept,new", [([0], [1]), ([0], [2048]), ([0, 100], [2049, 5]), ([31, 0, 5], [1, 0, 9000]), ([0] * 5, [1, 1000, 0, 30000, 7])])
def test_prompts(cuda, page, kept, new):
    """Long prompts (rows shared by a cluster), several page sizes; then all but the first request's pages go back."""
    width = -(-max(k + n for k, n in zip(kept, new)) // page)
    p = Pool(len(kept), width, sum(-(-(k + n) // page) for k, n in zip(kept, new)), seed=page, page=page)
    p.check(kept, [0] * len(kept), 0)
    p.check(kept, new, sum(new))
    assert int(p.top) == 0
    p.check([k if r == 0 else 0 for r, k in enumerate(kept)], [new[0]] + [0] * (len(kept) - 1), new[0] + 3)


def test_rejected_drafts_give_and_take_the_same_page(cuda):
    p = Pool(2, 4, 8, seed=1)
    p.check([0, 0], [15, 3], 18)
    p.check([15, 3], [6, 6], 12)
    page = int(p.table[0, 1])
    p.check([16, 5], [0, 0], 0)   # one token accepted: the second page is not needed
    assert int(p.held[0]) == 1
    p.check([16, 5], [6, 6], 12)
    assert int(p.table[0, 1]) == page


@pytest.mark.parametrize("B", [3, 1500])
@pytest.mark.parametrize("bad,site", [("stack", 710), ("negative", 711), ("long", 711), ("wide", 711), ("rows", 712), ("over", 713), ("top", 713)])
def test_nothing_is_written_where_it_does_not_fit(cuda, B, bad, site):
    from msgl import ops
    p = Pool(B, 4, 4 * B, seed=2)
    p.check([0] * B, [20] * B, 20 * B)
    kept, new, tokens = [20] * B, [1] * B, B
    if bad == "stack":
        p.top.fill_(1)
        new = [13] * B
        tokens = 13 * B
    elif bad == "negative":
        kept[B - 1] = -1
    elif bad == "long":
        new[B // 2], tokens = 45, 100 + B
    elif bad == "wide":
        p.held[B - 1] = 5
    elif bad == "rows":
        tokens = B - 1
    elif bad == "over":
        p.top.fill_(4 * B)
        kept, new = [0] * B, [0] * B
    elif bad == "top":
        p.top.fill_(-1)
    before = [t.clone() for t in (p.table, p.held, p.stack, p.top)]
    out = ops.StepTables(*(torch.full((n,), -5, dtype=torch.int32, device="cuda") for n in (B, B + 1, tokens, tokens, B)))
    p.call(kept, new, out=out)
    code, info = ops.device_error()
    assert info == site and code == (7 if site == 710 else 6)
    assert all(bool((t == -5).all()) for t in out)
    assert all(torch.equal(a, b) for a, b in zip(before, (p.table, p.held, p.stack, p.top)))


def test_one_row_each_is_decode_advance(cuda):
    """With one row a request: what msgl_decode_advance writes from the same stack."""
    from msgl import ops
    lens = [16, 5, 31, 32, 1]
    p = Pool(5, 8, 40, seed=3)
    p.check([0] * 5, lens, sum(lens))
    table, seq, stack, top = p.table.clone(), ints(lens), p.stack.clone(), p.top.clone()
    ids, pos, slots = (torch.zeros(5, dtype=torch.int32, device="cuda") for _ in range(3))
    ops.decode_advance(ints([1, 2, 3, 4, 5]), ids, pos, slots, table, seq, stack, top)
    got = p.check(lens, [1] * 5, 5)
    assert torch.equal(got.seq_lens, seq) and torch.equal(got.positions, pos) and torch.equal(got.slot_mapping, slots)
    assert torch.equal(p.table, table) and torch.equal(p.top, top)


def test_graph_replay(cuda):
    """A captured step replays on new lengths, padded to its size."""
    from msgl import ops
    p = Pool(6, 10, 60, seed=4)
    kept, new = ints([0] * 6), ints([3] * 6)
    out = ops.step_tables_buffers(6, 3000)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.step_tables(kept, new, p.table, p.held, p.stack, p.top, out=out)
        for k, n in (([0] * 6, [3, 0, 100, 17, 16, 1]), ([3, 0, 90, 17, 2, 1], [6] * 6), ([0, 6, 96, 20, 0, 7], [0, 1, 0, 5, 0, 1])):
            kept.copy_(ints(k)), new.copy_(ints(n))
            g.replay()
            s.synchronize()
            assert [t.tolist() for t in out] == list(p.step(k, n, 3000))
            assert p.stack[:len(p.free)].tolist() == p.free and int(p.top) == len(p.free)
