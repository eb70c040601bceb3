"""Page bounds, page selection and attention over page lists on a B200.

Bounds are copies of keys and selected pages are whole numbers: both are compared exactly, the
selection with scores in 64 bits. Attention outputs are compared per element: half a bf16 step of
the value (2^-8), the bf16 rounding of the weights (2^-8 of sum p |v|), and the fp32 scores: 128
products in 8 MMA steps, 2^-19 of sum |q k| in all, times scale and twice (weight and sum) as a
relative error of the weights, again of sum p |v|; exp2 and the joins add 2^-18.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE, D = 16, 128
INF = float("inf")


class Batch:
    """Requests of context lens[r] whose last q_lens[r] tokens are query rows; pages in random
    order, the slots behind each context and the unused pages hold NaN."""

    def __init__(self, lens, q_lens, hq, hkv, seed=0, spread=1.0, spare=3, width=0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.g, self.lens, self.q_lens, self.hq, self.hkv = g, lens, q_lens, hq, hkv
        need = [-(-n // PAGE) for n in lens]
        self.num_pages = sum(need) + spare
        ids = torch.randperm(self.num_pages, generator=g, device="cuda").int()
        self.page_table = torch.zeros(len(lens), max(max(need), width, 1), dtype=torch.int32, device="cuda")
        live = torch.zeros(self.num_pages, PAGE, dtype=torch.bool, device="cuda")
        at = 0
        for r, n in enumerate(need):
            self.page_table[r, :n] = ids[at:at + n]
            for p in range(n):
                live[ids[at + p], :min(PAGE, lens[r] - p * PAGE)] = True
            at += n
        k = torch.randn(self.num_pages, PAGE, hkv, D, generator=g, device="cuda") * spread
        v = torch.randn(self.num_pages, PAGE, hkv, D, generator=g, device="cuda")
        k[..., 5] += 3
        k[~live], v[~live] = float("nan"), float("nan")
        self.k = k.bfloat16().view(-1, hkv * D)
        self.v = v.bfloat16().view(-1, hkv * D)
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.T = sum(q_lens)
        self.q = torch.randn(self.T, hq, D, generator=g, device="cuda").bfloat16()
        self.indptr = torch.tensor([0] + torch.tensor(q_lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        self.bounds = torch.zeros(self.num_pages, hkv, 2, D, dtype=torch.bfloat16, device="cuda")
        self.max_q = max(q_lens)
        self.decode = all(n == 1 for n in q_lens)
        self.kw = {} if self.decode else dict(q_indptr=self.indptr, max_q_len=self.max_q)

    def all_bounds(self, ops):
        """Bounds of every page of every context."""
        whole = torch.tensor([0] + torch.tensor(self.lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        ops.kv_page_bounds_(self.bounds, self.k, self.page_table, self.seq_lens, self.hkv,
                            q_indptr=whole, max_q_len=max(max(self.lens), 1))

    def rows(self):
        """(request, row, position) of every query row."""
        t = 0
        for r, (n, m) in enumerate(zip(self.lens, self.q_lens)):
            for i in range(m):
                yield r, t, n - m + i
                t += 1

    def ref_select(self, top, sink, recent):
        G = self.hq // self.hkv
        ids = torch.full((self.T, self.hkv, top), -1, dtype=torch.int32)
        b = self.bounds.double()
        cache = {}
        for r, t, pos in self.rows():
            seen = pos // PAGE + 1 if pos >= 0 else 0
            for h in range(self.hkv):
                if seen <= top:
                    pick = list(range(seen))
                else:
                    if (r, h) not in cache:
                        cache = {(r, h): b[self.page_table[r].long(), h]}
                    lo, hi = cache[r, h][:, 0], cache[r, h][:, 1]
                    q = self.q[t, h * G:(h + 1) * G].double()
                    s = (q.clamp(min=0) @ hi.T + q.clamp(max=0) @ lo.T)
                    s = torch.where(s.isnan().any(0), INF, s.nan_to_num(nan=0.0, posinf=INF, neginf=-INF).amax(0))[sink:seen - recent]
                    order = torch.sort(s.cpu(), descending=True, stable=True).indices[:top - sink - recent]
                    pick = sorted(list(range(sink)) + [sink + i for i in order.tolist()] + list(range(seen - recent, seen)))
                ids[t, h, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
        return ids

    def ref_attend(self, ids, scale=D ** -0.5):
        G = self.hq // self.hkv
        out = torch.zeros(self.T, self.hq, D, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(out)
        ids = ids.cpu()
        k, v = self.k.view(-1, self.hkv, D), self.v.view(-1, self.hkv, D)
        for r, t, pos in self.rows():
            for h in range(self.hkv):
                pages = sorted({p for p in ids[t, h].tolist() if 0 <= p and p * PAGE <= pos})
                if not pages:
                    continue
                keys = torch.tensor([p * PAGE + o for p in pages for o in range(PAGE) if p * PAGE + o <= pos], device="cuda")
                slots = self.page_table[r, keys // PAGE].long() * PAGE + keys % PAGE
                q = self.q[t, h * G:(h + 1) * G].double()
                kk, vv = k[slots, h].double(), v[slots, h].double()
                p = torch.softmax(q @ kk.T * scale, -1)
                size = (q.abs() @ kk.abs().T).amax() * abs(scale) * 2 ** -18
                out[t, h * G:(h + 1) * G] = p @ vv
                tol[t, h * G:(h + 1) * G] = (p @ vv).abs() * 2 ** -8 + (p @ vv.abs()) * (2 ** -8 + size + 2 ** -18)
        return out, tol

    def select(self, ops, top, sink, recent, **kw):
        return ops.select_pages(self.q, self.bounds, self.page_table, self.seq_lens, max(max(self.lens), 1), top,
                                self.hq, self.hkv, sink_pages=sink, recent_pages=recent, **self.kw, **kw)

    def attend(self, ops, ids, **kw):
        return ops.paged_attention_pages(self.q, self.k, self.v, self.page_table, self.seq_lens, ids, self.hq,
                                         self.hkv, **self.kw, **kw)


def close(out, ref, tol):
    err = (out.double() - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


# ------------------------------------------------------------------ bounds
@pytest.mark.parametrize("lens,q_lens,hkv", [
    ([1], [1], 1), ([16, 17, 0, 33], [1, 1, 1, 1], 8), ([5, 100, 64], [5, 37, 0], 4), ([500], [500], 2),
    ([31, 32, 33, 300], [16, 17, 18, 2], 3)])
def test_bounds(cuda, lens, q_lens, hkv):
    from msgl import ops
    b = Batch(lens, q_lens, hkv, hkv, seed=len(lens))
    b.bounds.fill_(9.0)
    ops.kv_page_bounds_(b.bounds, b.k, b.page_table, b.seq_lens, hkv, **b.kw)
    ref = torch.full_like(b.bounds, 9.0)  # other pages stay
    keys = b.k.view(-1, PAGE, hkv, D)
    for r, (n, m) in enumerate(zip(lens, q_lens)):
        if n and m:
            for p in range((n - m) // PAGE, (n - 1) // PAGE + 1):
                phys = b.page_table[r, p]
                rows = keys[phys, :min(PAGE, n - p * PAGE)]
                ref[phys, :, 0], ref[phys, :, 1] = rows.amin(0), rows.amax(0)
    assert torch.equal(b.bounds, ref) and not bool(b.bounds.isnan().any())
    assert ops.device_error() == (0, 0)


def test_bounds_nan_and_infinite_keys(cuda):
    from msgl import ops
    b = Batch([40], [40], 2, 2, seed=1)
    slot = lambda i: int(b.page_table[0, i // PAGE]) * PAGE + i % PAGE
    b.k[slot(3), 7], b.k[slot(20), 130], b.k[slot(21), 130] = float("nan"), INF, -INF
    ops.kv_page_bounds_(b.bounds, b.k, b.page_table, b.seq_lens, 2, **b.kw)
    p0, p1 = b.page_table[0, 0], b.page_table[0, 1]
    assert bool(b.bounds[p0, 0, :, 7].isnan().all()) and int(b.bounds.isnan().sum()) == 2
    assert b.bounds[p1, 1, 0, 2] == -INF and b.bounds[p1, 1, 1, 2] == INF


# ------------------------------------------------------------------ selection
@pytest.mark.parametrize("lens,q_lens,hq,hkv,top,sink,recent", [
    ([1], [1], 8, 8, 1, 0, 1),
    ([900, 16, 17, 0, 1, 4099], [1] * 6, 16, 8, 8, 1, 2),
    ([5000, 3000], [1, 1], 8, 1, 64, 0, 1),
    ([2000], [1], 4, 4, 2, 1, 1),          # forced pages only
    ([700, 1200, 300], [130, 65, 1], 8, 4, 6, 1, 1),
    ([400, 50, 260], [400, 0, 7], 4, 4, 5, 0, 2),
    ([1000], [200], 16, 2, 40, 2, 3),
    ([20000], [3], 32, 4, 256, 1, 4),
    ([100000, 40000], [1, 2], 8, 1, 100, 1, 1),
    ([250000], [1], 8, 2, 1000, 2, 2),
    ([8000], [700], 8, 1, 64, 1, 1),
])
def test_selection(cuda, lens, q_lens, hq, hkv, top, sink, recent):
    from msgl import ops
    b = Batch(lens, q_lens, hq, hkv, seed=top)
    b.all_bounds(ops)
    ids = b.select(ops, top, sink, recent)
    assert torch.equal(ids.cpu(), b.ref_select(top, sink, recent))
    assert torch.equal(ids, b.select(ops, top, sink, recent))
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("kind", ["zero keys", "zero queries", "two kinds", "copies", "close", "huge", "inf", "nan"])
@pytest.mark.parametrize("pages,q_len", [(70, 1), (200, 330), (700, 1), (700, 310), (4000, 1), (12000, 2)])
def test_selection_ties_and_extremes(cuda, kind, pages, q_len):
    """Equal scores go to the lower page, near ones are told apart as in 64 bits, values that leave
    the fp32 range are still ordered, NaN ranks highest; at every way of spreading rows over warps,
    with more equal scores than are resolved in shared memory and with fewer."""
    from msgl import ops
    hq, hkv, top, n = 8, 2, 50, pages
    b = Batch([n * PAGE, 600], [q_len, 1], hq, hkv, seed=2)
    b.all_bounds(ops)
    pages = b.page_table[0, :n].long()
    if kind == "zero keys":
        b.bounds.zero_()
    elif kind == "zero queries":
        b.q.zero_()
    elif kind == "two kinds":
        b.bounds[pages[::2]] = b.bounds[pages[0]].clone()
        b.bounds[pages[1::2]] = b.bounds[pages[1]].clone()
    elif kind == "copies":
        b.bounds[pages[10:]] = b.bounds[pages[:60].repeat(n // 60 + 1)[:n - 10]]
    elif kind == "close":  # one element apart by a last place of a small bound
        b.bounds[pages] = b.bounds[pages[0]].clone()
        b.bounds[pages, :, :, 17] = (0.0078125 * (1 + torch.randint(0, 128, (n, hkv, 2), generator=b.g, device="cuda") / 128)).bfloat16()
        b.bounds[pages, :, 1, 17] = b.bounds[pages, :, 0, 17]
    elif kind == "huge":
        b.bounds.mul_(1e36)
        b.q.mul_(1e3)
    elif kind == "inf":
        b.bounds[pages[::3], 0, 1, 4] = INF
        b.bounds[pages[::5], 1, 0, 9] = -INF
        b.q[:, :, 4] = b.q[:, :, 4].abs() + 0.5
        b.q[:, :, 9] = -b.q[:, :, 9].abs() - 0.5
    else:
        b.bounds[pages[5:n - 40:7]] = float("nan")
    ids = b.select(ops, top, 1, 2)
    if kind != "inf":
        assert torch.equal(ids.cpu(), b.ref_select(top, 1, 2))
    else:  # infinite scores tie: the lower of the infinite pages come first
        pos = n * PAGE - q_len
        for h, step in ((0, 3), (1, 5)):
            seen = pos // PAGE + 1
            want = [p for p in range(step, seen - 2, step)][:47]
            got = [p for p in ids[0, h].tolist() if 0 < p < seen - 2]
            assert got[:len(want)] == want if len(want) == 47 else set(want) <= set(got)
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("times", [1e3, 1e36])
@pytest.mark.parametrize("n,m,hq,hkv", [(3200, 330, 8, 2), (16384, 512, 8, 2), (5000, 700, 4, 4), (3200, 300, 8, 1)])
def test_large_bounds_at_the_newest_pages(cuda, times, n, m, hq, hkv):
    """Near scores of a few pages whose bounds are much larger than the others', behind what the chunk's
    earlier rows see: their rows tell them apart by their own magnitude, whichever tile of rows was
    scored last."""
    from msgl import ops
    b = Batch([n], [m], hq, hkv, seed=33)
    b.all_bounds(ops)
    pages = b.page_table[0].long()
    end = (n - 1) // PAGE + 1
    # one element apart by a last place of a small bound
    large = pages[end - 18:end - 3]
    b.bounds[large] = (b.bounds[pages[0]].float() * times).bfloat16()
    last_place = torch.randint(0, 128, (15, hkv, 1), generator=b.g, device="cuda") / 128
    b.bounds[large, :, :, 17] = (times / 131072 * (1 + last_place)).bfloat16()
    if times > 1e30:
        b.q.mul_(1e3)  # products beyond fp32
    ref = b.ref_select(6, 1, 2)
    for _ in range(5):
        assert torch.equal(b.select(ops, 6, 1, 2).cpu(), ref)
    assert ops.device_error() == (0, 0)


def test_selection_in_several_passes(cuda):
    """More query rows than one pass holds (256 MB: 1024 rows of 2048 pages, 8 heads)."""
    from msgl import ops
    b = Batch([32768], [1500], 8, 8, seed=5)
    b.all_bounds(ops)
    assert ops.select_pages_workspace(1500, 32768, 8).numel() == 256 * 2 ** 20
    ids = b.select(ops, 20, 1, 1).cpu()
    # every row by a product per head in 64 bits
    pos = 32768 - 1500 + torch.arange(1500, device="cuda")
    seen = pos // PAGE + 1
    page = torch.arange(2048, device="cuda")
    for h in range(8):
        lo, hi = b.bounds[b.page_table[0].long(), h].double().unbind(1)
        q = b.q[:, h].double()
        s = q.clamp(min=0) @ hi.T + q.clamp(max=0) @ lo.T
        s = torch.where((page[None] == 0) | (page[None] == seen[:, None] - 1), INF, torch.where(page[None] < seen[:, None], s, -INF))
        ref = torch.sort(s, dim=1, descending=True, stable=True).indices[:, :20].sort(1).values
        assert torch.equal(ids[:, h].long(), ref.cpu()), h


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("lens,q_lens,hq,hkv,top", [
    ([1], [1], 8, 8, 1), ([17, 16, 0, 1, 900], [1] * 5, 16, 8, 8), ([3000, 200], [1, 1], 8, 1, 70),
    ([700, 130, 90], [70, 33, 1], 8, 4, 9), ([300, 40], [300, 0], 4, 4, 6), ([600, 21], [90, 21], 16, 2, 12),
    ([520], [45], 32, 8, 10), ([900, 330, 50], [300, 70, 3], 8, 4, 20), ([700], [280], 16, 2, 9),
    ([400, 300], [200, 120], 4, 4, 7), ([500, 600], [260, 33], 8, 1, 11)])
def test_attention_over_selected_pages(cuda, lens, q_lens, hq, hkv, top):
    from msgl import ops
    b = Batch(lens, q_lens, hq, hkv, seed=top + 1)
    b.all_bounds(ops)
    ids = b.select(ops, top, 0, 1)
    out = b.attend(ops, ids)
    close(out, *b.ref_attend(ids))
    assert torch.equal(out, b.attend(ops, ids, max_seq_len=max(max(lens), 1)))
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("m", [1, 30, 300])
@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 2), (8, 1)])
def test_cancelling_values(cuda, m, hq, hkv):
    """Values that nearly cancel over keys of much the same weight: what the weights are rounded by
    shows in the result. Two bf16 terms leave 2^-16 of each; fp32 scores and exp2 as above (size +
    2^-18), and the sums over n keys are off by at most 2^-22 of their magnitude a step of 16 products,
    two such steps (terms) a page, and as much again for the joins of up to 64 parts."""
    from msgl import ops
    n, top = 400 + m, 6
    b = Batch([n], [m], hq, hkv, seed=35)
    b.q.mul_(0.125)
    slots = (b.page_table[0].long()[:, None] * PAGE + torch.arange(PAGE, device="cuda")).view(-1)[:n]
    v = b.v[slots]
    v[1::2] = -v[:n // 2 * 2:2]
    b.v[slots] = v
    b.all_bounds(ops)
    ids = b.select(ops, top, 1, 2)
    ref, tol = b.ref_attend(ids)
    weight = (tol - ref.abs() * 2 ** -8)                 # (2^-8 + size + 2^-18) sum p |v|
    keys = b.k[slots].view(n, hkv, D).double().abs()
    size = max(float((b.q[:, h * hq // hkv:(h + 1) * hq // hkv].double().abs() @ keys[:, h].T).amax())
               for h in range(hkv)) * D ** -0.5 * 2 ** -18
    fine = (2 ** -16 + size + 2 ** -18 + (2 * top + 64) * 2 ** -22) / 2 ** -8
    close(b.attend(ops, ids), ref, ref.abs() * 2 ** -8 + weight * fine)
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("m", [1, 30, 300])
def test_infinite_values_that_rows_see(cuda, m):
    """An infinite value gives infinities of its sign in its dimension to every row that lists its page,
    and nothing to the others."""
    from msgl import ops
    n = 200 + m
    b = Batch([n], [m], 8, 2, seed=36)
    ids = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda").repeat(m, 2, 1)
    ids[1::2, :, 1] = 4
    slot = int(b.page_table[0, 3]) * PAGE + 7
    ref, tol = b.ref_attend(ids)
    b.v[slot, 9], b.v[slot, 128 + 40] = INF, -INF
    out = b.attend(ops, ids).double()
    hit = torch.arange(m, device="cuda") % 2 == 0
    assert bool((out[hit, :4, 9] == INF).all()) and bool((out[hit, 4:, 40] == -INF).all())
    at = torch.zeros_like(out, dtype=torch.bool)
    at[hit, :4, 9], at[hit, 4:, 40] = True, True
    close(out[~at], ref[~at], tol[~at])


@pytest.mark.parametrize("n,m,hq,hkv", [(900, 800, 8, 1), (500, 400, 8, 8), (600, 512, 16, 16), (700, 290, 4, 4)])
def test_tiles_shared_by_ctas(cuda, n, m, hq, hkv):
    """Tiles of one CTA, of two and of four, with one and two groups of pages among a CTA's warps."""
    from msgl import ops
    b = Batch([n], [m], hq, hkv, seed=31)
    b.all_bounds(ops)
    ids = b.select(ops, 9, 1, 1)
    out = b.attend(ops, ids)
    close(out, *b.ref_attend(ids))
    assert torch.equal(out, b.attend(ops, ids))
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [40, 7, 90], [220, 33, 40]])
@pytest.mark.parametrize("hq,hkv", [(8, 8), (8, 4), (16, 4), (16, 2)])
def test_attention_over_any_lists(cuda, q_lens, hq, hkv):
    """Lists of the caller's: unsorted, with repeats and gaps, empty rows, different per row; other
    pages hold NaN where only some rows see them."""
    from msgl import ops
    lens = [400, 333, 500]
    b = Batch(lens, q_lens, hq, hkv, seed=9)
    top = 11
    ids = torch.full((b.T, hkv, top), -1, dtype=torch.int32)
    g = torch.Generator().manual_seed(3)
    for r, t, pos in b.rows():
        for h in range(hkv):
            if (t + h) % 5 == 4:
                continue  # an empty list
            n = pos // PAGE + 1
            ids[t, h] = torch.randint(-2, n, (top,), generator=g).int()
            if t % 3 == 0:
                ids[t, h, 3] = n - 1
    for bad in (float("nan"), INF):
        # a page that even rows never list holds bad values in kv head 0, as does one that later rows see
        rows = [(r, t, pos) for r, t, pos in b.rows() if r == 2]
        for r, t, pos in rows:
            l = ids[t, 0]
            if t % 2 == 0:
                l[l == 4] = 5
            else:
                l[0] = 4
        slot = int(b.page_table[2, 4]) * PAGE
        b.v[slot:slot + PAGE, :D] = bad
        b.k[slot:slot + 3, :D] = bad
        out = b.attend(ops, ids.cuda())
        ref, tol = b.ref_attend(ids)
        G = hq // hkv
        hit = torch.zeros(b.T, hq, dtype=torch.bool, device="cuda")
        for r, t, pos in rows:
            hit[t, :G] = bool((ids[t, 0] == 4).any())
        close(out[~hit], ref[~hit], tol[~hit])
        assert not bool(out[hit].isfinite().all(-1).any()) if bool(hit.any()) else True
    empty = (ids < 0).all(-1).repeat_interleave(hq // hkv, 1)
    assert bool((out.cpu()[empty] == 0).all())
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("m", [40, 300])
def test_rows_do_not_see_later_tokens(cuda, m):
    """NaN and infinite keys and values of a chunk's later tokens do not reach the earlier rows, row by
    row and in tiles of rows."""
    from msgl import ops
    n = 170 + m
    b = Batch([n], [m], 8, 2, seed=12)
    b.all_bounds(ops)
    ids = b.select(ops, 6, 1, 2)
    clean = b.attend(ops, ids)
    for bad in (float("nan"), INF):
        for cut in (171, 175, 176, 190, n - 1):  # positions from `cut` on hold bad values
            k, v = b.k.clone(), b.v.clone()
            keys = torch.arange(cut, n, device="cuda")
            slots = b.page_table[0, keys // PAGE].long() * PAGE + keys % PAGE
            b.k[slots], b.v[slots] = bad, bad
            got = b.attend(ops, ids)
            b.k, b.v = k, v
            assert torch.equal(got[:cut - 170], clean[:cut - 170]), cut


def test_listed_pages_behind_the_row_and_bad_page_table(cuda):
    from msgl import ops
    b = Batch([100, 60], [1, 1], 8, 2, seed=13)
    ids = torch.tensor([[0, 2, 6, 7], [3, 1, 4, -1]], dtype=torch.int32, device="cuda").repeat_interleave(2, 0).view(2, 2, 4).contiguous()
    out = b.attend(ops, ids)  # pages 7 of request 0 and 4 of request 1 do not exist
    assert ops.device_error() == (6, 803)
    close(out, *b.ref_attend(ids))
    b.page_table[1, 1] = b.num_pages
    b.k.nan_to_num_(), b.v.nan_to_num_()
    ids[0, :, 3], ids[1, :, 2] = -1, -1
    out2 = b.attend(ops, ids)
    assert ops.device_error() == (6, 802)
    assert torch.equal(out2[0], out[0])
    b.all_bounds(ops)
    assert ops.device_error() == (6, 802)
    b.select(ops, 2, 0, 1)
    assert ops.device_error() == (6, 802)


@pytest.mark.parametrize("first,second", [(20, 12), (400, 40)])
def test_contexts_and_rows_outside_what_was_announced(cuda, first, second):
    from msgl import ops
    b = Batch([first + 180, second + 138], [first, second], 8, 2, seed=14)
    b.all_bounds(ops)
    ids = b.select(ops, 4, 1, 1)
    b.kw = dict(q_indptr=b.indptr, max_q_len=second)  # request 0 has `first` rows
    got = b.select(ops, 4, 1, 1)
    assert ops.device_error() == (6, 801)
    assert torch.equal(got[:second], ids[:second]) and torch.equal(got[first:], ids[first:])
    assert bool((got[second:first] == -1).all())
    out = b.attend(ops, ids)
    assert ops.device_error() == (6, 801) and bool((out[:first] == 0).all()) and not bool((out[first:] == 0).any())
    b.seq_lens[1] = 10 ** 6
    b.kw = dict(q_indptr=b.indptr, max_q_len=first)
    b.select(ops, 4, 1, 1)
    assert ops.device_error() == (6, 800)
    b.attend(ops, ids)
    assert ops.device_error()[0] == 6
    b.all_bounds(ops)
    assert ops.device_error() == (6, 800)


@pytest.mark.parametrize("first", [20, 330])
def test_rows_behind_the_last_request_stay(cuda, first):
    from msgl import ops
    b = Batch([first + 180, 40], [first, 3], 8, 2, seed=15)
    b.all_bounds(ops)
    ids0 = b.select(ops, 4, 1, 1)
    out0 = b.attend(ops, ids0)
    b.q = torch.cat([b.q, torch.full((5, 8, D), float("nan"), device="cuda").bfloat16()])
    n = first + 3
    ids = torch.full((n + 5, 2, 4), 77, dtype=torch.int32, device="cuda")
    out = torch.full((n + 5, 8, D), 3.0, device="cuda").bfloat16()
    b.select(ops, 4, 1, 1, out=ids)
    assert torch.equal(ids[:n], ids0) and bool((ids[n:] == 77).all())
    b.attend(ops, ids, out=out)
    assert torch.equal(out[:n], out0) and bool((out[n:] == 3).all())
    assert ops.device_error() == (0, 0)


def test_positions_before_the_context(cuda):
    """More query rows than context tokens: the rows before position 0 see nothing."""
    from msgl import ops
    b = Batch([10], [10], 4, 4, seed=16)
    b.all_bounds(ops)
    b.seq_lens.fill_(6), b.lens.__setitem__(0, 6)
    ids = b.select(ops, 2, 0, 1)
    assert bool((ids[:4] == -1).all()) and bool((ids[4:, :, 0] == 0).all()) and bool((ids[4:, :, 1] == -1).all())
    out = b.attend(ops, ids)
    assert bool((out[:4] == 0).all())
    close(out, *b.ref_attend(ids))


def test_offsets_past_32_bits(cuda):
    """A pool of more than 2^31 elements: pages at its end."""
    from msgl import ops
    hkv, pages = 8, 140000  # 140000 * 16 * 1024 = 2.29e9 elements
    k = torch.zeros(pages * PAGE, hkv * D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    bounds = torch.zeros(pages, hkv, 2, D, dtype=torch.bfloat16, device="cuda")
    b = Batch([640], [1], 16, hkv, seed=17)
    small, big = b.page_table[0].long(), pages - 1 - torch.arange(40, device="cuda") * 2
    k.view(pages, -1)[big], v.view(pages, -1)[big] = b.k.view(b.num_pages, -1)[small], b.v.view(b.num_pages, -1)[small]
    b.all_bounds(ops)
    ids = b.select(ops, 9, 1, 1)
    out = b.attend(ops, ids)
    b.k, b.v, b.bounds, b.page_table = k, v, bounds, big.int()[None].contiguous()
    b.all_bounds(ops)
    assert torch.equal(b.select(ops, 9, 1, 1), ids)
    assert torch.equal(b.attend(ops, ids), out)
    assert ops.device_error() == (0, 0)


def test_one_step_of_all_operators(cuda):
    """As a decode step uses them, captured once and replayed: adapters on the qkv projection's
    partials, three-axis rotation and append, bounds, selection, attention."""
    from msgl import ops
    hq, hkv, K, B, R, top = 16, 4, 512, 3, 8, 6
    N = (hq + 2 * hkv) * D
    lens = [333, 150, 48]
    b = Batch(lens, [1] * B, hq, hkv, seed=18, width=32)
    b.k.nan_to_num_(nan=0.0), b.v.nan_to_num_(nan=0.0)
    b.all_bounds(ops)
    g = b.g
    rn = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std).bfloat16()
    x, w = rn(B, K), rn(N, K, std=K ** -0.5)
    la, lb, sc = rn(2, R, K, std=K ** -0.5), rn(2, N, R, std=R ** -0.5), torch.ones(2, device="cuda")
    ad = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    ang = torch.arange(1024, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(64, dtype=torch.float64) / 64)
    tab = torch.cat([ang.cos(), ang.sin()], 1).float().cuda()
    one = torch.ones(D, dtype=torch.bfloat16, device="cuda")
    pos = (b.seq_lens - 1).expand(3, B)
    at = (b.seq_lens - 1).long()
    slots = (b.page_table[torch.arange(B, device="cuda"), at // PAGE] * PAGE + at % PAGE).int()
    S = ops.gemm_partials_splits(B, N, K)
    parts = torch.empty(S + 1, B, N, device="cuda")
    lws, sws = ops.lora_workspace(B, K, R), ops.select_pages_workspace(B, 512, hkv)
    q = torch.empty(B, hq, D, dtype=torch.bfloat16, device="cuda")
    ids = torch.empty(B, hkv, top, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)

    def step():
        ops.linear_partials(x, w, S, out=parts[:S])
        ops.lora_partial(x, la, lb, sc, ad, workspace=lws, out=parts[S])
        ops.qknorm_mrope_store_kv_partials(parts, b.k, b.v, pos, slots, tab, one, one, hq, hkv, 1e-6,
                                           (24, 20, 20), True, out=q)
        ops.kv_page_bounds_(b.bounds, b.k, b.page_table, b.seq_lens, hkv)
        ops.select_pages(q, b.bounds, b.page_table, b.seq_lens, 512, top, hq, hkv, 1, 1, workspace=sws, out=ids)
        ops.paged_attention_pages(q, b.k, b.v, b.page_table, b.seq_lens, ids, hq, hkv, max_seq_len=512, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    x.copy_(rn(B, K))
    graph.replay()
    torch.cuda.synchronize()
    qkv = x.double() @ w.double().T
    for r, a in enumerate(ad.tolist()):
        if a >= 0:
            qkv[r] += (x[r].double() @ la[a].double().T) @ lb[a].double().T
    # v rows of this step (one bf16 rounding; fp32 sums of 512 products of magnitude 14 in all, 2^-22
    # a step of 16 and 30 more additions: 2e-4), then selection and attention from the stored state
    v = qkv[:, -hkv * D:]
    assert bool(((b.v[slots.long()].double() - v).abs() <= v.abs() * 2 ** -8 + 2e-4).all())
    keys = b.k.view(-1, PAGE, hkv, D)
    for r, n in enumerate(lens):
        phys = b.page_table[r, (n - 1) // PAGE]
        rows = keys[phys, :(n - 1) % PAGE + 1]
        assert torch.equal(b.bounds[phys, :, 0], rows.amin(0)) and torch.equal(b.bounds[phys, :, 1], rows.amax(0))
    b.q = q
    assert torch.equal(ids.cpu(), b.ref_select(top, 1, 1))
    close(out, *b.ref_attend(ids))
    eager = out.clone()
    step()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)  # same bits eagerly
    assert ops.device_error() == (0, 0)


def test_full_lists_equal_dense_attention(cuda):
    """With every page listed the operator is the framework's decode / extend attention."""
    from msgl import ops
    b = Batch([300, 77], [1, 1], 16, 4, seed=19)
    b.all_bounds(ops)
    b.k.nan_to_num_(nan=0.0), b.v.nan_to_num_(nan=0.0)
    ids = b.select(ops, 20, 0, 1)
    out = b.attend(ops, ids)
    dense = ops.paged_attention_decode(b.q, b.k, b.v, b.page_table, b.seq_lens, 300, 16, 4)
    ref, tol = b.ref_attend(ids)
    close(out, ref, tol), close(dense.view_as(out), ref, tol)
    b = Batch([300, 77], [50, 77], 16, 4, seed=20)
    b.all_bounds(ops)
    b.k.nan_to_num_(nan=0.0), b.v.nan_to_num_(nan=0.0)
    ids = b.select(ops, 20, 0, 1)
    out = b.attend(ops, ids)
    dense = ops.paged_attention_extend(b.q, b.k, b.v, b.page_table, b.seq_lens, b.indptr, 77, 16, 4)
    ref, tol = b.ref_attend(ids)
    close(out, ref, tol), close(dense.view_as(out), ref, tol)


def test_chunk_contexts_longer_than_a_window(cuda):
    """Tiles whose context spans several windows of 2048 pages, with lists that touch some of them."""
    from msgl import ops
    b = Batch([100000], [270], 4, 1, seed=21)
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 6232, (270, 1, 12), generator=g).int()
    ids[::3, 0, :6] = torch.tensor([0, 2047, 2048, 4095, 4096, 6231], dtype=torch.int32)
    ids[5:40, 0] = torch.randint(2048, 4096, (35, 12), generator=g).int()
    close(b.attend(ops, ids.cuda()), *b.ref_attend(ids))
    assert ops.device_error() == (0, 0)


def test_largest_context_and_list(cuda):
    from msgl import ops
    b = Batch([524288, 40], [1, 1], 2, 1, seed=22)
    b.all_bounds(ops)
    ids = b.select(ops, 1024, 3, 5)
    assert torch.equal(ids.cpu(), b.ref_select(1024, 3, 5))
    close(b.attend(ops, ids), *b.ref_attend(ids))
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("m", [1, 700])
def test_nan_queries(cuda, m):
    """A row of NaN ties all its pages (the lowest are taken) and gives NaN; its neighbours' lists stay
    and their outputs stay right (in tiles not bit for bit: where a tile's joined list is cut into
    shares follows from all of its rows' lists)."""
    from msgl import ops
    b = Batch([9000, 9000], [m, m], 8, 2, seed=23)
    b.all_bounds(ops)
    ids0 = b.select(ops, 10, 1, 2)
    out0 = b.attend(ops, ids0)
    b.q[0, :4] = float("nan")
    ids = b.select(ops, 10, 1, 2)
    last = (9000 - m) // PAGE
    assert ids[0, 0].tolist() == list(range(8)) + [last - 1, last]
    ids0[0, 0] = ids[0, 0]
    assert torch.equal(ids, ids0)
    out = b.attend(ops, ids)
    assert bool(out[0, :4].isnan().all())
    ref, tol = b.ref_attend(ids)
    close(out[1:], ref[1:], tol[1:]), close(out[0, 4:], ref[0, 4:], tol[0, 4:]), close(out0[1:], ref[1:], tol[1:])


def test_tensors_elsewhere_are_refused(cuda):
    from msgl import ops
    b = Batch([40], [1], 4, 2, seed=24)
    with pytest.raises(ValueError):
        ops.kv_page_bounds_(b.bounds, b.k.cpu(), b.page_table, b.seq_lens, 2)
    with pytest.raises(ValueError):
        ops.kv_page_bounds_(b.bounds, b.k, b.page_table, b.seq_lens.long(), 2)
    with pytest.raises(ValueError):
        ops.select_pages(b.q.transpose(1, 2), b.bounds, b.page_table, b.seq_lens, 40, 2, 4, 2)
    with pytest.raises(AssertionError):
        ops.select_pages(b.q, b.bounds, b.page_table, b.seq_lens, 40, 2, 4, 2, max_q_len=2)
    with pytest.raises(ValueError):
        ops.paged_attention_pages(b.q, b.k, b.v.cpu(), b.page_table, b.seq_lens,
                                  torch.zeros(1, 2, 1, dtype=torch.int32, device="cuda"), 4, 2)
