"""Append to and attention over the 8-bit key / value pool on a B200, against the definitions in 64 bits.

Tolerances. Appended values are the nearest e4m3 value of something that fp32 knows to 2^-17 of the
rotated pair's magnitude (the norm's scale 2^-18, the rotation 2^-22): half a step of e4m3 (2^-4 of the value, 2^-10
of the scale below its normal range) plus that; copies of bf16 are exact. The attention is compared with softmax
over what the pool holds: half a bf16 step of the result (2^-8); f16 weights, 2^-11 of each and 2^-25 of the
largest below f16's normal range; logits in fp32 from exact products, off by 2^-17 of sum |q k| at
most (128 additions), which is as much of a weight and twice that of a normalised one.
"""
import math

import pytest
import torch

from kv8_plain import D, PAGE, decode, exponent, fill, ints, page_table, places, pool_values, quantise

pytestmark = pytest.mark.gpu
EPS = 1e-6
NAN = float("nan")


def table(n):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(64, dtype=torch.float64) / 64)
    return torch.cat([ang.cos(), ang.sin()], 1).float().cuda()


# ------------------------------------------------------------------ append
def turned(rows, pos, tab, w):
    """Normed and rotated heads (float64) and the magnitude of the pairs."""
    y = rows / torch.sqrt(rows.square().mean(-1, keepdim=True) + EPS) * w.double()
    row = tab.double()[pos.long()][:, None]
    lo, hi, c, s = y[..., :64], y[..., 64:], row[..., :64], row[..., 64:]
    return torch.cat([lo * c - hi * s, lo * s + hi * c], -1), (lo.abs() + hi.abs()).repeat(1, 1, 2)


class Append:
    """A pool with earlier tokens of B requests and the rows that a call appends to them."""

    def __init__(self, kept, new, hq, hkv, parts=0, seed=0, size=1.0):
        self.g = g = torch.Generator("cuda").manual_seed(seed)
        self.kept, self.new, self.hq, self.hkv, self.parts = kept, new, hq, hkv, parts
        self.lens = [a + b for a, b in zip(kept, new)]
        self.table, pages = page_table([max(1, n) for n in self.lens], g)
        self.kv8 = torch.randint(0, 256, (pages, hkv, 4096), generator=g, device="cuda").to(torch.uint8)  # any bytes
        self.scales = torch.randint(0, 255, (pages, hkv, 2), generator=g, device="cuda").to(torch.uint8)
        held = [self.table[r, :-(-n // PAGE)] for r, n in enumerate(kept) if n]
        if held:
            held = torch.cat(held).long()
            for kind in (0, 1):
                fill(self.kv8, self.scales, held, kind, 3 * size * torch.randn(len(held), hkv, PAGE, D, generator=g, device="cuda", dtype=torch.float64))
        self.T, self.nh = sum(new), hq + 2 * hkv
        shape = (parts, self.T, self.nh * D) if parts else (self.T, self.nh * D)
        self.x = torch.randn(shape, generator=g, device="cuda") * size
        if not parts:
            self.x = self.x.bfloat16()
        self.qn = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).bfloat16()
        self.kn = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).bfloat16()
        self.pos = ints([a + i for a, n in zip(kept, new) for i in range(n)]).view(-1)
        self.tab = table(max(self.lens) + 40)
        self.indptr = ints([sum(new[:i]) for i in range(len(new) + 1)])

    def call(self, x=None, **k):
        from msgl import ops
        f = ops.qknorm_rope_store_kv8_partials if self.parts else ops.qknorm_rope_store_kv8
        a = dict(q_indptr=self.indptr, max_q_len=max(1, max(self.new)))
        a.update(k)
        return f(self.x if x is None else x, self.kv8, self.scales, self.pos, self.table, ints(self.lens), self.tab, self.qn,
                 self.kn, self.hq, self.hkv, EPS, **a)

    def check(self, q, before, before_scales):
        full = (self.x.double().sum(0) if self.parts else self.x.double()).view(self.T, self.nh, D)
        w = torch.cat([self.qn.expand(self.hq, D), self.kn.expand(self.hkv, D)])
        ref, mag = turned(full[:, :self.hq + self.hkv], self.pos, self.tab, w)
        err = (q.double() - ref[:, :self.hq]).abs()
        assert bool((err <= ref[:, :self.hq].abs() * 2 ** -8 + mag[:, :self.hq] * 2 ** -17).all())
        rest = torch.ones(len(self.kv8), dtype=torch.bool, device="cuda")
        row = 0
        got, was = [pool_values(self.kv8, self.scales, k) for k in (0, 1)], [pool_values(before, before_scales, k) for k in (0, 1)]
        for r, (kept, n) in enumerate(zip(self.kept, self.new)):
            for p in range(kept // PAGE, -(-(kept + n) // PAGE) if n else 0):
                phys = int(self.table[r, p])
                rest[phys] = False
                old, first, end = max(0, kept - p * PAGE), max(kept, p * PAGE), min(kept + n, (p + 1) * PAGE)
                at = row + first - kept
                rows = slice(at, at + end - first)
                for kind, src, off in ((0, ref[:, self.hq:], mag[:, self.hq:] * 2 ** -17),
                                       (1, full[:, self.hq + self.hkv:], full[:, self.hq + self.hkv:].abs() * self.parts * 2 ** -22)):
                    want = torch.zeros(self.hkv, PAGE, D, dtype=torch.float64, device="cuda")
                    slack = torch.zeros_like(want)
                    want[:, :min(old, PAGE)] = was[kind][phys, :, :min(old, PAGE)]
                    want[:, first - p * PAGE:end - p * PAGE] = src[rows].transpose(0, 1)
                    slack[:, first - p * PAGE:end - p * PAGE] = off[rows].transpose(0, 1)
                    e = self.scales[phys, :, kind].double() - 127
                    amax = want.abs().amax((1, 2))
                    near = slack.amax((1, 2))
                    assert bool(((e >= exponent(amax - near)) & (e <= exponent(amax + near))).all())
                    s = torch.exp2(e)[:, None, None]
                    bound = torch.maximum(want.abs() * 2 ** -4, s * 2 ** -10) + slack * (1 + 2 ** -4)
                    assert bool(((got[kind][phys] - want).abs() <= bound).all())
                    if kind == 1 and not self.parts:  # a function of exact values: the very codes
                        assert torch.equal(got[kind][phys], quantise(want)[0])
                    if old:  # earlier tokens alone: exact
                        v = want[:, :old] / s
                        fine = v.abs() >= 2.0 ** -6
                        assert torch.equal(got[kind][phys][:, :old][fine], want[:, :old][fine])
                    assert bool((got[kind][phys][:, end - p * PAGE:] == 0).all())
            row += n
        assert torch.equal(self.kv8[rest], before[rest]) and torch.equal(self.scales[rest], before_scales[rest])


KEPT_NEW = [([0], [1]), ([15], [1]), ([16], [1]), ([5, 0, 31, 100], [1, 1, 1, 1]), ([0, 3], [16, 13]), ([7, 0, 40], [50, 0, 17]),
            ([100, 31, 0, 9], [5, 5, 5, 5]), ([0], [33]), ([1], [257])]


@pytest.mark.parametrize("kept,new", KEPT_NEW)
@pytest.mark.parametrize("hq,hkv", [(8, 1), (16, 8), (32, 4), (5, 3)])
@pytest.mark.parametrize("parts", [0, 1, 6])
def test_append(cuda, kept, new, hq, hkv, parts):
    from msgl import ops
    a = Append(kept, new, hq, hkv, parts, seed=sum(kept) + parts + hq)
    before, scales = a.kv8.clone(), a.scales.clone()
    q = a.call()
    a.check(q, before, scales)
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("size", [1e-30, 1e-10, 1e6, 1e30])
def test_append_sizes(cuda, size):
    """Values far from one: the values' exponent follows, down to 2^-96."""
    a = Append([9, 0], [7, 20], 8, 2, seed=3, size=size)
    before, scales = a.kv8.clone(), a.scales.clone()
    a.check(a.call(), before, scales)


def test_append_without_indptr_and_twice(cuda):
    """Single rows without q_indptr; the same call again leaves what the first one left."""
    a = Append([5, 16, 47], [1, 1, 1], 8, 2, seed=4)
    before, scales = a.kv8.clone(), a.scales.clone()
    q = a.call(q_indptr=None, max_q_len=1)
    a.check(q, before, scales)
    kv8, sc = a.kv8.clone(), a.scales.clone()
    assert torch.equal(a.call(), q) and torch.equal(a.kv8, kv8) and torch.equal(a.scales, sc)


def test_append_zeros_and_nan(cuda):
    """Rows of zeros; NaN and infinities stay where they are and do not move the scale, in the same call and
    when their page is written again."""
    a = Append([3], [6], 8, 2, seed=5)
    v = a.x.view(6, a.nh, D)
    v[:, 10] = 0  # values of head 0
    v[2, 11, 5], v[3, 11, 6], v[4, 11, 7] = NAN, math.inf, -math.inf
    v[1, 8, 9] = NAN  # a key: its whole row is NaN behind the norm
    before = [pool_values(a.kv8, a.scales, k)[int(a.table[0, 0])] for k in (0, 1)]
    for again in range(2):
        a.call()
        phys = int(a.table[0, 0])
        keys, values = (pool_values(a.kv8, a.scales, k)[phys] for k in (0, 1))
        assert bool(torch.isnan(keys[0, 4]).all()) and bool(torch.isfinite(keys[1]).all())
        assert not bool(torch.isnan(keys[0, [0, 1, 2, 3, 5, 6, 7, 8]]).any())
        want = torch.cat([before[1][1, :3], v[:, 11].double()])
        fine = torch.isfinite(want)
        assert int((~fine).sum()) == 3 and torch.equal(torch.isnan(values[1, :9]), ~fine)
        assert torch.equal(values[1, :9][fine], quantise(torch.where(fine, want, 0.0)[None])[0][0][fine])
        assert bool((values[0, 3:] == 0).all())
    a.kept, a.new, a.lens = [9], [1], [10]  # the page once more, behind the NaN
    held = pool_values(a.kv8, a.scales, 1)[phys][1, :9]
    a.x, a.T, a.pos, a.indptr = a.x[:1].clone(), 1, ints([9]), ints([0, 1])
    a.call()
    now = pool_values(a.kv8, a.scales, 1)[phys][1, :9]
    assert torch.equal(torch.isnan(now), torch.isnan(held))


def test_append_all_zero_page(cuda):
    a = Append([0], [4], 8, 1, seed=6)
    a.x.zero_()
    a.call()
    phys = int(a.table[0, 0])
    assert a.scales[phys].tolist() == [[127 - 96] * 2] and bool((decode(a.kv8[phys]) == 0).all())  # -0 among them


@pytest.mark.parametrize("size", [1.0, 300.0])
def test_append_behind_rejected_rows(cuda, size):
    """Tokens 20 .. 26 stored, then only 20 and 21 kept: storing others behind them gives the exponents of a pool
    that never saw the rejected ones, and its values but where those, being large, made earlier ones subnormal."""
    a, b = Append([20], [2], 8, 2, seed=7), Append([20], [2], 8, 2, seed=7)
    b.kv8.copy_(a.kv8), b.scales.copy_(a.scales)
    a.call(), b.call()
    big = Append([22], [5], 8, 2, seed=8, size=size)
    big.kv8, big.scales, big.table = a.kv8, a.scales, a.table
    big.call()
    phys = int(a.table[0, 1])
    large = torch.exp2(a.scales[phys].double() - 127)
    for p in (a, b):
        p.kept, p.new, p.lens = [22], [3], [25]
        p.x, p.T, p.pos, p.indptr = big.x[:3] / size, 3, ints([22, 23, 24]), ints([0, 3])
        p.call()
    for kind in (0, 1):
        x, y = (pool_values(p.kv8, p.scales, kind)[phys] for p in (a, b))
        step = large[:, kind, None, None] * 2.0 ** -9
        assert bool(((x - y).abs() <= torch.where(y.abs() < 8 * step, step / 2, 0.0)).all())
        assert torch.equal(x[:, 6:], y[:, 6:])
    assert torch.equal(a.scales[phys], b.scales[phys])


def test_append_does_not_read_behind_the_kept_tokens(cuda):
    """Any codes in the slots behind the kept tokens, NaN among them."""
    a, b = Append([20], [3], 8, 2, seed=10), Append([20], [3], 8, 2, seed=10)
    phys = int(a.table[0, 1])
    for at in places():
        b.kv8[phys][:, at[4:].reshape(-1)] = 0x7f
    a.call(), b.call()
    assert torch.equal(a.kv8[phys], b.kv8[phys]) and torch.equal(a.scales, b.scales)


def test_append_bounds(cuda):
    """Rows behind the last request stay; bad lengths, positions and pages are recorded and skipped."""
    from msgl import ops
    a = Append([0, 10], [3, 4], 8, 2, seed=9)
    out = torch.full((7, 8, D), 7.0, device="cuda").bfloat16()
    before, scales = a.kv8.clone(), a.scales.clone()
    a.call(q_indptr=ints([0, 3, 5]), max_q_len=3, out=out)  # two rows nobody owns
    assert bool((out[5:] == 7).all()) and not bool((out[:5] == 7).all(-1).any())
    assert ops.device_error() == (0, 0)
    a.kv8.copy_(before), a.scales.copy_(scales)
    a.call(max_q_len=3)  # request 1 has four
    assert ops.device_error() == (6, 911)
    assert torch.equal(a.kv8[a.table[1, 0].long()], before[a.table[1, 0].long()])
    a.pos[2] = 10 ** 6
    a.call()
    assert ops.device_error() == (6, 912)
    a.pos[2] = 2
    a.table[1, 0] = len(a.kv8)
    a.call()
    assert ops.device_error() == (6, 913)
    a.table[1, 0] = 0
    a.lens = [3, 3]  # shorter than its rows
    a.call()
    assert ops.device_error() == (6, 910)
    assert ops.device_error() == (0, 0)


# ------------------------------------------------------------------ attention
class Attend:
    def __init__(self, lens, rows, hq, hkv, seed=0, spread=True, std=1.0):
        self.g = g = torch.Generator("cuda").manual_seed(seed)
        self.lens, self.rows, self.hq, self.hkv = lens, rows, hq, hkv
        self.table, pages = page_table(lens, g)
        self.kv8 = torch.full((pages, hkv, 4096), 0x7f, dtype=torch.uint8, device="cuda")  # NaN where nothing is stored
        self.scales = torch.full((pages, hkv, 2), 127, dtype=torch.uint8, device="cuda")
        self.k, self.v = [], []
        for r, n in enumerate(lens):
            need = -(-n // PAGE)
            if not need:
                self.k.append(torch.zeros(hkv, 0, D, device="cuda")), self.v.append(torch.zeros(hkv, 0, D, device="cuda"))
                continue
            at = self.table[r, :need].long()
            for kind, keep in ((0, self.k), (1, self.v)):
                x = std * torch.randn(need, hkv, PAGE, D, generator=g, device="cuda", dtype=torch.float64)
                if spread:
                    x = x * 2.0 ** torch.randint(-3, 3, (need, hkv, 1, 1), generator=g, device="cuda")
                fill(self.kv8, self.scales, at, kind, x)
                keep.append(None)
            self.hide(r, n)
        self.T = sum(rows)
        self.q = torch.randn(max(self.T, 1), hq, D, generator=g, device="cuda").bfloat16()[:self.T]
        self.indptr = ints([sum(rows[:i]) for i in range(len(rows) + 1)])

    def hide(self, r, n):
        """NaN codes in the slots of request r from token n on."""
        need = -(-n // PAGE)
        for at in places():
            if n % PAGE:
                self.kv8[int(self.table[r, need - 1]), :, at[n % PAGE:].reshape(-1)] = 0x7f

    def call(self, **k):
        from msgl import ops
        a = dict(q_indptr=self.indptr, max_q_len=max(self.rows))
        a.update(k)
        return ops.paged_attention_kv8(self.q, self.kv8, self.scales, self.table, ints(self.lens), a.pop("max_seq", max(self.lens)),
                                       self.hq, self.hkv, **a)

    def check(self, out, scale=D ** -0.5):
        G = self.hq // self.hkv
        row = 0
        for r, (n, m) in enumerate(zip(self.lens, self.rows)):
            if m == 0:
                continue
            at = self.table[r, :-(-n // PAGE)].long()
            keys, values = (pool_values(self.kv8[at], self.scales[at], k).transpose(0, 1).reshape(self.hkv, -1, D)[:, :n] for k in (0, 1))
            vs = torch.exp2(self.scales[at][:, :, 1].double() - 127).repeat_interleave(PAGE, 0)[:n].T
            q = self.q[row:row + m].double().view(m, self.hkv, G, D)
            got = out[row:row + m].double().view(m, self.hkv, G, D)
            row += m
            if n == 0:
                assert bool((got == 0).all())
                continue
            pos = torch.arange(n - m, n, device="cuda")
            for h in range(self.hkv):
                s = torch.einsum("mgd,nd->mgn", q[:, h], keys[h]) * scale
                seen = torch.arange(n, device="cuda") <= pos[:, None]
                size = torch.einsum("mgd,nd->mgn", q[:, h].abs(), keys[h].nan_to_num(0).abs()).masked_fill(~seen[:, None], 0).amax(-1) * scale
                p = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1).nan_to_num(0.0)
                # keys behind the row do not reach it: as if they were not there
                val = torch.where(seen[:, None, :, None].any(0).any(0), values[h], 0.0)
                ref = torch.einsum("mgn,nd->mgd", p, val.nan_to_num(0.0))
                mass = torch.einsum("mgn,nd->mgd", p, val.nan_to_num(0.0).abs())
                tiny = n * 2.0 ** -25 * 448 * (p * vs[h]).amax(-1)
                tol = ref.abs() * 2 ** -8 + mass * (2 ** -11 + 2 ** -20 + 2 * size[..., None] * 2 ** -17) + tiny[..., None]
                bad = torch.isnan(val).any(1)
                if bool(bad.any()):  # a NaN value that a row sees makes that dimension of its result NaN
                    nan = torch.einsum("mn,nd->md", (seen & bad).double(), torch.isnan(val).double()) > 0
                    nan = nan[:, None].expand_as(ref)
                else:
                    nan = torch.zeros_like(ref, dtype=torch.bool)
                gone = (torch.isnan(keys[h]).any(1) & seen).any(1)  # a NaN key makes the row NaN
                nan = nan | gone[:, None, None]
                assert torch.equal(torch.isnan(got[:, h]), nan), (r, h)
                err = (got[:, h] - ref).abs()
                assert bool((err <= tol)[~nan].all()), (r, h, float((err / tol)[~nan].max()))
        return row


LENS = [1, 2, 15, 16, 17, 31, 33, 64, 100, 129, 255, 400]


@pytest.mark.parametrize("hq,hkv", [(8, 1), (8, 8), (16, 8), (32, 4), (32, 8), (6, 3)])
@pytest.mark.parametrize("lens", [[1], [4099], LENS, [0, 5, 0, 70], [9000, 3, 700]])
def test_single_tokens(cuda, hq, hkv, lens):
    from msgl import ops
    a = Attend(lens, [1] * len(lens), hq, hkv, seed=len(lens) + hq)
    out = a.call(q_indptr=None, max_q_len=1, max_seq=max(lens))
    a.check(out)
    assert torch.equal(out, a.call())  # given as ranges of one row
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("rows", [2, 3, 5, 7, 8, 13, 16])
@pytest.mark.parametrize("hq,hkv", [(8, 1), (8, 8), (16, 8), (32, 8)])
def test_drafted_rows(cuda, rows, hq, hkv):
    from msgl import ops
    lens = [rows, rows + 1, 40, 161, 1000, 2047]
    a = Attend([max(n, rows) for n in lens], [rows] * len(lens), hq, hkv, seed=rows)
    a.check(a.call())
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("lens,rows", [([300, 40, 17, 130], [100, 40, 1, 0]), ([17], [17]), ([1500, 1100], [1100, 333]), ([129, 128, 127], [129, 128, 127]),
                                       ([2500], [64]), ([700, 900, 65], [65, 33, 65])])
@pytest.mark.parametrize("hq,hkv", [(8, 1), (4, 4), (16, 8), (32, 8)])
def test_chunks(cuda, lens, rows, hq, hkv):
    from msgl import ops
    a = Attend(lens, rows, hq, hkv, seed=sum(rows))
    a.check(a.call())
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("lens,rows,hq,hkv", [([1500, 1100], [1100, 333], 32, 8), ([2048], [2048], 32, 8), ([2000] * 24, [6] * 24, 8, 1),
                                              ([1000] * 9, [30] * 9, 16, 4), ([900] * 30, [1] * 30, 32, 8)])
def test_the_same_call_again_gives_the_same_bits(cuda, lens, rows, hq, hkv):
    """No part of a result hangs on which warp or copy came first."""
    a = Attend(lens, rows, hq, hkv, seed=5)
    first = a.call()
    for _ in range(40):
        assert torch.equal(a.call(), first)


@pytest.mark.parametrize("rows", [[1, 1, 1], [6, 6, 6], [70, 33, 90]])
def test_values_behind_a_row_do_not_reach_it(cuda, rows):
    """NaN keys and values in tokens that only later rows see, and in all slots behind the context (Attend)."""
    lens = [100, 47, 250]
    a = Attend(lens, rows, 8, 2, seed=11)
    keys, values = places()
    for r, (n, m) in enumerate(zip(lens, rows)):
        for back, kind in ((1, 0), (2, 1)) if m > 2 else ():
            t = n - back  # its own row and later ones see it
            where = (keys if kind == 0 else values)[t % PAGE, 7 * kind:7 * kind + 1]
            a.kv8[int(a.table[r, t // PAGE]), 1, where] = 0x7f
    a.check(a.call())


def test_nan_in_the_open(cuda):
    """NaN values and keys that rows see: the dimension, and the whole row."""
    a = Attend([300], [4], 8, 2, seed=12)
    keys, values = places()
    a.kv8[int(a.table[0, 3]), 0, values[5, 77]] = 0xff
    a.kv8[int(a.table[0, 4]), 1, keys[6, 1]] = 0x7f
    a.check(a.call())
    a = Attend([300, 20], [1, 1], 8, 2, seed=13)
    a.q[0, 1, 3], a.q[1, 7, 2] = math.inf, NAN
    out = a.call()
    nan = torch.isnan(out).all(-1)
    assert nan.sum() == 2 and bool(nan[0, 1]) and bool(nan[1, 7]) and int(torch.isnan(out).sum()) == 2 * D


@pytest.mark.parametrize("rows", [1, 4, 100])
def test_far_scales(cuda, rows):
    """Pages whose values differ by 2^40 and queries far from one: weights are taken with the values' scale."""
    a = Attend([500], [rows], 8, 2, seed=14, spread=False)
    g = a.g
    at = a.table[0, :32].long()
    x = torch.randn(32, 2, PAGE, D, generator=g, device="cuda", dtype=torch.float64) * 2.0 ** torch.randint(-20, 20, (32, 2, 1, 1), generator=g, device="cuda")
    fill(a.kv8, a.scales, at, 1, x)
    a.hide(0, 500)
    a.check(a.call())
    a.q = (a.q.float() * 2.0 ** 30).bfloat16()
    out = a.call(scale=D ** -0.5 * 2.0 ** -30)
    a.check(out, scale=D ** -0.5 * 2.0 ** -30)


def test_large_logits(cuda):
    """Logits of hundreds: the softmax picks one key."""
    a = Attend([3000, 700], [1, 1], 16, 4, seed=15, std=3.0)
    a.q = (a.q.float() * 8).bfloat16()
    a.check(a.call())


@pytest.mark.parametrize("rows", [1, 6, 80])
def test_rows_before_the_context(cuda, rows):
    """More rows than tokens: rows at negative positions are zeros; rows behind the last request stay."""
    from msgl import ops
    a = Attend([40, 3], [rows, rows], 8, 2, seed=16)
    out = torch.full_like(a.q, 7.0)
    a.call(out=out)
    got = out.clone()
    lost = max(0, rows - 3)
    assert bool((got[rows:rows + lost] == 0).all())
    a.lens[1], a.rows = 3, [rows, rows - lost]
    keep = torch.cat([got[:rows], got[rows + lost:]])
    a.q = torch.cat([a.q[:rows], a.q[rows + lost:]])
    lost0 = max(0, rows - 40)
    if lost0:
        assert bool((keep[:lost0] == 0).all())
        keep, a.q, a.rows = keep[lost0:], a.q[lost0:], [rows - lost0, a.rows[1]]
    a.check(keep)
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("rows", [1, 5, 70])
def test_bounds(cuda, rows):
    from msgl import ops
    a = Attend([200, 100, 150], [rows] * 3, 8, 2, seed=17)
    good = a.call()
    out = torch.full_like(a.q, 7.0)
    a.call(out=out, q_indptr=ints([0, rows, 2 * rows, 2 * rows]))
    assert bool((out[2 * rows:] == 7).all()) and torch.equal(out[:2 * rows], good[:2 * rows])
    assert ops.device_error() == (0, 0)
    if rows > 1:
        out.fill_(7.0)
        a.call(out=out, q_indptr=ints([0, rows, 3 * rows, 3 * rows]))  # too many rows: skipped
        assert ops.device_error() == (6, 901) and bool((out[rows:] == 7).all()) and torch.equal(out[:rows], good[:rows])
    a.table[1, 2] = len(a.kv8)
    a.call()
    assert ops.device_error() == (6, 902)
    a.table[1, 2] = -1
    a.call()
    assert ops.device_error() == (6, 902)
    a.lens[0] = -3
    a.table[1, 2] = 0
    a.call(max_seq=160)
    assert ops.device_error() == (6, 900)
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("rows", [1, 6, 90])
def test_same_bits_again_and_in_a_graph(cuda, rows):
    """The result does not hang on an order of arrival, and a captured call replays on new lengths."""
    lens = [1000, 90, 3000, 500]
    a = Attend(lens, [rows] * 4, 16, 4, seed=18)
    from msgl import ops
    seq = ints(lens)
    ws = ops.attention_kv8_workspace(4, rows, 16, 4)
    out = torch.empty_like(a.q)
    args = (a.q, a.kv8, a.scales, a.table, seq, 3000, 16, 4)
    kw = dict(q_indptr=a.indptr, max_q_len=rows, workspace=ws, out=out)
    first = ops.paged_attention_kv8(*args, **kw).clone()
    for _ in range(5):
        assert torch.equal(ops.paged_attention_kv8(*args, **kw), first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.paged_attention_kv8(*args, **kw)
        out.zero_()
        g.replay()
        s.synchronize()
        assert torch.equal(out, first)
        seq.copy_(ints([999, 90, 1234, 97]))
        g.replay()
        s.synchronize()
    got = out.clone()
    assert torch.equal(ops.paged_attention_kv8(*args, **kw), got)
    a.lens = [999, 90, 1234, 97]
    a.check(got)


def test_many_short_requests(cuda):
    """More items than CTAs, several requests a CTA; more requests than threads of a CTA."""
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(1, 60, (700,), generator=g).tolist()
    a = Attend(lens, [1] * 700, 4, 2, seed=19)
    a.check(a.call())


def test_workspace_serves_smaller_calls(cuda):
    from msgl import ops
    ws = ops.attention_kv8_workspace(5, 100, 8, 2)
    for lens, rows in (([700, 20], [100, 3]), ([900] * 5, [1] * 5), ([50, 1200, 8], [8, 8, 8]), ([2000], [17])):
        a = Attend(lens, rows, 8, 2, seed=len(lens))
        a.check(a.call(workspace=ws))


def test_many_short_requests_of_several_rows(cuda):
    """Many items a CTA, short ones, in every tile form; a NaN that only later rows see in each of them."""
    keys, values = places()
    for rows, hq, hkv in ((9, 4, 2), (20, 16, 8), (70, 4, 2), (40, 16, 2)):
        g = torch.Generator().manual_seed(rows)
        lens = torch.randint(rows, rows + 50, (90,), generator=g).tolist()
        a = Attend(lens, [rows] * 90, hq, hkv, seed=rows)
        for r, n in enumerate(lens):
            if r % 3 == 0:
                a.kv8[int(a.table[r, (n - 2) // PAGE]), r % hkv, values[(n - 2) % PAGE, r % D]] = 0x7f
        a.check(a.call())


def test_pool_beyond_2_gib(cuda):
    """Pages whose offsets pass 32 bits: the same bits as from a small pool."""
    from msgl import ops
    pages, hq, hkv = 70000, 16, 8  # 2.3 GB
    far = torch.zeros(pages, hkv, 4096, dtype=torch.uint8, device="cuda")
    far_scales = torch.zeros(pages, hkv, 2, dtype=torch.uint8, device="cuda")
    for rows in (1, 8, 20, 60, 200):
        a = Attend([400, 310], [rows] * 2, hq, hkv, seed=rows)
        near = a.call()
        n = len(a.kv8)
        far[pages - n:], far_scales[pages - n:] = a.kv8, a.scales
        a.kv8, a.scales, a.table = far, far_scales, a.table + (pages - n)
        assert torch.equal(a.call(), near)
    b = Append([100, 0], [30, 50], hq, hkv)
    n, before = len(b.kv8), (b.kv8.clone(), b.scales.clone())
    far[pages - n:], far_scales[pages - n:] = before
    b.call()
    want = b.kv8, b.scales
    b.kv8, b.scales, b.table = far, far_scales, b.table + (pages - n)
    b.call()
    assert torch.equal(far[pages - n:], want[0]) and torch.equal(far_scales[pages - n:], want[1])
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("rows", [1, 6, 40, 150])
def test_two_streams_and_padding_rows(cuda, rows):
    """Two calls at once, each with its workspace, on a stream of its own; rows behind the last request keep what they held."""
    from msgl import ops
    calls = [Attend([3000, 500, 1200], [rows] * 3, 16, 4, seed=21), Attend([900, 2500], [rows] * 2, 16, 4, seed=22)]
    want = [a.call() for a in calls]
    runs = []
    torch.cuda.synchronize()
    for a in calls:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            q = torch.cat([a.q, torch.full((5, 16, D), float("nan"), device="cuda").bfloat16()])
            runs.append((s, a, q, ints(a.lens), torch.full_like(q, 7.0), ops.attention_kv8_workspace(3, rows, 16, 4)))
    torch.cuda.synchronize()
    for _ in range(10):
        for s, a, q, seq, out, ws in runs:
            with torch.cuda.stream(s):
                ops.paged_attention_kv8(q, a.kv8, a.scales, a.table, seq, max(a.lens), 16, 4, q_indptr=a.indptr, max_q_len=rows, workspace=ws, out=out)
    torch.cuda.synchronize()
    for (s, a, q, seq, out, ws), w in zip(runs, want):
        assert torch.equal(out[:a.T], w) and bool((out[a.T:] == 7).all())
