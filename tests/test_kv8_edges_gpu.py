"""Attention over the 8-bit pool where factors underflow or weights are far apart, against softmax in 64 bits
(Attend.check of test_kv8_gpu.py and its tolerances: half a bf16 step, 2^-11 of each weight, fp32 logits)."""
import math

import pytest
import torch

from kv8_plain import D, PAGE, fill, ints, pool_values
from test_kv8_gpu import Attend

pytestmark = pytest.mark.gpu
NAN = float("nan")
# rows of a request with 4 heads a group: warp MMAs of 8 and 16 rows, tcgen05 of 64, 128 and 256
ROWS = [1, 2, 4, 6, 16, 30, 40, 150]


@pytest.mark.parametrize("rows", ROWS)
def test_zero_queries_over_zero_keys(cuda, rows):
    """Every logit is 0: the mean of the values that a row sees, the last pages' masked keys among them."""
    a = Attend([rows + 75, rows, rows + 16], [rows] * 3, 8, 2, seed=rows)
    pages = torch.arange(len(a.kv8), device="cuda")
    fill(a.kv8, a.scales, pages, 0, torch.zeros(len(pages), 2, PAGE, D, device="cuda"))
    for r, n in enumerate(a.lens):
        a.hide(r, n)
    a.q.zero_()
    a.check(a.call())


@pytest.mark.parametrize("rows", ROWS)
def test_some_zero_queries(cuda, rows):
    """Zero rows among others, keys of any size."""
    a = Attend([rows + 75, rows], [rows] * 2, 8, 2, seed=rows + 1)
    pages = torch.arange(len(a.kv8), device="cuda")
    keys = torch.randn(len(pages), 2, PAGE, D, generator=a.g, device="cuda", dtype=torch.float64)
    fill(a.kv8, a.scales, pages, 0, keys * 2.0 ** torch.randint(-70, 2, (len(pages), 2, 1, 1), generator=a.g, device="cuda"))
    for r, n in enumerate(a.lens):
        a.hide(r, n)
    a.q[::2, 1] = 0
    a.q[0] = 0
    a.check(a.call())


@pytest.mark.parametrize("rows", ROWS)
def test_scale_zero(cuda, rows):
    a = Attend([rows + 75, rows], [rows] * 2, 8, 2, seed=rows + 2)
    a.check(a.call(scale=0.0), scale=0.0)


@pytest.mark.parametrize("rows", ROWS)
def test_scale_nan(cuda, rows):
    a = Attend([rows + 75], [rows], 8, 2, seed=rows + 2)
    assert bool(torch.isnan(a.call(scale=NAN)).all())


@pytest.mark.parametrize("rows", ROWS)
def test_a_pool_that_was_only_cleared(cuda, rows):
    """Zero codes and zero scale bytes (kv8_pool): zeros, whatever the query."""
    from msgl import ops
    a = Attend([rows + 75, rows], [rows] * 2, 8, 2, seed=rows + 3)
    a.kv8, a.scales = ops.kv8_pool(len(a.kv8), 2)
    for zero in (False, True):
        if zero:
            a.q.zero_()
        out = a.call(out=torch.full_like(a.q, 7.0))
        assert bool((out == 0).all())


@pytest.mark.parametrize("rows", [2, 6, 30, 80])
@pytest.mark.parametrize("what", [NAN, math.inf])
def test_bad_queries_before_the_context(cuda, rows, what):
    """A row before its context's first token gives zeros whatever its query holds, and a NaN or infinite query of
    another row gives NaN, on every call."""
    kept = 4 if rows > 6 else 1
    a = Attend([rows - kept, 90], [rows, rows], 8, 2, seed=rows + 5)
    a.q[0, 1, 3], a.q[kept, 2, 5], a.q[2 * rows - 1, 7, 9] = what, what, what
    for _ in range(20):
        out = a.call(out=torch.full_like(a.q, 7.0))
        assert bool((out[:kept] == 0).all())
        bad = torch.isnan(out).all(-1)
        assert bool(bad[kept, 2]) and bool(bad[2 * rows - 1, 7]) and int(bad.sum()) == 2 and int(torch.isnan(out).sum()) == 2 * D


@pytest.mark.parametrize("rows", ROWS)
def test_pages_that_were_only_cleared(cuda, rows):
    """Such pages among others: their keys count with logit 0, their values are 0."""
    a = Attend([rows + 700, rows + 40], [rows] * 2, 8, 2, seed=rows + 4)
    for r, column in ((0, 0), (0, 17), (0, 39), (1, 1)):
        page = int(a.table[r, column])
        a.kv8[page], a.scales[page] = 0, 0
    a.check(a.call())


def shared_pages(reqs, n, rows, seed):
    """Requests over the same pages, so that each is one CTA's: every key zero, every value in [1, 1.5]."""
    a = Attend([n], [rows], 8, 2, seed=seed)
    need = -(-n // PAGE)
    at = a.table[0, :need].long()
    keys = torch.zeros(need, 2, PAGE, D, dtype=torch.float64, device="cuda")
    values = 1 + torch.randint(0, 5, keys.shape, generator=a.g, device="cuda").double() / 8
    a.at, a.keys, a.values = at, keys, values
    a.table, a.lens, a.rows, a.T = a.table.expand(reqs, -1).contiguous(), [n] * reqs, [rows] * reqs, reqs * rows
    a.q = torch.zeros(a.T, 8, D, device="cuda").bfloat16()
    a.q[..., 0] = 8
    a.indptr = ints([rows * i for i in range(reqs + 1)])
    return a


# reqs x rows: two CTAs an SM (296), one (148)
SINKS = [(600, 1), (300, 4), (300, 6), (300, 20), (150, 50)]


@pytest.mark.parametrize("reqs,rows", SINKS)
@pytest.mark.parametrize("bits", [12.4, 16.4, 20.4, 24.4])
@pytest.mark.parametrize("at", [0, 1500])
def test_a_key_that_takes_the_weight(cuda, reqs, rows, bits, at):
    """One key's logit is `bits` octaves above the others' and its value is 0 (an attention sink): the result is the
    others' values with their small weights."""
    n = 1900
    a = shared_pages(reqs, n, rows, seed=rows)
    a.keys[at // PAGE, :, at % PAGE, 0] = 20
    a.values[at // PAGE, :, at % PAGE] = 0
    fill(a.kv8, a.scales, a.at, 0, a.keys), fill(a.kv8, a.scales, a.at, 1, a.values)
    a.hide(0, n)
    scale = bits * math.log(2) / 160
    out = a.call(scale=scale)
    check_mean(a, out, n, scale)


@pytest.mark.parametrize("reqs,rows", SINKS)
@pytest.mark.parametrize("bits", [12, 18, 24])
def test_a_value_that_sets_its_pages_scale(cuda, reqs, rows, bits):
    """A value of 2^bits with hardly any weight: the page's other tokens and other pages count as before."""
    n = 1900
    a = shared_pages(reqs, n, rows, seed=rows)
    a.keys[3, :, 1, 0] = -240
    a.keys[3, :, 2, 0] = 0.75  # keeps the page's weights off the powers of two
    a.values[3] = 0
    a.values[3, :, 1] = 2.0 ** bits
    fill(a.kv8, a.scales, a.at, 0, a.keys), fill(a.kv8, a.scales, a.at, 1, a.values)
    a.hide(0, n)
    scale = 0.07
    check_mean(a, a.call(scale=scale), n, scale)


def check_mean(a, out, n, scale):
    """The definition for queries that are all the same, [1st row .. last] of each request. Weights: 2^-11 of each, and
    2^-36 of the largest; a logit of x: fp32, 2^-17 |x|, twice (as much of a normalised weight)."""
    m = a.rows[0]
    for row in {0, m - 1}:
        seen = n - m + row + 1
        for h in range(2):
            x = a.keys[:, h].reshape(-1, D)[:seen, 0] * 8 * scale
            p = torch.softmax(x, 0)
            v = a.values[:, h].reshape(-1, D)[:seen]
            ref = p @ v
            page = torch.exp2(a.scales[a.at, h, 1].double() - 127).repeat_interleave(PAGE)[:seen]
            tiny = seen * 2.0 ** -36 * 448 * float((p * page).max())
            tol = ref * 2 ** -8 + ref * (2 ** -11 + 2 ** -20 + 2 * float(x.abs().max()) * 2 ** -17) + tiny
            got = out.view(len(a.lens), m, 2, 4, D)[:, row, h].double()
            err = (got - ref).abs()
            assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("rows,hq,hkv", [(6, 64, 8), (12, 32, 8), (20, 8, 8)])
def test_items_of_one_step_among_longer_ones(cuda, rows, hq, hkv):
    """Blocks of up to 64 rows, whose second stream has no step in items of up to 64 keys: eight items a CTA, in every order of
    one, two and three steps, the same bits each time."""
    from msgl import ops
    lens = [max(rows, [30, 64, 65, 40, 128, 50, 20, 150, 60][r * r % 9] + r % 5) for r in range(150)]
    a = Attend(lens, [rows] * 150, hq, hkv, seed=rows)
    out = a.call()
    a.check(out)
    for _ in range(60):
        assert torch.equal(a.call(), out)
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("big", [2.0 ** 12, 2.0 ** 20, -3e38])
def test_a_large_query_element_that_meets_zeros(cuda, rows, big):
    """Dimension 77 of every key is 0: the row's other elements, which are that much smaller, make its logits."""
    a = Attend([rows + 300, rows], [rows] * 2, 8, 2, seed=rows + 6)
    pages = torch.arange(len(a.kv8), device="cuda")
    keys = torch.randn(len(pages), 2, PAGE, D, generator=a.g, device="cuda", dtype=torch.float64) * 2
    keys[..., 77] = 0
    fill(a.kv8, a.scales, pages, 0, keys)
    for r, n in enumerate(a.lens):
        a.hide(r, n)
    if abs(big) > 1e30:
        a.q = (a.q.float() * 2.0 ** 100).bfloat16()
    a.q[..., 77] = big
    scale = 0.1 if abs(big) < 1e30 else 0.1 * 2.0 ** -100
    out = a.call(scale=scale)
    a.check(out, scale=scale)
    a.q = -a.q
    assert torch.equal(a.call(scale=-scale), out)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 16, 2.0 ** 19, 2.0 ** 20, 2.0 ** 21])
def test_huge_logits(cuda, rows, size):
    """Logits of `size` and more: the value of the one key that is ahead of the others by more than fp32's rounding."""
    a = Attend([rows + 500, rows + 30], [rows] * 2, 8, 2, seed=rows + 7)
    a.q = (a.q.float() * size).bfloat16()
    out = a.call()
    row = sure = 0
    for r, n in enumerate(a.lens):
        page = a.table[r, :-(-n // PAGE)].long()
        keys, values = (pool_values(a.kv8[page], a.scales[page], k).transpose(0, 1).reshape(2, -1, D)[:, :n] for k in (0, 1))
        pos = torch.arange(n - rows, n, device="cuda")
        q = a.q[row:row + rows].double().view(rows, 2, 4, D)
        for h in range(2):
            s = torch.einsum("mgd,nd->mgn", q[:, h], keys[h]) * D ** -0.5
            s = s.masked_fill((torch.arange(n, device="cuda") > pos[:, None])[:, None], -math.inf)
            off = torch.einsum("mgd,nd->mgn", q[:, h].abs(), keys[h].abs()).amax(-1) * D ** -0.5 * 2 ** -17
            top = torch.topk(s, 2, -1)
            alone = top.values[..., 0] - top.values[..., 1] > 2 * off + 60
            want = values[h][top.indices[..., 0]]
            got = out[row:row + rows].double().view(rows, 2, 4, D)[:, h]
            assert bool(((got - want).abs() <= want.abs() * 2 ** -8 + 2.0 ** -40)[alone].all())
            assert bool(torch.isfinite(got).all())
            sure += int(alone.sum())
        row += rows
    assert sure > 8 * row // 2
