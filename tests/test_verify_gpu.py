"""Token probabilities and draft verification on a B200, against 64-bit restatements.

Probabilities: p = exp((x - m) / T) / sum. fp32 knows x - m to 2^-24 of itself, 1 / T and the product with log2(e)
to 2^-23: the exponent is off by 2^-22 of itself at most; exp2, the sums and the division add 2^-20. Verification
decides by comparisons in 64 bits: equal tokens, but where the uniform number lies within 1e-12 of a border (the order
of 64-bit sums), which the restatement reports.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
NAN = float("nan")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check_probs(got, x, t):
    x, t = x.double(), t.double()[:, None]
    top = x.amax(1, keepdim=True)
    ref = torch.softmax(x / t, 1)
    tol = ref * (2 ** -20 + (x - top).abs().nan_to_num(0.0, posinf=0.0) / t * 2 ** -21) + 2.0 ** -125
    assert bool(((got.double() - ref).abs() <= tol).all()), float(((got.double() - ref).abs() / tol).max())


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 5), (7, 1000), (5, 1003), (1, 20480), (1, 20481), (2, 50257), (40, 32000), (1, 151936), (200, 4096),
                                        (3, 163844), (2, 327680), (2, 327677)])
def test_probs(cuda, rows, vocab):
    from msgl import ops
    g = torch.Generator("cuda").manual_seed(rows + vocab)
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 5
    t = torch.rand(rows, generator=g, device="cuda") + 0.3
    check_probs(ops.token_probs(x, t), x, t)
    check_probs(ops.token_probs(x), x, torch.ones(rows, device="cuda"))


@pytest.mark.parametrize("vocab", [1000, 1003, 50257])
def test_probs_strided_and_in_place(cuda, vocab):
    from msgl import ops
    g = torch.Generator("cuda").manual_seed(vocab)
    wide = torch.randn(6, vocab + 29, generator=g, device="cuda") * 3
    t = torch.rand(6, generator=g, device="cuda") + 0.5
    x = wide[:, 3:3 + vocab]
    want = ops.token_probs(x.contiguous(), t)
    out = torch.full((6, vocab + 5), 7.0, device="cuda")
    ops.token_probs(x, t, out=out[:, :vocab])
    assert torch.equal(out[:, :vocab], want) or bool((out[:, :vocab] - want).abs().max() < 1e-6)
    check_probs(out[:, :vocab], x, t)
    assert bool((out[:, vocab:] == 7).all())
    kept = wide.clone()
    ops.token_probs(x, t, out=x)
    check_probs(wide[:, 3:3 + vocab], kept[:, 3:3 + vocab], t)
    assert torch.equal(wide[:, :3], kept[:, :3]) and torch.equal(wide[:, 3 + vocab:], kept[:, 3 + vocab:])


@pytest.mark.parametrize("vocab", [7, 1000, 50257, 151936])
def test_probs_greedy(cuda, vocab):
    """Temperature 0 and below: one at the first maximum, as msgl_sample's greedy rows take it."""
    from msgl import ops
    g = torch.Generator("cuda").manual_seed(vocab)
    x = torch.randint(-3, 4, (5, vocab), generator=g, device="cuda").float()  # many ties
    x[3] = -math.inf
    x[4, vocab // 2:] = math.inf
    t = torch.tensor([0.0, -1.0, 0.0, 0.0, 0.0], device="cuda")
    p = ops.token_probs(x, t)
    pick = ops.sample(x, t, ints([0] * 5), torch.ones(5, device="cuda"))
    want = torch.zeros_like(p)
    want[torch.arange(5), pick.long()] = 1
    assert torch.equal(p, want) and int(pick[3]) == 0 and int(pick[4]) == vocab // 2


@pytest.mark.parametrize("vocab", [10, 1001, 151936])
def test_probs_masked(cuda, vocab):
    """Masked logits (-inf, the lowest value), rows without any, NaN and +inf."""
    from msgl import ops
    g = torch.Generator("cuda").manual_seed(vocab)
    x = torch.randn(8, vocab, generator=g, device="cuda")
    low = torch.finfo(torch.float32).min
    x[0, 1:] = -math.inf
    x[1, ::2] = -math.inf
    x[2] = -math.inf
    x[3, 2:] = low
    x[4] = low
    x[5, vocab // 2] = NAN
    x[6, 0] = math.inf
    x[7, :] = 3e38
    t = torch.full((8,), 0.7, device="cuda")
    p = ops.token_probs(x, t)
    assert torch.equal(p[0], (torch.arange(vocab, device="cuda") == 0).float())
    assert bool((p[1, ::2] == 0).all()) and bool((p[2] == 0).all()) and bool((p[3, 2:] == 0).all())
    assert bool(torch.isnan(p[5:7]).all())
    for r in (4, 7):
        assert bool(((p[r] * vocab - 1).abs() < 2 ** -20).all())
    fine = [0, 1, 3]
    check_probs(p[fine], x[fine], t[fine])


# ------------------------------------------------------------------ verification
def restate(p, q, tokens, indptr, u, last, most):
    """accepted, token rows, and whether each request's last token is off every border."""
    acc, rows, sure = [], [], []
    p, u, last = p.double().cpu(), u.double().cpu(), last.double().cpu()
    q = None if q is None else q.double().cpu()
    ptr, x = indptr.tolist(), tokens.tolist()
    for r in range(len(ptr) - 1):
        d, k = ptr[r], ptr[r + 1] - ptr[r]
        n = 0
        while n < k:
            v = x[d + n]
            if not (0 <= v < p.shape[1]) or not float(u[d + n]) * (1.0 if q is None else float(q[d + n, v])) < float(p[d + r + n, v]):
                break
            n += 1
        w = p[d + r + n].clone()
        if n < k:
            rest = w.clone()
            if q is None:
                if 0 <= x[d + n] < p.shape[1]:
                    rest[x[d + n]] -= 1
            else:
                rest -= q[d + n]
            rest = torch.where(rest > 0, rest, 0.0)
            w = rest if float(rest.sum()) > 0 else w
        c = torch.where(w > 0, w, 0.0).cumsum(0)
        goal = float(last[r]) * float(c[-1])
        at = int(torch.searchsorted(c, goal, right=True)) if float(c[-1]) > 0 else -1
        gap = float((c - goal).abs().min())
        sure.append(goal == 0.0 or gap > 1e-12)
        acc.append(n)
        rows.append(x[d:d + n] + [at] + [-1] * (most - n))
    return acc, rows, sure


def problem(ks, vocab, seed, closeness=0.7, point=False):
    g = torch.Generator("cuda").manual_seed(seed)
    B, n = len(ks), sum(ks)
    logits = torch.randn(n + B, vocab, generator=g, device="cuda") * 3
    p = torch.softmax(logits, 1)
    of = torch.tensor([sum(ks[:r]) + r + i for r in range(B) for i in range(ks[r])], dtype=torch.int64, device="cuda")
    q = torch.softmax(logits[of] + closeness * torch.randn(n, vocab, generator=g, device="cuda"), 1)
    tokens = (torch.multinomial(q, 1, generator=g)[:, 0] if n else of).int()
    indptr = ints([sum(ks[:r]) for r in range(B + 1)])
    return p, None if point else q, tokens, indptr, torch.rand(n, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")


def check(a, most):
    from msgl import ops
    accepted, tokens = ops.verify_drafts(*a, most)
    acc, rows, sure = restate(*a, most)
    assert accepted.tolist() == acc
    got = tokens.tolist()
    for r, ok in enumerate(sure):
        if ok:
            assert got[r] == rows[r], (r, got[r], rows[r])
        else:
            assert got[r][:acc[r]] == rows[r][:acc[r]]
    assert sum(sure) >= len(sure) - 1
    return acc


@pytest.mark.parametrize("ks", [[0], [4], [1, 0, 3, 7, 2], [5] * 40, [0, 0, 0], [33, 2], [1] * 200])
@pytest.mark.parametrize("vocab", [2, 100, 1003, 32000])
@pytest.mark.parametrize("point", [False, True])
def test_verify(cuda, ks, vocab, point):
    from msgl import ops
    acc = check(problem(ks, vocab, len(ks) + vocab, point=point), max(ks) + 2)
    if len(ks) >= 40 and vocab > 2 and not point:
        assert 0 < sum(acc) < sum(ks)  # both outcomes
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("vocab", [50257, 151936])
@pytest.mark.parametrize("closeness", [0.0, 0.3, 3.0])
def test_verify_large(cuda, vocab, closeness):
    check(problem([4, 0, 2, 4, 1, 3], vocab, vocab, closeness), 4)


def test_verify_borders(cuda):
    """Uniform numbers at 0 and next to 1, equal rows (the rest is empty: the target's own), one-hot rows, zero
    probabilities of the drafted token."""
    from msgl import ops
    V = 640
    p = torch.zeros(9, V, device="cuda")
    q = torch.zeros(5, V, device="cuda")
    p[0, 7] = 1.0                       # request 0: draft 7 certain -> accepted, even with u next to 1
    q[0, 7] = 1.0
    p[1, 600] = 1.0                     # its last row
    p[2, [3, 500]] = torch.tensor([0.25, 0.75], device="cuda")   # request 1: draft 9 impossible -> rejected at u = 0
    q[1, [9, 3]] = torch.tensor([0.5, 0.5], device="cuda")
    p[4] = 1.0 / V                      # request 2: p = q, u = 0 accepts; then the last row
    q[2] = 1.0 / V
    p[5, V - 1] = 1.0
    p[6, 100] = 0.5                     # request 3: p <= q everywhere, rejected -> the target's row
    q[3, 100] = 1.0
    p[8, 0] = 1.0                       # request 4: no draft of its own rows
    ptr = ints([0, 1, 2, 3, 4, 4])
    tok = ints([7, 9, 33, 100])
    eps = 1 - 2.0 ** -24
    u = torch.tensor([eps, 0.0, 0.0, eps], device="cuda")
    last = torch.tensor([eps, 0.0, eps, 0.5, 0.0], device="cuda")
    acc, rows = ops.verify_drafts(p, q[:4], tok, ptr, u, last, 2)
    assert acc.tolist() == [1, 0, 1, 0, 0]
    assert rows.tolist() == [[7, 600, -1], [500, -1, -1], [33, V - 1, -1], [100, -1, -1], [0, -1, -1]]
    assert ops.device_error() == (0, 0)


def test_verify_bad_inputs(cuda):
    from msgl import ops
    p, q, tok, ptr, u, last = problem([2, 2, 2], 1000, 5)
    tok[2] = 1000  # request 1's first draft
    acc, rows = ops.verify_drafts(p, q, tok, ptr, u, last, 2)
    a, b, _ = restate(p, q, tok, ptr, u, last, 2)
    assert acc.tolist() == a and rows.tolist() == b and acc[1] == 0 and ops.device_error() == (6, 921)
    tok[2] = -1
    acc, rows = ops.verify_drafts(p, None, tok, ptr, u, last, 2)
    a, b, _ = restate(p, None, tok, ptr, u, last, 2)
    assert acc.tolist() == a and rows.tolist() == b and ops.device_error() == (6, 921)
    tok[2] = 1
    for bad in ([0, 3, 4, 6], [0, 2, 1, 3], [0, 2, 4, 7]):
        acc, rows = ops.verify_drafts(p, q, tok, ints(bad), u, last, 2)
        assert ops.device_error() == (6, 920)
        wrong = [r for r in range(3) if not 0 <= bad[r + 1] - bad[r] <= 2 or bad[r + 1] > 6]
        for r in wrong:
            assert int(acc[r]) == 0 and rows[r].tolist() == [-1] * 3
    p[0:3] = 0.0
    q[0:2] = 0.0
    acc, rows = ops.verify_drafts(p, q, tok, ptr, u, last, 2)
    assert int(acc[0]) == 0 and rows[0].tolist() == [-1] * 3 and ops.device_error() == (6, 922)
    p[3:6] = NAN
    acc, rows = ops.verify_drafts(p, q, tok, ptr, u, last, 2)
    assert int(acc[1]) == 0 and rows[1].tolist() == [-1] * 3 and ops.device_error() == (6, 922)


def test_verify_strided_rows(cuda):
    from msgl import ops
    p, q, tok, ptr, u, last = problem([3, 1, 4, 0], 1001, 6)
    wide, qwide = torch.full((12, 1024), NAN, device="cuda"), torch.full((8, 1010), NAN, device="cuda")
    wide[:, 1:1002], qwide[:, :1001] = p, q
    want = ops.verify_drafts(p, q, tok, ptr, u, last, 4)
    got = ops.verify_drafts(wide[:, 1:1002], qwide[:, :1001], tok, ptr, u, last, 4)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_verified_tokens_follow_the_target(cuda):
    """Over many uniform numbers the first token is distributed as the target's row, whatever the draft proposes:
    20000 draws of 6 tokens, each share within 5 standard deviations of its probability."""
    from msgl import ops
    g = torch.Generator("cuda").manual_seed(7)
    n, V = 20000, 6
    p = torch.softmax(torch.randn(2, V, generator=g, device="cuda"), 1)
    q = torch.softmax(torch.randn(1, V, generator=g, device="cuda"), 1)
    tok = torch.multinomial(q[0], n, replacement=True, generator=g).int()
    acc, rows = ops.verify_drafts(p.repeat(n, 1), q.expand(n, V).contiguous(), tok, ints(list(range(n + 1))),
                                  torch.rand(n, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda"), 1)
    share = torch.bincount(rows[:, 0].long(), minlength=V).double() / n
    sd = (p[0].double() * (1 - p[0].double()) / n).sqrt()
    assert bool(((share - p[0].double()).abs() < 5 * sd).all())


def test_graph_replay(cuda):
    """Captured with the probabilities in front of it, on new logits and numbers."""
    from msgl import ops
    p, q, tok, ptr, u, last = problem([2, 3, 0, 1], 5000, 8)
    logits = torch.randn(10, 5000, device="cuda")
    t = torch.full((10,), 0.8, device="cuda")
    probs, out = torch.empty_like(logits), (torch.empty(4, dtype=torch.int32, device="cuda"), torch.empty(4, 4, dtype=torch.int32, device="cuda"))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.token_probs(logits, t, out=probs)
            ops.verify_drafts(probs, q, tok, ptr, u, last, 3, out=out)
        for _ in range(3):
            logits.copy_(torch.randn(10, 5000, device="cuda") * 2)
            u.copy_(torch.rand(6, device="cuda"))
            g.replay()
            s.synchronize()
            acc, rows, sure = restate(probs, q, tok, ptr, u, last, 3)
            assert out[0].tolist() == acc and all(not ok or a == b for ok, a, b in zip(sure, out[1].tolist(), rows))
