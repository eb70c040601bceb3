"""Low-rank adapters of many requests on a B200, against the formula in 64 bits.

Tolerance per element. The two products accumulate in fp32: each MMA step of 16 products rounds or
truncates its partial sum by at most 2^-22 of the magnitudes it adds, over K / 16 steps, at most 16
K-range sums, and (three bf16 terms) 3 rank / 16 steps: (K / 16 + 3 rank / 16 + 20) 2^-22 of
M = |scale| sum_r |B| sum_k |A| |x|. The bf16 result rounds once (2^-8 of the value) and takes h, up
to 16 rows a request, as two bf16 terms (2^-16 of M: 2^-8 of a remainder of at most 2^-8), in longer
chunks as one: each of the rank's h off by at most 2^-8 of itself, in all 2^-8 of
H = |scale| sum_r |B| |h_r|.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(lens, K, N, R, n, seed=0, none=()):
    g = torch.Generator("cuda").manual_seed(seed)
    T = sum(lens)
    x = torch.randn(T, K, generator=g, device="cuda").bfloat16()
    a = (torch.randn(n, R, K, generator=g, device="cuda") * K ** -0.5).bfloat16()
    b = (torch.randn(n, N, R, generator=g, device="cuda") * R ** -0.5).bfloat16()
    sc = torch.rand(n, generator=g, device="cuda") + 0.5
    ids = torch.tensor([-1 if r in none else (r * 7 + 3) % n for r in range(len(lens))],
                       dtype=torch.int32, device="cuda")
    y = torch.randn(T, N, generator=g, device="cuda").bfloat16()
    indptr = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    return x, a, b, sc, ids, y, indptr


def reference(x, a, b, sc, ids, lens):
    d = torch.zeros(x.shape[0], b.shape[1], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(d)
    mag.one_term = torch.zeros_like(d)  # H, where h is one bf16 term
    t = 0
    for r, q in zip(ids.tolist(), lens):
        if r >= 0:
            A, B, X = a[r].double(), b[r].double(), x[t:t + q].double()
            d[t:t + q] = sc[r].double() * (X @ A.T) @ B.T
            mag[t:t + q] = sc[r].double() * (X.abs() @ A.abs().T) @ B.abs().T
            if max(lens) > 16:
                mag.one_term[t:t + q] = sc[r].double() * (X @ A.T).abs() @ B.abs().T
        t += q
    return d, mag


def steps(K, R):
    return (K / 16 + 3 * R / 16 + 20) * 2 ** -22


def check_partial(p, d, mag, K, R):
    assert bool(((p.double() - d).abs() <= mag * steps(K, R)).all()), float(((p.double() - d).abs() / (mag + 1e-30)).max())


def check_add(o, y, d, mag, K, R):
    ref = y.double() + d
    tol = ref.abs() * 2 ** -8 + mag * (steps(K, R) + 2 ** -16) + mag.one_term * 2 ** -8 + y.double().abs() * 2 ** -23
    assert bool(((o.double() - ref).abs() <= tol).all())


CASES = [
    # lens, K, N, R, adapters, requests without one
    ([1], 1024, 4096, 16, 4, ()),
    ([1], 8, 8, 8, 1, ()),                       # the smallest sizes
    ([1] * 9, 1000, 264, 24, 3, (2, 5)),         # sizes that end inside tiles
    ([1] * 130, 2048, 1024, 8, 48, (0, 129)),
    ([1] * 40, 4096, 6144, 128, 5, ()),
    ([3, 1, 0, 16, 7], 1024, 520, 32, 4, (1,)),  # short chunks, an empty request
    ([17, 1, 0, 64, 65, 130], 1032, 776, 64, 3, (3,)),
    ([500, 700], 2048, 1024, 48, 2, ()),
    ([257], 4096, 512, 128, 1, ()),
    ([5, 20], 256, 128, 16, 2, (0, 1)),          # nobody has an adapter
]


@pytest.mark.parametrize("lens,K,N,R,n,none", CASES)
def test_against_formula(cuda, lens, K, N, R, n, none):
    from msgl import ops
    x, a, b, sc, ids, y, indptr = make(lens, K, N, R, n, seed=K + N, none=none)
    d, mag = reference(x, a, b, sc, ids, lens)
    kw = {} if max(lens) == 1 and 0 not in lens else dict(q_indptr=indptr, max_q_len=max(lens))
    p = ops.lora_partial(x, a, b, sc, ids, **kw)
    check_partial(p, d, mag, K, R)
    o = ops.lora_add(x, a, b, sc, ids, y, **kw)
    check_add(o, y, d, mag, K, R)
    t = 0
    for r, q in zip(ids.tolist(), lens):  # rows without an adapter: zero, and y bit for bit
        if r < 0:
            assert bool((p[t:t + q] == 0).all()) and torch.equal(o[t:t + q], y[t:t + q])
        t += q
    assert torch.equal(p, ops.lora_partial(x, a, b, sc, ids, **kw))  # same bits again
    inplace = y.clone()
    ops.lora_add(x, a, b, sc, ids, inplace, out=inplace, **kw)
    assert torch.equal(inplace, o)
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("lens", [[1] * 20, [9, 16], [17, 40], [90, 200, 1]])
@pytest.mark.parametrize("R", [16, 24, 64, 128])
def test_cancelling_ranks(cuda, lens, R):
    """Ranks in pairs whose terms nearly cancel, and cancel y: what h is rounded by shows in the result.
    Two bf16 terms leave 2^-16 of each h, 2^-16 of H in all, however many rows a request has."""
    from msgl import ops
    K, N = 64, 264
    x, a, b, sc, ids, _, indptr = make(lens, K, N, R, 3, seed=R)
    a[:, 1::2] = (a[:, ::2].float() * (1 + 2 ** -6)).bfloat16()
    b[:, :, 1::2] = -b[:, :, ::2]
    d, mag = reference(x, a, b, sc, ids, lens)
    H = torch.cat([sc[r].double() * (X @ a[r].double().T).abs() @ b[r].double().abs().T
                   for r, X in zip(ids.tolist(), x.double().split(lens))])
    y = (-d).bfloat16()
    for _y in (torch.zeros_like(y), y):
        ref = _y.double() + d
        out = ops.lora_add(x, a, b, sc, ids, _y, q_indptr=indptr, max_q_len=max(lens))
        tol = ref.abs() * 2 ** -8 + mag * steps(K, R) + H * 2 ** -16 + _y.double().abs() * 2 ** -23
        assert bool(((out.double() - ref).abs() <= tol).all()), float(((out.double() - ref).abs() / tol).max())
    assert ops.device_error() == (0, 0)


def test_strided_rows_and_rows_behind_the_last_request(cuda):
    """A column range of a fused projection, x as a column range, and padding rows."""
    from msgl import ops
    lens = [9, 30]
    K, N, R = 512, 256, 16
    x, a, b, sc, ids, _, indptr = make(lens, K, N, R, 2, seed=1)
    T = sum(lens)
    wide_x = torch.full((T + 4, K + 24), float("nan"), device="cuda").bfloat16()
    wide_x[:T, 8:8 + K] = x
    g = torch.Generator("cuda").manual_seed(2)
    fused = torch.randn(T + 4, 3 * N, generator=g, device="cuda").bfloat16()
    before = fused.clone()
    view = fused[:, N:2 * N]
    ops.lora_add(wide_x[:, 8:8 + K], a, b, sc, ids, view, q_indptr=indptr, max_q_len=30, out=view)
    d, mag = reference(x, a, b, sc, ids, lens)
    check_add(view[:T], before[:T, N:2 * N], d, mag, K, R)
    assert torch.equal(fused[:, :N], before[:, :N]) and torch.equal(fused[:, 2 * N:], before[:, 2 * N:])
    assert torch.equal(fused[T:], before[T:])  # rows behind the last request
    part = torch.full((T + 4, N + 8), 5.0, device="cuda")
    ops.lora_partial(wide_x[:, 8:8 + K], a, b, sc, ids, q_indptr=indptr, max_q_len=30, out=part[:, :N])
    check_partial(part[:T, :N], d, mag, K, R)
    assert bool((part[T:] == 5).all()) and bool((part[:, N:] == 5).all())
    assert ops.device_error() == (0, 0)


def test_one_row_of_a_tensor_of_any_width(cuda):
    from msgl import ops
    K, N, R = 1000, 264, 16
    x, a, b, sc, ids, y, _ = make([1], K, N, R, 2, seed=3)
    wide = [torch.zeros(3, n + 3, dtype=t.dtype, device="cuda") for t, n in ((x, K), (y, N), (y.float(), N))]
    wide[0][:1, :K], wide[1][:1, :N] = x, y
    x1, y1 = wide[0][:1, :K], wide[1][:1, :N]
    d, mag = reference(x, a, b, sc, ids, [1])
    check_partial(ops.lora_partial(x1, a, b, sc, ids, out=wide[2][:1, :N]), d, mag, K, R)
    assert ops.lora_add(x1, a, b, sc, ids, y1, out=y1) is y1
    check_add(y1, y, d, mag, K, R)
    assert all(bool((w[1:] == 0).all()) and bool((w[0, -3:] == 0).all()) for w in wide)
    assert ops.device_error() == (0, 0)


@pytest.mark.parametrize("lens", [[1, 1, 1], [20, 40, 70]])
def test_a_row_does_not_reach_another(cuda, lens):
    """NaN and infinite rows, adapters and weights of others change nothing for a request."""
    from msgl import ops
    K, N, R = 256, 128, 16
    x, a, b, sc, ids, y, indptr = make(lens, K, N, R, 3, seed=4)
    kw = dict(q_indptr=indptr, max_q_len=max(lens))
    ids.copy_(torch.tensor([0, 1, 2], dtype=torch.int32))
    clean = ops.lora_add(x, a, b, sc, ids, y, **kw)
    x[lens[0]:lens[0] + lens[1]] = float("nan")
    a[1], b[1] = float("inf"), float("nan")
    x[-1] = float("-inf")
    got = ops.lora_add(x, a, b, sc, ids, y, **kw)
    assert torch.equal(got[:lens[0]], clean[:lens[0]])
    assert torch.equal(got[lens[0] + lens[1]:-1], clean[lens[0] + lens[1]:-1])
    assert bool(got[lens[0]:lens[0] + lens[1]].isnan().all())


@pytest.mark.parametrize("lens", [[1], [1] * 20, [3, 16, 1], [20, 70]])
@pytest.mark.parametrize("R", [8, 16, 24, 40, 72])
def test_infinities_are_those_of_the_formula(cuda, lens, R):
    """An infinite element of x, then an infinite weight: infinities of the formula's sign where the formula
    has them, at ranks that end inside the MMA's 16 and at full ones, and finite values elsewhere."""
    from msgl import ops
    K, N, n = 64, 136, 2
    x, a, b, sc, ids, y, indptr = make(lens, K, N, R, n, seed=R)
    T = sum(lens)
    x.fill_(1.0), a.fill_(2.0 ** -6), sc.fill_(1.0)
    b.copy_(b.abs() + 2.0 ** -7)
    b[:, 5::7] *= -1
    kws = [dict(q_indptr=indptr, max_q_len=max(lens))] + ([{}] if max(lens) == 1 else [])
    for kind in ("x", "weight"):
        if kind == "x":
            x[T // 2, 9] = float("inf")
        else:
            x.fill_(1.0)  # every h is 1: nothing is left of it behind its first term
            b[:, 3, R - 1], b[:, 12, 0] = float("inf"), float("-inf")
        d, mag = reference(x, a, b, sc, ids, lens)
        ref = y.double() + d
        assert bool(ref.isinf().any()) and not bool(ref.isnan().any())
        fin = ref.isfinite()
        for kw in kws:
            o, p = ops.lora_add(x, a, b, sc, ids, y, **kw).double(), ops.lora_partial(x, a, b, sc, ids, **kw).double()
            assert torch.equal(o[~fin], ref[~fin]) and torch.equal(p[~fin], d[~fin])
            assert bool(((o - ref).abs()[fin] <= (ref.abs() * 2 ** -8 + mag * (steps(K, R) + 2 ** -16))[fin]).all())
            assert bool(((p - d).abs()[fin] <= (mag * steps(K, R))[fin]).all())
    assert ops.device_error() == (0, 0)


def test_bad_ids_and_rows_are_recorded(cuda):
    from msgl import ops
    lens = [4, 6]
    x, a, b, sc, ids, y, indptr = make(lens, 128, 64, 8, 2, seed=6)
    ids[1] = 2  # no such adapter
    o = ops.lora_add(x, a, b, sc, ids, y, q_indptr=indptr, max_q_len=6)
    assert ops.device_error() == (6, 810)
    assert torch.equal(o[4:], y[4:]) and not torch.equal(o[:4], y[:4])
    ids[1] = 1
    o = ops.lora_add(x, a, b, sc, ids, y, q_indptr=indptr, max_q_len=5)  # request 1 has 6 rows
    assert ops.device_error() == (6, 811)
    assert torch.equal(o[4:], y[4:]) and not torch.equal(o[:4], y[:4])
    indptr[2] = 11  # behind the last row
    o = ops.lora_add(x, a, b, sc, ids, y, q_indptr=indptr, max_q_len=16)
    assert ops.device_error() == (6, 811)
    assert torch.equal(o[4:], y[4:])


def test_two_captured_graphs(cuda):
    """Two graphs with a workspace each, replayed in turn on new inputs."""
    from msgl import ops
    K, N, R = 512, 256, 16
    sets, graphs = [], []
    for s in range(2):
        lens = [1] * (5 + s)
        x, a, b, sc, ids, y, _ = make(lens, K, N, R, 2, seed=20 + s)
        ws, out = ops.lora_workspace(len(lens), K, R), torch.empty_like(y)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            ops.lora_add(x, a, b, sc, ids, y, workspace=ws, out=out)
        sets.append((lens, x, a, b, sc, ids, y, ws, out))
        graphs.append(g)
    for _ in range(2):
        for (lens, x, a, b, sc, ids, y, _, out), g in zip(sets, graphs):
            x.mul_(-0.5)
            g.replay()
        torch.cuda.synchronize()
        for lens, x, a, b, sc, ids, y, _, out in sets:
            d, mag = reference(x, a, b, sc, ids, lens)
            check_add(out, y, d, mag, K, R)


def test_as_one_more_partial_of_a_projection(cuda):
    """qkv projection as split-K partials, the adapters as the slab behind them, summed by the QK-norm
    kernel: V rows against the product in 64 bits (fp32 sums, one bf16 rounding)."""
    from msgl import ops
    T, K, hq, hkv, R = 12, 1024, 8, 2, 16
    N = (hq + 2 * hkv) * 128
    x, a, b, sc, ids, _, _ = make([1] * T, K, N, R, 3, seed=8, none=(4,))
    w = (torch.randn(N, K, generator=torch.Generator("cuda").manual_seed(9), device="cuda") * K ** -0.5).bfloat16()
    S = ops.gemm_partials_splits(T, N, K)
    parts = torch.empty(S + 1, T, N, device="cuda")
    ops.linear_partials(x, w, S, out=parts[:S])
    ops.lora_partial(x, a, b, sc, ids, out=parts[S])
    kp = torch.zeros(T, hkv * 128, dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    tab = torch.ones(16, 128, device="cuda")
    one = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(3, T, dtype=torch.int32, device="cuda")
    slots = torch.arange(T, dtype=torch.int32, device="cuda")
    ops.qknorm_mrope_store_kv_partials(parts, kp, vp, pos, slots, tab, one, one, hq, hkv, 1e-6, (64, 0, 0))
    d, mag = reference(x, a, b, sc, ids, [1] * T)
    v = (x.double() @ w.double().T + d)[:, -hkv * 128:]
    size = (x.double().abs() @ w.double().abs().T + mag)[:, -hkv * 128:]
    assert bool(((vp.double() - v).abs() <= v.abs() * 2 ** -8 + size * 2 * steps(K, R)).all())


@pytest.mark.parametrize("partial", [False, True])
@pytest.mark.parametrize("B,n,R", [(300, 2, 16), (300, 7, 40), (260, 200, 8), (33, 1, 128), (129, 40, 64)])
def test_many_requests_per_adapter(cuda, partial, B, n, R):
    """Decode batches with fewer adapters than requests: more than 16 rows of one adapter, adapters
    that nobody uses, rows without one, an id that does not exist."""
    from msgl import ops
    K, N = 1000, 776
    x, a, b, sc, ids, y, _ = make([1] * B, K, N, R, n, seed=B + n)
    g = torch.Generator("cuda").manual_seed(7)
    ids.copy_(torch.randint(-1, max(1, n - 1), (B,), generator=g, device="cuda").int())
    ids[B // 2] = n  # no such adapter: none
    d, mag = reference(x, a, b, sc, torch.where(ids < n, ids, -1), [1] * B)
    if partial:
        check_partial(ops.lora_partial(x, a, b, sc, ids), d, mag, K, R)
    else:
        check_add(ops.lora_add(x, a, b, sc, ids, y), y, d, mag, K, R)
    assert ops.device_error() == (6, 810)
