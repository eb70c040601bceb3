"""QK-norm + rotary positions of three axes + KV append on a B200, against the formula in 64 bits.

Tolerance per element: half a bf16 step of the value (2^-8, the one rounding of the output) plus
the fp32 evaluation: the norm's scale (sum of 128 squares, square root, division, weight) is good
to 2^-18 and the two rotation products with their sum add 2^-22, both relative to the pair's
magnitude |lo| + |hi|; 2^-17 of it covers them. V rows of bf16 input are copies: bit-exact.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

D, EPS = 128, 1e-6


def axis_map(sections, interleaved):
    s0, s1, s2 = sections
    out = []
    for d in range(D // 2):
        if interleaved:
            out.append(1 if d % 3 == 1 and d < 3 * s1 else 2 if d % 3 == 2 and d < 3 * s2 else 0)
        else:
            out.append(0 if d < s0 else 1 if d < s0 + s1 else 2)
    return out


def table(n):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(64, dtype=torch.float64) / 64)
    return torch.cat([ang.cos(), ang.sin()], 1).float().cuda()


def reference(rows, pos, axes, tab, w, eps=EPS):
    """rows [T, n, 128] (float64) normed with weights w [n, 128] and turned; also the magnitudes."""
    y = rows / torch.sqrt(rows.square().mean(-1, keepdim=True) + eps) * w.double()
    at = pos.long()[torch.tensor(axes, device=pos.device)].T
    pair = torch.arange(64, device=pos.device)
    c, s = tab.double()[at, pair][:, None], tab.double()[at, pair + 64][:, None]
    lo, hi = y[..., :64], y[..., 64:]
    mag = (lo.abs() + hi.abs()).repeat(1, 1, 2)
    return torch.cat([lo * c - hi * s, lo * s + hi * c], -1), mag


def inputs(T, hq, hkv, parts, seed=0, max_pos=4096, slots_extra=7):
    g = torch.Generator("cuda").manual_seed(seed)
    nh = hq + 2 * hkv
    if parts:
        x = torch.randn(parts, T, nh * D, generator=g, device="cuda")
        full = x.double().sum(0).view(T, nh, D)
    else:
        x = torch.randn(T, nh * D, generator=g, device="cuda").bfloat16()
        full = x.double().view(T, nh, D)
    pos = torch.randint(0, max_pos, (3, T), generator=g, device="cuda", dtype=torch.int32)
    slots = torch.randperm(T + slots_extra, generator=g, device="cuda")[:T].int()
    kp = torch.full((T + slots_extra, hkv * D), 7.0, device="cuda").bfloat16()
    vp = torch.full_like(kp, -7.0)
    qn = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).bfloat16()
    kn = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).bfloat16()
    return x, full, pos, slots, kp, vp, qn, kn


def call(ops, x, parts, *a, **k):
    return (ops.qknorm_mrope_store_kv_partials if parts else ops.qknorm_mrope_store_kv)(x, *a, **k)


def check(got, ref, mag):
    err = (got.double() - ref).abs()
    assert bool((err <= ref.abs() * 2 ** -8 + mag * 2 ** -17).all()), float((err / mag).max())


@pytest.mark.parametrize("T,hq,hkv", [(1, 16, 8), (5, 8, 1), (37, 32, 8), (300, 32, 4), (3, 5, 3), (1300, 9, 4)])
@pytest.mark.parametrize("sections,interleaved", [((24, 20, 20), True), ((16, 24, 24), False),
                                                  ((64, 0, 0), True), ((0, 0, 64), False),
                                                  ((22, 21, 21), True), ((1, 62, 1), False)])
@pytest.mark.parametrize("parts", [0, 1, 6, 9])
def test_against_formula(cuda, T, hq, hkv, sections, interleaved, parts):
    from msgl import ops
    tab = table(4096)
    x, full, pos, slots, kp, vp, qn, kn = inputs(T, hq, hkv, parts, seed=T + parts)
    if T > 2:
        slots[1] = -1  # a padding token
    q = call(ops, x, parts, kp, vp, pos, slots, tab, qn, kn, hq, hkv, EPS, sections=sections,
             interleaved=interleaved)
    w = torch.cat([qn.expand(hq, D), kn.expand(hkv, D)])
    ref, mag = reference(full[:, :hq + hkv], pos, axis_map(sections, interleaved), tab, w)
    check(q, ref[:, :hq], mag[:, :hq])
    keep = slots >= 0
    at = slots[keep].long()
    check(kp[at].view(-1, hkv, D), ref[keep, hq:], mag[keep, hq:])
    v = full[keep, hq + hkv:].reshape(-1, hkv * D)
    if parts:
        assert bool(((vp[at].double() - v).abs() <= v.abs() * 2 ** -8 + 2 ** -20 * parts).all())
    else:
        assert torch.equal(vp[at].double(), v)
    rest = torch.ones(kp.shape[0], dtype=torch.bool, device="cuda")
    rest[at] = False
    assert bool((kp[rest] == 7).all()) and bool((vp[rest] == -7).all())  # no other slot written
    assert ops.device_error() == (0, 0)


def test_equal_axes_match_the_one_axis_operator(cuda):
    """Positions given once for all axes (row stride 0) turn as msgl_qknorm_rope_store_kv does: both
    round the same fp32 formula, whose sums of squares differ in order (2^-17, as above)."""
    from msgl import ops
    T, hq, hkv = 33, 16, 4
    tab = table(4096)
    x, _, pos, slots, kp, vp, qn, kn = inputs(T, hq, hkv, 0, seed=3)
    one = pos[:1].expand(3, T)
    assert one.stride(0) == 0
    q = ops.qknorm_mrope_store_kv(x, kp, vp, one, slots, tab, qn, kn, hq, hkv, EPS, (24, 20, 20), True)
    kp2, vp2 = torch.full_like(kp, 7.0), torch.full_like(vp, -7.0)
    q2 = ops.qknorm_rope_store_kv(x, kp2, vp2, pos[0].contiguous(), slots, tab, qn, kn, hq, hkv, EPS)
    # one rounding step apart at most where the fp32 values straddle a border
    assert bool(((q.float() - q2.float()).abs() <= q2.float().abs() * 2 ** -7 + 1e-5).all())
    assert bool(((kp.float() - kp2.float()).abs() <= kp2.float().abs() * 2 ** -7 + 1e-5).all())
    assert torch.equal(vp, vp2)


def test_strided_positions_and_out_of_range(cuda):
    """Axis rows of a longer buffer; a position behind the table counts as 0 and a slot behind the
    pool is skipped, both recorded."""
    from msgl import ops
    T, hq, hkv = 6, 8, 2
    tab = table(64)
    x, full, pos, slots, kp, vp, qn, kn = inputs(T, hq, hkv, 0, seed=5, max_pos=64)
    wide = torch.full((3, 50), 63, dtype=torch.int32, device="cuda")
    wide[:, :T] = pos
    q = ops.qknorm_mrope_store_kv(x, kp, vp, wide[:, :T], slots, tab, qn, kn, hq, hkv, EPS, (24, 20, 20), True)
    w = torch.cat([qn.expand(hq, D), kn.expand(hkv, D)])
    ref, mag = reference(full[:, :hq + hkv], pos, axis_map((24, 20, 20), True), tab, w)
    check(q, ref[:, :hq], mag[:, :hq])
    assert ops.device_error() == (0, 0)

    bad, zero = pos.clone(), pos.clone()
    bad[2, 4], zero[2, 4] = 64, 0
    bad[0, 1], zero[0, 1] = -3, 0
    q = ops.qknorm_mrope_store_kv(x, kp, vp, bad, slots, tab, qn, kn, hq, hkv, EPS, (24, 20, 20), True)
    ref, mag = reference(full[:, :hq + hkv], zero, axis_map((24, 20, 20), True), tab, w)
    check(q, ref[:, :hq], mag[:, :hq])
    assert ops.device_error() == (6, 102)

    kp.fill_(7.0), vp.fill_(-7.0)
    slots[3] = kp.shape[0]
    ops.qknorm_mrope_store_kv(x, kp, vp, pos, slots, tab, qn, kn, hq, hkv, EPS, (24, 20, 20), True)
    assert ops.device_error() == (6, 103)
    rest = torch.ones(kp.shape[0], dtype=torch.bool, device="cuda")
    rest[slots[torch.arange(T, device="cuda") != 3].long()] = False
    assert bool((kp[rest] == 7).all()) and bool((vp[rest] == -7).all())


def test_graph_replay_and_side_stream(cuda):
    from msgl import ops
    T, hq, hkv = 12, 16, 8
    tab = table(4096)
    x, full, pos, slots, kp, vp, qn, kn = inputs(T, hq, hkv, 0, seed=9)
    out = torch.empty(T, hq, D, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.qknorm_mrope_store_kv(x, kp, vp, pos, slots, tab, qn, kn, hq, hkv, EPS, (24, 20, 20), True, out=out)
    pos.copy_((pos + 11) % 4096)  # new positions, same buffers
    graph.replay()
    torch.cuda.synchronize()
    w = torch.cat([qn.expand(hq, D), kn.expand(hkv, D)])
    ref, mag = reference(full[:, :hq + hkv], pos, axis_map((24, 20, 20), True), tab, w)
    check(out, ref[:, :hq], mag[:, :hq])
    check(kp[slots.long()].view(T, hkv, D), ref[:, hq:], mag[:, hq:])
