"""Step tables on a B200: refusals in every warp, calls without requests, requests over borrowed pages."""
import pytest
import torch

from test_step_tables_gpu import PAGE, Pool, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [1, 33, 1000, 1100])
def test_refused_whichever_request_is_bad(cuda, B):
    """One bad length, of another request each time: nothing is written."""
    from msgl import ops
    p = Pool(B, 4, 4 * B, seed=B)
    p.check([0] * B, [20] * B, 20 * B)
    before = [t.clone() for t in (p.table, p.held, p.stack, p.top)]
    out = ops.StepTables(*(torch.full((n,), -5, dtype=torch.int32, device="cuda") for n in (B, B + 1, B, B, B)))
    kept, new = ints([20] * B), ints([1] * B)
    for i in range(200):
        r = i * 31 % B
        kept[r] = -1
        ops.step_tables(kept, new, p.table, p.held, p.stack, p.top, out=out)
        kept[r] = 20
        assert ops.device_error() == (6, 711)
    assert all(bool((t == -5).all()) for t in out)
    assert all(torch.equal(a, b) for a, b in zip(before, (p.table, p.held, p.stack, p.top)))


def test_requests_that_share_a_cached_prefix(cuda):
    """Two requests over the same three leading pages, which a prefix cache owns. Finishing with kept = the borrowed
    tokens gives back their own pages alone; the slot is empty once its held count is 0."""
    from msgl import ops
    p = Pool(3, 10, 24, seed=5)
    cached = [p.free.pop() for _ in range(3)]  # the cache took them before
    p.top.fill_(len(p.free))
    for r in (0, 1):
        p.table[r, :3] = ints(cached)
        p.held[r] = 3
        p.rows[r], p.entries[r][:3] = list(cached), list(cached)
    p.check([48, 48, 0], [30, 5, 40], 75)
    p.check([70, 50, 40], [6, 6, 6], 18)    # rejected drafts
    p.check([48, 56, 46], [0, 6, 6], 12)    # request 0 is done
    assert p.rows[0] == cached and int(p.held[0]) == 3 and not set(p.free) & set(cached)
    p.held[0], p.rows[0] = 0, []
    p.check([0, 62, 52], [100, 6, 6], 112)  # another in its place
    assert not set(p.rows[0]) & set(cached)
    p.check([0, 48, 0], [0, 0, 0], 0)
    p.held[1], p.rows[1] = 0, []
    assert sorted(p.free + cached) == list(range(24)) and ops.device_error() == (0, 0)
