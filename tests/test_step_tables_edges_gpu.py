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
