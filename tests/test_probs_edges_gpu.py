"""Token probabilities on a B200 at temperatures out of the ordinary."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [1, 1001, 50256, 151936])
def test_temperatures_out_of_the_ordinary(cuda, vocab):
    """NaN gives NaN, an infinite one equal probabilities, the smallest one the largest logit."""
    from msgl import ops
    x = torch.randn(4, vocab, generator=torch.Generator("cuda").manual_seed(vocab), device="cuda")
    p = ops.token_probs(x, torch.tensor([math.nan, math.inf, 1e-45, 0.8], device="cuda"))
    assert bool(torch.isnan(p[0]).all())
    assert bool(((p[1] * vocab - 1).abs() <= 2.0 ** -20).all())
    assert int(p[2].argmax()) == int(x[2].argmax()) and float(p[2].max()) == 1 and int((p[2] != 0).sum()) == 1
    ref = torch.softmax(x[3].double() / torch.tensor(0.8).double(), 0)
    assert bool(((p[3] - ref).abs() <= ref * 2.0 ** -16).all())
