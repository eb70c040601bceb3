"""Argument checks of the torch front end that need no GPU."""
import pytest
import torch


def test_row_strides():
    """A single row's stride is never used: a row of a tensor of any width is taken."""
    from msgl.ops import _row_stride
    wide = torch.zeros(5, 1001, dtype=torch.bfloat16)
    assert _row_stride(-1, wide[:1, :1000], torch.bfloat16, 1, 1000) == 1000
    assert _row_stride(-1, wide[:, :1000], torch.bfloat16, 5, 1000) == 1001
    assert _row_stride(-1, torch.zeros(5, 1008, dtype=torch.bfloat16)[:, 8:], torch.bfloat16, 5, 1000) == 1008
    for bad in (wide[:, :999], wide.float(), torch.zeros(1000, 5, dtype=torch.bfloat16).t()):
        with pytest.raises(ValueError):
            _row_stride(-1, bad, torch.bfloat16, 5, 1000)
