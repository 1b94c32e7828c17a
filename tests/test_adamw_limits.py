"""Bounds on a gradient norm that fp32 cannot tell from 0 are refused, not taken as no bound."""

import pytest
import torch

from smo_optimizer_b200 import AdamW, AdamW8bit, clip_grad_norm_

SMALLEST = 2.0 ** -149  # of fp32


def _p():
    return torch.nn.Parameter(torch.zeros(3))


@pytest.mark.parametrize("bad", [0.0, -1.0, float("nan"), 1e-60, SMALLEST / 2])
def test_refused(bad):
    with pytest.raises(ValueError, match="max_norm"):
        clip_grad_norm_([_p()], bad)
    for cls in (AdamW, AdamW8bit):
        with pytest.raises(ValueError, match="max_grad_norm"):
            cls([_p()], max_grad_norm=bad)
        opt = cls([_p()])
        opt.max_grad_norm = bad
        with pytest.raises(ValueError, match="max_grad_norm"):
            opt._norm_buffers(0, 1)
        assert opt.last_grad_norm is None


@pytest.mark.parametrize("good", [SMALLEST, 1e-30, 1, 1e38, 1e300, float("inf")])
def test_taken(good):
    assert float(clip_grad_norm_([_p()], good)) == 0.0
    for cls in (AdamW, AdamW8bit):
        assert cls([_p()], max_grad_norm=good).max_grad_norm == good
