"""The quotient of the 8-bit step takes subnormal denominators as 0: an eps among them is refused."""

import numpy as np
import pytest
import torch

from smo_optimizer_b200 import AdamW, AdamW8bit, _lib

LEAST = 2.0 ** -126  # fp32's smallest normal number


def _p():
    return torch.nn.Parameter(torch.zeros(3))


@pytest.mark.parametrize("eps", [1e-40, LEAST / 2, 2.0 ** -149])
def test_refused_with_8bit_moments(eps):
    with pytest.raises(ValueError, match="epsilon"):
        AdamW8bit([_p()], eps=eps)
    with pytest.raises(ValueError, match="epsilon"):
        AdamW8bit([dict(params=[_p()], eps=eps)])
    AdamW([_p()], eps=eps)
    opt = AdamW8bit([_p()])
    sd = opt.state_dict()
    sd["param_groups"][0]["eps"] = eps
    with pytest.raises(ValueError, match="epsilon"):
        opt.load_state_dict(sd)
    # and by the C entry, where it is a host value
    t = np.zeros(1, dtype=_lib.ADAMW_DTYPE)
    for i, k in enumerate(("param", "grad", "exp_avg", "exp_avg_sq", "m_q", "m_s", "v_q", "v_s")):
        t[k] = (i + 1) << 20
    t["n"], t["q_block"], t["kind"], t["hp"]["eps"] = 16, 64, _lib.SMO_ADAMW_8BIT, eps
    assert _lib.load().smo_adamw_step(t.ctypes.data, 1, None, 0.0, None, None, 0, None) == 1


@pytest.mark.parametrize("eps", [0.0, LEAST, 1e-30, 1e-8, 1.0])
def test_taken(eps):
    for cls in (AdamW, AdamW8bit):
        assert cls([dict(params=[_p()], eps=eps)], eps=eps).param_groups[0]["eps"] == eps
