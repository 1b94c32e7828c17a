"""Descriptors of 8-bit moments are made of codes and scales that fit their parameter only."""

import numpy as np
import pytest
import torch

from smo_optimizer_b200 import _lib, adamw


def _coded(n, block):
    nb = -(-n // block)
    return {"step": 1, "m_q": torch.zeros((nb, block), dtype=torch.int8), "m_s": torch.zeros((nb, 1)),
            "v_q": torch.zeros((nb, block), dtype=torch.uint8), "v_s": torch.zeros((nb, 1))}


def _row(p, state):
    rec = np.zeros(1, dtype=_lib.ADAMW_DTYPE)
    adamw._coded_row(rec[0], p, state)
    return rec[0]


@pytest.mark.parametrize("block", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 64, 1000])
def test_codes_that_fit(n, block):
    p, st = torch.nn.Parameter(torch.zeros(n)), _coded(n, block)
    rec = _row(p, st)
    assert rec["n"] == n and rec["q_block"] == block and rec["kind"] == _lib.SMO_ADAMW_8BIT
    assert all(rec[k] == st[k].data_ptr() for k in ("m_q", "m_s", "v_q", "v_s"))


@pytest.mark.parametrize("key, change, error", [
    ("m_q", lambda t: t[:-1], ValueError), ("v_q", lambda t: t[:-1], ValueError),
    ("m_s", lambda t: t[:-1], ValueError), ("v_s", lambda t: t[:-1], ValueError),
    ("m_q", lambda t: t.view(-1, 32), ValueError), ("m_q", lambda t: t.view(-1), ValueError),
    ("v_q", lambda t: t.t().contiguous().t(), ValueError), ("m_s", lambda t: torch.cat([t, t], 1)[:, :1], ValueError),
    ("m_q", lambda t: t.float(), TypeError), ("v_q", lambda t: t.to(torch.int8), TypeError),
    ("v_s", lambda t: t.half(), TypeError), ("m_s", lambda t: t.to("meta"), TypeError), ("v_s", lambda t: None, TypeError)])
def test_codes_that_do_not_fit_are_refused(key, change, error):
    p, st = torch.nn.Parameter(torch.zeros(1000)), _coded(1000, 128)
    st[key] = change(st[key])
    with pytest.raises(error, match=key):
        _row(p, st)


def test_codes_of_a_smaller_parameter_are_refused():
    with pytest.raises(ValueError, match="m_q"):
        _row(torch.nn.Parameter(torch.zeros(1025)), _coded(1024, 128))
