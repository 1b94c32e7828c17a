"""Element counts near the end of 64 bits are refused by the C entry points before any launch."""

import ctypes

import numpy as np
import pytest

from smo_optimizer_b200 import _lib

HUGE = [2 ** 63 - 1, 2 ** 63 - 2048, 2 ** 62, 2 ** 41 + 1]


def _row(kind, n):
    t = np.zeros(1, dtype=_lib.ADAMW_DTYPE)
    t["kind"], t["n"], t["q_block"] = kind, n, 64
    for i, k in enumerate(("param", "grad", "exp_avg", "exp_avg_sq", "m_q", "m_s", "v_q", "v_s")):
        t[k] = (i + 1) << 20
    return t


@pytest.mark.parametrize("n", HUGE)
def test_adamw(n):
    lib = _lib.load()
    for kind in (_lib.SMO_ADAMW_F32, _lib.SMO_ADAMW_8BIT):
        t = _row(kind, n)
        assert lib.smo_adamw_step(t.ctypes.data, 1, None, 0.0, None, None, 0, None) == 1
    for fn in (lib.smo_adamw_decode, lib.smo_adamw_encode):
        assert fn(_row(_lib.SMO_ADAMW_8BIT, n).ctypes.data, 1, None) == 1


@pytest.mark.parametrize("sizes", [[n] for n in (2 ** 63 - 1, 2 ** 63 - 8192, 2 ** 62, 2 ** 44 + 1)] +
                         [[2 ** 63 - 1] * 2, [5, 2 ** 63 - 1, 7], [2 ** 43 + 1] * 2], ids=str)
def test_gradient_norm(sizes):
    lib = _lib.load()
    g = np.zeros(len(sizes), dtype=_lib.GRAD_DTYPE)
    g["grad"], g["n"] = 1 << 20, sizes
    need = lib.smo_grad_norm_workspace_size(len(sizes))
    buf = (ctypes.c_uint8 * (need + 256))()
    ws = (ctypes.addressof(buf) + 255) // 256 * 256
    for max_norm in (0.0, 1.0):
        assert lib.smo_grad_norm(g.ctypes.data, len(sizes), max_norm, 1 << 21, ws, need, None) == 1
