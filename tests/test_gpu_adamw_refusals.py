"""Calls that AdamW, AdamW8bit and the gradient norms refuse on the GPU, and that leave everything as it was."""

import numpy as np
import pytest
import torch

from smo_optimizer_b200 import AdamW, AdamW8bit

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device: GPU tests need a B200")


def _params(sizes, dtype=torch.float32, seed=0):
    r = np.random.default_rng(seed)
    params = []
    for n in sizes:
        p, g = (torch.from_numpy(r.normal(0, s, n).astype(np.float32)).cuda().to(dtype) for s in (0.1, 0.01))
        params.append(torch.nn.Parameter(p))
        params[-1].grad = g
    return params


@pytest.mark.parametrize("key, change, error", [
    ("m_q", lambda t: t[:-1].clone(), ValueError), ("v_s", lambda t: t[:-1].clone(), ValueError),
    ("v_q", lambda t: t.float(), TypeError), ("m_s", lambda t: t.cpu(), TypeError)])
def test_moments_of_codes_that_do_not_fit(key, change, error):
    params = _params([5000, 6000])
    opt = AdamW8bit(params)
    opt.step()
    want = opt.moments()
    out = [tuple(torch.zeros_like(p) for _ in range(2)) for p in params]
    st = opt.state[params[1]]
    kept, st[key] = st[key], change(st[key])
    for call in (lambda: opt.moments(), lambda: opt.moments(params[1]), lambda: opt.moments(params, out=out), opt.step):
        with pytest.raises(error, match=key):
            call()
    st[key] = kept
    assert all(torch.equal(a, b) for x, y in zip(opt.moments(params, out=out), want) for a, b in zip(x, y))
    assert st["step"] == 1


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_parameters_that_share_memory(cls):
    params = _params([5000, 6000])
    shared = torch.nn.Parameter(params[1].data[10:20])
    shared.grad = torch.ones_like(shared)
    opt = cls(params + [shared])
    before = [p.detach().clone() for p in params]
    for _ in range(2):
        with pytest.raises(ValueError, match="share memory"):
            opt.step()
    assert all(torch.equal(p.detach(), q) for p, q in zip(params, before))
    shared.grad = None
    opt.step()
    assert all(opt.state[p]["step"] == 1 for p in params)
    shared.grad = torch.ones_like(shared)  # the plan of the last step does not hold it
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    params[0].data = params[1].data[:5000]
    shared.grad = None
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    assert all(opt.state[p]["step"] == 1 for p in params)
