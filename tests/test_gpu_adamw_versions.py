"""What the library writes in place, autograd sees as written."""

import pytest
import torch

from smo_optimizer_b200 import AdamW, AdamW8bit, clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device: GPU tests need a B200")


def _params(sizes):
    params = [torch.nn.Parameter(torch.ones(n, device="cuda")) for n in sizes]
    for p in params:
        p.grad = torch.full_like(p, 0.5)
    return params


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_inference_tensors_are_written_in_inference_mode_only(cls):
    """As by torch's own operations; refused before anything is written."""
    with torch.inference_mode():
        params = _params([5000, 30])
        out = [tuple(torch.zeros_like(p) for _ in range(2)) for p in params]
        opt = cls(params, max_grad_norm=1.0)
        opt.step()
        clip_grad_norm_(params, 0.25)
    everything = params + [p.grad for p in params] + [t for p in params for t in opt.state[p].values() if torch.is_tensor(t)]
    before = [t.clone() for t in everything]
    calls = [opt.step, lambda: clip_grad_norm_(params, 0.125), lambda: clip_grad_norm_(params[::-1], 0.125)]
    if cls is AdamW8bit:
        calls += [lambda: opt.moments(params, out=out), lambda: opt.moments(params[0], out=out[:1])]
    for call in calls:
        with pytest.raises(RuntimeError, match="inference"):
            call()
    assert all(torch.equal(a, b) for a, b in zip(everything, before)) and not any(t.any() for pair in out for t in pair)
    assert all(opt.state[p]["step"] == 1 for p in params)
    assert float(grad_norm(params)) == pytest.approx(0.25, rel=1e-4)  # reads only
    with torch.inference_mode():
        opt.step()
        if cls is AdamW8bit:
            assert opt.moments(params, out=out) is not None and out[0][1].any()
    assert all(opt.state[p]["step"] == 2 for p in params)


@pytest.mark.parametrize("mixed", [False, True])
def test_moments_written_to_tensors_of_the_caller(mixed):
    """All parameters coded, and one with fp32 moments among them (another path)."""
    params = _params([5000, 30] if mixed else [5000, 6000])
    opt = AdamW8bit(params)
    opt.step()
    out = [tuple(torch.zeros_like(p) for _ in range(2)) for p in params]
    w = torch.ones(params[0].shape, device="cuda", requires_grad=True)
    loss = (w * out[0][1]).sum()  # keeps out[0][1] for the gradient of w
    before = [t._version for pair in out for t in pair]
    opt.moments(params, out=out)
    assert all(t._version > v for t, v in zip((t for pair in out for t in pair), before))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
