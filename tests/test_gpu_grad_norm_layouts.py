"""grad_norm and clip_grad_norm_ over gradients with repeated, missing or shared elements."""

import numpy as np
import pytest
import torch

from smo_optimizer_b200 import clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device: GPU tests need a B200")


def _holder(grad):
    p = torch.nn.Parameter(torch.empty_strided(grad.shape, grad.stride(), dtype=grad.dtype, device="cuda")
                           if 0 not in grad.stride() else torch.empty(grad.shape, dtype=grad.dtype, device="cuda"))
    p.grad = grad
    return p


def _randn(*shape, seed=0, dtype=torch.float32):
    r = np.random.default_rng(seed)
    return torch.from_numpy(r.normal(0, 1, shape).astype(np.float32)).cuda().to(dtype)


def _exact(params):
    return float(np.sqrt(np.sum([np.square(p.grad.double().cpu().numpy()).sum() for p in params])))


def _close(got, want):
    # sums in 64 bits, one rounding to fp32
    return abs(float(got) - want) <= 1.01 * EPS32 * want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("expand", [lambda t: t[:, :1].expand(40, 30), lambda t: t[:1].expand(40, 30),
                                    lambda t: t[0, 0].expand(40, 30), lambda t: t[:, None, ::2].expand(40, 7, 15),
                                    lambda t: t[:20, ::3][:, :, None].expand(20, 10, 3)])
def test_repeated_elements_are_scaled_once(expand, dtype):
    base = _randn(40, 30, seed=1, dtype=dtype)
    params = [_holder(_randn(500, seed=2, dtype=dtype)), _holder(expand(base)), _holder(_randn(300, seed=3))]
    kept = [p.grad.clone() for p in params]
    untouched = base.clone()
    want = _exact(params)
    assert _close(grad_norm(params), want)
    norm = clip_grad_norm_(params, 0.5)
    assert _close(norm, want)
    c = torch.tensor(0.5, device="cuda") / (norm + 1e-6)
    for p, g in zip(params, kept):
        assert torch.equal(p.grad, (g.float() * c).to(g.dtype))
    # elements of the buffer that the gradient does not show stay
    shown = expand(torch.arange(base.numel(), device="cuda").view(40, 30)).reshape(-1)
    hidden = torch.ones(base.numel(), dtype=torch.bool, device="cuda")
    hidden[shown] = False
    assert torch.equal(base.view(-1)[hidden], untouched.view(-1)[hidden])


def test_elements_that_overlap_otherwise_are_not_clipped():
    a, buffer = _holder(_randn(500, seed=2)), _randn(40, seed=4)
    params = [a, torch.nn.Parameter(torch.empty(10, 10, device="cuda"))]
    params[1].grad = buffer.as_strided((10, 10), (2, 1))
    kept = a.grad.clone(), buffer.clone()
    assert _close(grad_norm(params), _exact(params))
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grad_norm_(params, 0.5)
    assert torch.equal(a.grad, kept[0]) and torch.equal(buffer, kept[1])


def test_a_view_with_a_gap_and_the_span_around_it():
    """A strided gradient inside another one: each of its elements is scaled once all the same."""
    buffer = _randn(64, 32, seed=5)
    params = [_holder(buffer), _holder(buffer[:, 3:20])]
    kept, want = buffer.clone(), _exact(params)
    norm = clip_grad_norm_(params, 0.5)
    assert _close(norm, want)
    assert torch.equal(buffer, kept * (torch.tensor(0.5, device="cuda") / (norm + 1e-6)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_spans_that_share_elements_are_not_clipped(dtype):
    buffer = _randn(1000, seed=6, dtype=dtype)
    kept = buffer.clone()
    for a, b in ((buffer[:600], buffer[599:]), (buffer, buffer[400:410]), (buffer[1:3], buffer[:2])):
        params = [_holder(a), _holder(b)]
        assert _close(grad_norm(params), _exact(params))
        for order in (params, params[::-1]):
            with pytest.raises(RuntimeError, match="share"):
                clip_grad_norm_(order, 0.5)
        assert torch.equal(buffer, kept)
    # neighbours share nothing
    norm = clip_grad_norm_([_holder(buffer[:600]), _holder(buffer[600:])], 0.5)
    assert torch.equal(buffer, (kept.float() * (torch.tensor(0.5, device="cuda") / (norm + 1e-6))).to(dtype))


@pytest.mark.parametrize("call", [grad_norm, lambda ps: clip_grad_norm_(ps, 0.5)], ids=["norm", "clip"])
def test_copies_are_made_of_the_gradients_that_need_one_only(call):
    big, gap = _holder(_randn(4_000_000, seed=7)), _holder(_randn(40, 33, seed=8)[:, :30])
    call([big, gap])
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    norm = call([big, gap])
    # the gradient is 16 MB; a workspace is a few times 4736 sums of 8 bytes
    assert torch.cuda.max_memory_allocated() - before < 1 << 20, norm
