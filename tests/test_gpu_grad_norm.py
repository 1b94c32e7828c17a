"""grad_norm and clip_grad_norm_ on the GPU against 64 bits."""

import numpy as np
import pytest
import torch

from smo_optimizer_b200 import clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device: GPU tests need a B200")


def _set(sizes, dtypes, seed=0, scale=1.0):
    r = np.random.default_rng(seed)
    params = []
    for i, n in enumerate(sizes):
        p = torch.nn.Parameter(torch.zeros(n, dtype=dtypes[i % len(dtypes)], device="cuda"))
        p.grad = torch.from_numpy(r.normal(0, scale, n).astype(np.float32)).cuda().to(p.dtype)
        params.append(p)
    return params


def _exact(params):
    return float(np.sqrt(np.sum([np.square(p.grad.double().cpu().numpy()).sum() for p in params])))


def _close(got, want):
    # the sum is in 64 bits; the result is rounded to fp32 once
    return abs(float(got) - want) <= 1.01 * EPS32 * want


# a chunk is 8192 elements, a launch sums up to 1184 chunks before it wraps around
SETS = [[1], [7], [8191], [8192], [8193], [3, 9000, 1, 20000], [1184 * 8192 + 5], [2 * 1184 * 8192 + 8192, 11],
        [0, 5, 0], list(range(1, 1500))]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SETS, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_against_64_bits(sizes, dtype):
    params = _set(sizes, [dtype])
    got = grad_norm(params)
    assert got.dtype == torch.float32 and got.dim() == 0 and got.is_cuda
    assert _close(got, _exact(params))
    assert all(torch.equal(grad_norm(params), got) for _ in range(3))


def test_mixed_types_views_and_missing_gradients():
    params = _set([100, 9001, 30, 77777], TYPES)
    flat = torch.randn(5000, device="cuda")
    around = flat[:1].clone(), flat[4002:].clone()
    odd = torch.nn.Parameter(torch.zeros(4001, device="cuda"))
    odd.grad = flat[1:4002]
    turned = torch.nn.Parameter(torch.zeros(40, 30, device="cuda"))
    turned.grad = torch.randn(30, 40, device="cuda").t()
    gap = torch.nn.Parameter(torch.zeros(40, 30, device="cuda"))
    gap.grad = torch.randn(40, 33, device="cuda")[:, :30]
    none = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    assert _close(grad_norm(params + [odd, turned, none]), _exact(params + [odd, turned]))
    everything = params + [odd, turned, gap]
    want = [p.grad.float().cpu() for p in everything]
    total = grad_norm(everything)
    assert _close(total, _exact(everything))
    assert torch.equal(clip_grad_norm_(iter(everything + [none]), 1.5), total)
    c = torch.tensor(1.5) / (total.cpu() + 1e-6)
    for p, w in zip(everything, want):
        assert torch.equal(p.grad.cpu(), (w * c).to(p.dtype))
    assert torch.equal(flat[:1], around[0]) and torch.equal(flat[4002:], around[1]) and none.grad is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[1], [8191, 8192, 8193, 40000], [2048 * 1184 * 4 + 7]], ids=str)
def test_clip_scales_in_place(sizes, dtype):
    params = _set(sizes, [dtype], seed=2)
    kept = [p.grad.clone() for p in params]
    addresses = [p.grad.data_ptr() for p in params]
    norm = clip_grad_norm_(params, 0.5)
    assert _close(norm, float(np.sqrt(sum(np.square(g.double().cpu().numpy()).sum() for g in kept))))
    c = torch.clamp(torch.tensor(0.5, device="cuda") / (norm + 1e-6), max=1.0)
    for p, g, a in zip(params, kept, addresses):
        assert p.grad.data_ptr() == a
        assert torch.equal(p.grad, (g.float() * c).to(dtype))
    # small enough already: unchanged
    kept = [p.grad.clone() for p in params]
    clip_grad_norm_(params, 1e6)
    assert all(torch.equal(p.grad, g) for p, g in zip(params, kept))


def test_large_small_and_not_finite_values():
    p = _set([10000], [torch.float32])[0]
    p.grad.mul_(1e30)  # squares overflow fp32
    assert _close(grad_norm([p]), _exact([p]))
    p.grad.mul_(1e-30).mul_(1e-35)  # squares underflow fp32
    assert _close(grad_norm(p), _exact([p]))
    p.grad.zero_()
    assert float(clip_grad_norm_(p, 1.0)) == 0.0 and not p.grad.any()
    p.grad[77] = float("inf")
    assert float(grad_norm(p)) == float("inf")
    p.grad[78] = float("nan")
    assert np.isnan(float(clip_grad_norm_(p, 1.0)))
    assert torch.isnan(p.grad).all()


def test_two_streams_at_once():
    a, b = _set([3_000_000, 17], [torch.float32], seed=1), _set([2_000_000, 900], [torch.float32], seed=2)
    want = _exact(a), _exact(b)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        with torch.cuda.stream(s):
            got.append((grad_norm(a), want[0]))
        with torch.cuda.stream(t):
            got.append((grad_norm(b), want[1]))
    torch.cuda.synchronize()
    assert all(_close(x, w) for x, w in got)


def test_captured_norm_and_clip_replay():
    params = _set([5000, 123], [torch.float32, torch.bfloat16])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip_grad_norm_(params, 1e9)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(params, 1.0)
    for seed in (5, 6):
        fresh = _set([5000, 123], [torch.float32, torch.bfloat16], seed=seed)
        for p, q in zip(params, fresh):
            p.grad.copy_(q.grad)
        graph.replay()
        want = clip_grad_norm_(fresh, 1.0)
        assert torch.equal(norm, want)
        assert all(torch.equal(p.grad, q.grad) for p, q in zip(params, fresh))


def test_a_parameter_given_twice_counts_once():
    params = _set([5000, 300], [torch.float32])
    want = _exact(params)
    kept = [p.grad.clone() for p in params]
    twice = params + [params[0]]
    assert _close(grad_norm(twice), want)
    norm = clip_grad_norm_(twice, 0.5)
    c = torch.tensor(0.5, device="cuda") / (norm + 1e-6)
    for p, g in zip(params, kept):
        assert torch.equal(p.grad, g * c)
    other = torch.nn.Parameter(torch.zeros(5000, device="cuda"))
    other.grad = params[0].grad
    with pytest.raises(RuntimeError, match="share"):
        grad_norm(params + [other])
