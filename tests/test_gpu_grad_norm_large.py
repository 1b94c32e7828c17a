"""grad_norm over sets of more chunks than a launch has CTAs: each then goes on to chunks of later tensors."""

import math

import pytest
import torch

from smo_optimizer_b200 import clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24
CHUNK, CTAS = 8192, 148 * 8 * 4  # elements of a chunk; most CTAs of one launch


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device: GPU tests need a B200")


SETS = [[CTAS * CHUNK], [CTAS * CHUNK + 5], [CTAS * CHUNK - CHUNK + 1, 9, CHUNK],
        # more than two rounds: a CTA passes over small tensors from one chunk to its next
        [30_000_001, 8191, 5, 25_000_003] + [8193, 1, 300, 16384] * 40 + [29_000_011, 4],
        [700 * CHUNK - 3] * 15]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", SETS, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_clip_against_64_bits(sizes, dtype):
    gen = torch.Generator(device="cuda").manual_seed(len(sizes))
    params = []
    for i, n in enumerate(sizes):
        p = torch.nn.Parameter(torch.empty(n, dtype=dtype, device="cuda"))
        p.grad = torch.randn(n, device="cuda", generator=gen).mul_(0.5 + i % 3).to(dtype)
        params.append(p)
    assert sum(-(-n // CHUNK) for n in sizes) > CTAS or sizes == SETS[0]
    # 64-bit sums of 64-bit squares, here by torch and then by math.fsum: off by far less than an fp32 rounding
    want = math.sqrt(math.fsum(float(p.grad.double().square().sum()) for p in params))
    norm = grad_norm(params)
    assert abs(float(norm) - want) <= 1.01 * EPS32 * want
    assert all(torch.equal(grad_norm(params), norm) for _ in range(2))
    kept = [p.grad.clone() for p in params]
    assert torch.equal(clip_grad_norm_(params, 2.0), norm)
    c = torch.tensor(2.0, device="cuda") / (norm + 1e-6)
    assert all(torch.equal(p.grad, (g.float() * c).to(dtype)) for p, g in zip(params, kept))
