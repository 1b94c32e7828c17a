"""AdamW8bit's moments over long runs, against moments in 64 bits that never were coded."""

import numpy as np
import pytest
import torch

from smo_optimizer_b200 import AdamW, AdamW8bit

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device: GPU tests need a B200")


def _half(state, key, top, block):
    """Half a code's width at each element, and its block's scale, in 64 bits."""
    c = state[key + "_q"].double().abs()
    s = state[key + "_s"].double().expand(-1, block).reshape(-1)
    # rounding to code c covers (c - 1/2)^2 .. (c + 1/2)^2 steps; a root that would be 0 is lifted to 1
    return ((c + 0.25 + (c == 1)) / top ** 2).reshape(-1) * s, s


@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.9, 0.99), (0.9, 0.999), (0.0, 0.5)], ids=str)
@pytest.mark.parametrize("block", [64, 256])
def test_errors_stay_within_what_roundings_add_up_to(block, betas):
    """m -> beta1 m + .. and u -> sqrt(beta2 u^2 + ..) shrink an error by beta1 and sqrt(beta2) at least, and each
    coding adds half a code at most; with the fp32 roundings of a step: 12 relative to the scales before and after."""
    n, steps = 4 * 256, 1200
    b1, b2 = betas
    gen = torch.Generator(device="cuda").manual_seed(3)
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = AdamW8bit([p], lr=1e-3, betas=betas, block_size=block, min_8bit_numel=0)
    size = torch.randn(n, device="cuda", generator=gen).exp_().mul_(1e-2)
    m = torch.zeros(n, dtype=torch.float64, device="cuda")
    v, tol_m, tol_u, old_m, old_u = (torch.zeros_like(m) for _ in range(5))
    out = [(torch.empty(n, device="cuda"), torch.empty(n, device="cuda"))]
    worst = torch.zeros((), dtype=torch.float64, device="cuda")
    for step in range(steps):
        # gradients whose size falls and rises, some elements without any from a third of the run on
        p.grad = torch.randn(n, device="cuda", generator=gen) * size * float(1.2 + np.sin(step / 100))
        if step > steps // 3:
            p.grad[::5] = 0.0
        opt.step()
        opt.moments([p], out=out)
        g = p.grad.double()
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        half_m, s_m = _half(opt.state[p], "m", 127, block)
        half_u, s_u = _half(opt.state[p], "v", 255, block)
        tol_m = b1 * tol_m + half_m + 12 * EPS32 * (s_m + old_m)
        tol_u = b2 ** 0.5 * tol_u + half_u + 12 * EPS32 * (s_u + old_u)
        old_m, old_u = s_m, s_u
        worst = torch.maximum(worst, ((out[0][0].double() - m).abs() / tol_m).max())
        worst = torch.maximum(worst, ((out[0][1].double().sqrt() - v.sqrt()).abs() / tol_u).max())
    assert float(worst) <= 1.0


def test_codes_beside_a_live_element_keep_what_rounding_keeps():
    """Elements without gradients in a block that another element keeps at its size: codes below
    0.5 / (1 - sqrt(beta1)) and 0.5 / (1 - beta2^(1/4)) stay, as documented; without the live one all of the block falls."""
    block, live = 128, 5
    for b1, b2 in ((0.9, 0.95), (0.9, 0.99), (0.9, 0.999)):
        m = torch.linspace(0.0, 1.0, block, device="cuda").square_()
        m = torch.cat([m, m])
        m[live] = m[block - 1] = 1.0
        p = torch.nn.Parameter(torch.zeros(2 * block, device="cuda"))
        wide = AdamW([p], betas=(b1, b2))
        wide.state[p] = {"step": 100, "exp_avg": m.clone(), "exp_avg_sq": m.square()}
        opt = AdamW8bit([p], betas=(b1, b2), block_size=block, min_8bit_numel=0)
        opt.load_state_dict(wide.state_dict())
        p.grad = torch.zeros(2 * block, device="cuda")
        p.grad[live] = 1.0  # m and v of 1 stay 1
        first = {k: opt.state[p][k + "_q"].clone().double() for k in "mv"}
        steps = 300
        for _ in range(steps):
            opt.step()
        for k, factor, whole in (("m", b1 ** 0.5, b1), ("v", b2 ** 0.25, b2 ** 0.5)):
            now, then = opt.state[p][k + "_q"].double(), first[k]
            others = torch.arange(block, device="cuda") != live
            least = 0.5 / (1 - factor)
            keeps = others & (then[0] < least - 0.01)
            assert torch.equal(now[0][keeps], then[0][keeps]), (k, b1, b2)
            falls = others & (then[0] > least + 0.01)
            assert (now[0][falls] < then[0][falls]).all() and (now[0][falls] >= int(least)).all(), (k, b1, b2)
            # the block without a live element: the codes stand for the same parts of a scale that falls as it should
            assert torch.equal(now[1], then[1])
            scale = float(opt.state[p][k + "_s"][1])
            assert abs(scale - whole ** steps) <= 1e-3 * whole ** steps, (k, scale)


@pytest.mark.parametrize("eps", [2.0 ** -126, 1e-30])
def test_the_least_eps_and_no_gradient(eps):
    """Moments of 0 over eps alone: the parameter only decays."""
    for cls in (AdamW, AdamW8bit):
        p = torch.nn.Parameter(torch.ones(5000, device="cuda"))
        p.grad = torch.zeros_like(p)
        opt = cls([p], lr=0.5, eps=eps, weight_decay=0.5)
        opt.step()
        assert torch.equal(p.detach(), torch.full_like(p, 0.75))
