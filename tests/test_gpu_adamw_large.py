"""AdamW and AdamW8bit over sets for which a CTA takes several chunks, and over more tensors than a launch holds."""

import numpy as np
import pytest
import torch

from _adamw_ref import Plain32
from smo_optimizer_b200 import AdamW, AdamW8bit, _lib

pytestmark = pytest.mark.gpu

HP = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
ARGS = (HP["lr"], HP["betas"], HP["eps"], HP["weight_decay"])
# chunks of 2048 elements that make a CTA of the 8-bit step take one more: 148 SMs, 4 CTAs each, 8 waves of them
CHUNK, PER_UNIT = 2048, 148 * 4 * 8


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device: GPU tests need a B200")


def _normal(n, scale, gen, dtype):
    x = torch.randn(n, device="cuda", generator=gen).mul_(scale)
    # stretches of other sizes, zeros among them: blocks and chunks differ
    k = -(-n // 700)
    size = torch.randn(k, device="cuda", generator=gen).exp_()
    size[::17] = 0.0
    return x.mul_(size.repeat_interleave(700)[:n]).to(dtype)


def _sizes(units):
    """Odd sizes of one set that gives CTAs `units` chunks; each tensor alone gives them one."""
    total = (units * PER_UNIT + 200) * CHUNK
    big = [total // 13 + 1237 * (i - 6) + 1 for i in range(13)]
    assert max(big) < 2 * PER_UNIT * CHUNK
    return big[:6] + [1, 70, 2048, 2049, 4096 * units - 1, 2048 * units + 64] + big[6:]


@pytest.mark.parametrize("units, dtype, master, block, clip", [
    (2, torch.float32, False, 64, False), (3, torch.float32, False, 128, True), (8, torch.float32, False, 256, False),
    (2, torch.bfloat16, False, 256, True), (3, torch.bfloat16, True, 64, False), (8, torch.bfloat16, False, 128, True),
    (8, torch.bfloat16, True, 256, True), (2, torch.float16, False, 128, False), (3, torch.float16, True, 256, True),
    (8, torch.float16, False, 64, False), (5, torch.float32, False, 64, True)])
def test_sets_of_several_chunks_a_cta_give_the_bits_of_single_tensors(units, dtype, master, block, clip):
    gen = torch.Generator(device="cuda").manual_seed(units)
    sizes = _sizes(units)
    total = sum(-(-n // CHUNK) for n in sizes)
    assert min(units, 8) == min(total // PER_UNIT, 8)
    kw = dict(HP, block_size=block, min_8bit_numel=0, master_weights=master)
    params = [torch.nn.Parameter(_normal(n, 0.1, gen, dtype)) for n in sizes]
    # one tensor whose first element is not aligned
    params[3] = torch.nn.Parameter(torch.cat([params[3].detach(), params[3].detach()[:1]])[1:])
    alone = [torch.nn.Parameter(p.detach().clone()) for p in params]
    opt = AdamW8bit(params, max_grad_norm=0.25 if clip else None, **kw)
    opts = [AdamW8bit([p], **kw) for p in alone]
    for _ in range(3):
        for p, q in zip(params, alone):
            p.grad = q.grad = _normal(p.numel(), 1e-2, gen, dtype)
        opt.step()
        scale = None
        if clip:
            scale = torch.tensor(0.25, device="cuda") / (opt.last_grad_norm + 1e-6)
            assert float(scale) < 1.0
        for o in opts:
            o.step(grad_scale=scale)
    for p, q, o in zip(params, alone, opts):
        assert torch.equal(p.detach(), q.detach()), p.numel()
        for k, t in o.state[q].items():
            got = opt.state[p][k]
            assert (t == got) if k == "step" else torch.equal(t, got), (k, p.numel())
        assert p.numel() < 10_000 or int(opt.state[p]["m_q"].ne(0).sum()) > p.numel() // 2
    pairs = opt.moments()
    for (m, v), q, o in zip(pairs, alone, opts):
        (m1, v1), = o.moments(q)
        assert torch.equal(m, m1) and torch.equal(v, v1)


def _launches(call):
    lib = _lib.load()
    before = lib.smo_launch_count()
    call()
    return lib.smo_launch_count() - before


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("clip", [False, True])
@pytest.mark.parametrize("block", [None, 64, 128])
def test_more_tensors_of_one_kind_than_a_launch_holds(block, clip, capturable):
    r = np.random.default_rng(5)
    sizes = [int(x) for x in r.integers(1, 400, 1100)]
    normal = lambda n, s: torch.from_numpy(r.normal(0, s, n).astype(np.float32)).cuda()  # noqa: E731
    params = [torch.nn.Parameter(normal(n, 0.1)) for n in sizes]
    kw = dict(HP, max_grad_norm=0.25 if clip else None, capturable=capturable)
    opt = AdamW(params, **kw) if block is None else AdamW8bit(params, block_size=block, min_8bit_numel=0, **kw)
    refs = [Plain32(p.detach().cpu().numpy(), block) for p in params]
    for _ in range(3):
        grads = [normal(n, 1e-2) for n in sizes]
        c = None
        if clip:
            total = np.float32(np.sqrt(sum(np.square(g.double().cpu().numpy()).sum() for g in grads)))
            c = min(np.float32(1), np.float32(0.25) / (total + np.float32(1e-6)))
        for p, g, ref in zip(params, grads, refs):
            p.grad = g
            ref.step(g.cpu().numpy(), *ARGS, scale=c)
        # 340 tensors a launch of the step, 1024 a launch of the norm and one that joins its sums, 512 step counts
        assert _launches(opt.step) == 4 + (3 if clip else 0) + (3 if capturable else 0)
    for p, ref in zip(params, refs):
        st, got = opt.state[p], p.detach().cpu().numpy()
        assert float(st["step"]) == 3
        if block is None:
            assert (got == ref.p).all()
            assert (st["exp_avg"].cpu().numpy() == ref.m).all() and (st["exp_avg_sq"].cpu().numpy() == ref.v).all()
        else:
            assert (np.abs(got.astype(np.float64) - ref.p) <= ref.tol_p).all()
            for k, (q, s) in zip("mv", ref.codes):
                assert (st[k + "_q"].cpu().numpy() == q).all() and (st[k + "_s"].cpu().numpy() == s).all()


def test_a_few_fp32_tensors_before_a_large_8bit_set():
    """Two kinds in one step without a norm: the second kind's launch reads while the first one's ends."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    sizes = [100, 9_000_001, 7, 8_000_003, 3000, 8_500_000]
    params = [torch.nn.Parameter(_normal(n, 0.1, gen, torch.float32)) for n in sizes]
    alone = [torch.nn.Parameter(p.detach().clone()) for p in params]
    opt, opts = AdamW8bit(params, **HP), [AdamW8bit([p], **HP) for p in alone]
    for _ in range(3):
        for p, q in zip(params, alone):
            p.grad = q.grad = _normal(p.numel(), 1e-2, gen, torch.float32)
        assert _launches(opt.step) == 2
        for o in opts:
            o.step()
    for p, q, o in zip(params, alone, opts):
        assert torch.equal(p.detach(), q.detach()), p.numel()
        assert all(torch.equal(t, opt.state[p][k]) for k, t in o.state[q].items() if k != "step")
