"""AdamW, AdamW8bit and the gradient norm on the GPU give the same bits whatever torch's default dtype is."""

import copy

import numpy as np
import pytest
import torch

from smo_optimizer_b200 import AdamW, AdamW8bit, clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu

SIZES = [1, 7, 300, 4097, 20003] * 8  # more scalars than the allocator's rounding would hide


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("no CUDA device: GPU tests need a B200")


def _run(cls, default):
    """Three clipped steps with scalars formed on the device, from a loaded step count of 1001."""
    kept = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        r = np.random.default_rng(0)
        normal = lambda n, s: torch.from_numpy(r.normal(0, s, n).astype(np.float32)).cuda().bfloat16()  # noqa: E731
        params = [torch.nn.Parameter(normal(n, 0.1)) for n in SIZES]
        opt = cls(params, lr=1e-2, betas=(0.9, 0.9999), master_weights=True, max_grad_norm=0.5, capturable=True)
        for step in range(3):
            for p in params:
                p.grad = normal(p.numel(), 1e-2)
            opt.step()
            if step == 0:
                saved = opt.state_dict()
                for st in saved["state"].values():
                    st["step"] = 1001
                opt.load_state_dict(saved)
        norms = [opt.last_grad_norm, grad_norm(params), clip_grad_norm_(params, 0.25)]
        states = [t for p in params for t in opt.state[p].values()]
        return [t.detach().cpu() for t in params + states + norms + [p.grad for p in params]]
    finally:
        torch.set_default_dtype(kept)


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float16, torch.float64], ids=str)
@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_the_default_dtype_changes_nothing(cls, default):
    want, got = _run(cls, torch.float32), _run(cls, default)
    assert len(got) == len(want)
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(got, want))
    assert 1003.0 in [float(t) for t in got if t.dtype == torch.float32 and t.dim() == 0]


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_a_load_between_replays_of_a_captured_step(cls):
    """A graph goes on with the state that was loaded, as eager steps do."""
    r = np.random.default_rng(1)
    sizes = [5000, 30, 2049]
    normal = lambda n, s: torch.from_numpy(r.normal(0, s, n).astype(np.float32)).cuda()  # noqa: E731
    start = [normal(n, 0.1) for n in sizes]
    grads = [[normal(n, 1e-2) for n in sizes] for _ in range(6)]
    kw = dict(capturable=True, max_grad_norm=0.1)
    lr, lr2 = torch.tensor(1e-2, device="cuda"), torch.tensor(1e-2, device="cuda")
    params, plain = ([torch.nn.Parameter(t.clone()) for t in start] for _ in range(2))
    opt, ref = cls(params, lr=lr, **kw), cls(plain, lr=lr2, **kw)

    def set_grads(step):
        for ps in (params, plain):
            for p, g in zip(ps, grads[step]):
                if p.grad is None:
                    p.grad = g.clone()
                else:
                    p.grad.copy_(g)

    set_grads(0)
    opt.step()
    ref.step()
    saved = copy.deepcopy(opt.state_dict())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for step in range(1, 6):
        set_grads(step)
        if step == 3:
            saved["param_groups"][0]["lr"] = torch.tensor(0.5)
            opt.load_state_dict(saved)
            ref.load_state_dict(saved)
            assert opt.param_groups[0]["lr"] is lr and float(lr) == 0.5
            ref.param_groups[0]["lr"] = torch.tensor(0.5, device="cuda")
        graph.replay()
        ref.step()
        assert torch.equal(opt.last_grad_norm, ref.last_grad_norm), step
        for p, q in zip(params, plain):
            assert torch.equal(p.detach(), q.detach()), step
            assert opt.state[p].keys() == ref.state[q].keys()
            assert all(torch.equal(t, ref.state[q][k]) for k, t in opt.state[p].items()), step
    assert float(opt.state[params[0]]["step"]) == 4.0
    opt.step()
    ref.step()
    assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(params, plain))
