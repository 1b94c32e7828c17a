"""CPU checks of AdamW, AdamW8bit and the gradient norms: refusals, descriptor
validation, scalars, layout of the binding, ZeRO cost model."""

import ctypes

import numpy as np
import pytest
import torch
from torch.optim.optimizer import register_optimizer_step_post_hook

from smo_optimizer_b200 import AdamW, AdamW8bit, _host, _lib, clip_grad_norm_, grad_norm
from smo_optimizer_b200.optimizers import _host_ext
from smo_optimizer_b200.zero import adamw_step_bytes


def _p(n=10, dtype=torch.float32):
    return torch.nn.Parameter(torch.zeros(n, dtype=dtype))


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
@pytest.mark.parametrize("bad", [dict(lr=-1.0), dict(eps=-1e-8), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
                                 dict(weight_decay=-0.1), dict(max_grad_norm=0.0), dict(max_grad_norm=float("nan"))])
def test_constructor_refusals(cls, bad):
    with pytest.raises(ValueError, match="Invalid"):
        cls([_p()], **bad)


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_lr_as_a_tensor_needs_capturable(cls):
    with pytest.raises(ValueError, match="capturable"):
        cls([_p()], lr=torch.tensor(1e-3))
    assert cls([_p()], lr=torch.tensor(1e-3), capturable=True).capturable


def test_constructor_refusals_of_8bit():
    for bad in (dict(block_size=32), dict(block_size=100), dict(min_8bit_numel=-1)):
        with pytest.raises(ValueError, match="Invalid"):
            AdamW8bit([_p()], **bad)
    with pytest.raises(ValueError, match="named"):
        AdamW8bit([_p()], protect_output=True)
    opt = AdamW8bit([("tok_emb.weight", _p(5000)), ("fc.weight", _p(5000)), ("fc.bias", _p(10))], protect_output=True)
    regular, protected = opt.param_groups
    assert [opt._eight_bit(p, regular) for p in regular["params"]] == [True, False]
    assert [opt._eight_bit(p, protected) for p in protected["params"]] == [False]


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_a_parameter_given_twice_is_refused(cls):
    p, q = _p(), _p()
    with pytest.warns(UserWarning), pytest.raises(ValueError, match="more than once"):
        cls([p, p])
    opt = cls([p])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [p]})
    with pytest.warns(UserWarning), pytest.raises(ValueError, match="more than once"):
        opt.add_param_group({"params": [q, q]})
    assert len(opt.param_groups) == 1


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_step_refusals(cls):
    p = _p()
    opt = cls([p])
    opt.step()  # no gradient: nothing to do
    assert not opt.state
    p.grad = torch.zeros(10)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        opt.step()
    q = torch.nn.Parameter(torch.zeros(4, 3))
    q.grad = torch.sparse_coo_tensor(torch.tensor([[0], [1]]), torch.tensor([1.0]), (4, 3))
    with pytest.raises(RuntimeError, match="sparse"):
        cls([q]).step()
    assert opt.step.__self__ is opt and cls([q], lr=0.0).param_groups[0]["lr"] == 0.0
    with pytest.raises(TypeError, match="grad_scale"):
        opt.step(grad_scale=1.0)


def test_gradient_norm_refusals():
    p = _p()
    assert float(grad_norm([p])) == 0.0 and float(clip_grad_norm_([], 1.0)) == 0.0
    p.grad = torch.ones(10)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        grad_norm([p])
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([p], bad)
    p.grad = torch.sparse_coo_tensor(torch.tensor([[0]]), torch.tensor([1.0]), (10,))
    with pytest.raises(RuntimeError, match="sparse"):
        clip_grad_norm_(p, 1.0)


def test_binding_layout():
    lib = _lib.load()
    assert lib.smo_adamw_tensor_struct_size() == _lib.ADAMW_DTYPE.itemsize == 136
    assert _lib.GRAD_DTYPE.itemsize == 24
    assert _host_ext().sizeof_smo_adamw_tensor == 136


def _row(kind, n=16):
    t = np.zeros(1, dtype=_lib.ADAMW_DTYPE)
    t["kind"], t["n"] = kind, n
    for i, k in enumerate(("param", "grad", "exp_avg", "exp_avg_sq", "m_q", "m_s", "v_q", "v_s")):
        t[k] = (i + 1) << 20
    t["q_block"] = 64
    return t


def test_step_descriptors_are_validated_before_any_launch():
    lib = _lib.load()

    def step(t, n=1, max_norm=0.0, ws=None, nbytes=0, scale=None):
        return lib.smo_adamw_step(t.ctypes.data, n, scale, max_norm, None, ws, nbytes, None)

    assert step(_row(1), n=0) == 0
    assert step(_row(1), n=-1) == 1
    assert step(_row(9)) == 1                                            # unknown kind
    for field, value, want in [("param", 0, 1), ("grad", 0, 1), ("exp_avg", 0, 1), ("exp_avg_sq", 0, 1),
                               ("n", -1, 1), ("dtype", 3, 1), ("reserved", 1, 1), ("master", 1 << 22, 1),
                               ("param", 2, 2), ("grad", 1026, 2), ("exp_avg", 1022, 2), ("hp_dev", 2, 2)]:
        t = _row(1)
        t[field] = value
        assert step(t) == want, field
    for field, value, want in [("q_block", 32, 1), ("q_block", 0, 1), ("m_q", 0, 1), ("v_s", 0, 1),
                               ("m_q", (1 << 20) + 8, 2), ("v_q", 4, 2), ("m_s", 2, 2)]:
        t = _row(2)
        t[field] = value
        assert step(t) == want, field
    t = _row(1)
    t["dtype"], t["master"] = _lib.SMO_DTYPE_BF16, (1 << 22) + 2
    assert step(t) == 2                                                  # misaligned master copy
    assert step(_row(1), max_norm=float("nan")) == 1 and step(_row(1), max_norm=-1.0) == 1
    assert step(_row(1), scale=2) == 2
    for name in ("smo_adamw_decode", "smo_adamw_encode"):
        fn = getattr(lib, name)
        assert fn(_row(1).ctypes.data, 1, None) == 1                     # fp32 moments have no codes
        t = _row(2)
        t["exp_avg"] = 0
        assert fn(t.ctypes.data, 1, None) == 1
        t["exp_avg"] = 2
        assert fn(t.ctypes.data, 1, None) == 2
        assert fn(t.ctypes.data, 0, None) == 0


def test_gradient_descriptors_are_validated():
    lib = _lib.load()
    g = np.zeros(1, dtype=_lib.GRAD_DTYPE)
    g["grad"], g["n"] = 1 << 20, 5
    buf = (ctypes.c_uint8 * (1 << 20))()
    ws = (ctypes.addressof(buf) + 255) // 256 * 256
    need = lib.smo_grad_norm_workspace_size(1)
    assert lib.smo_grad_norm_workspace_size(0) == 0 and 0 < need <= lib.smo_grad_norm_workspace_size(5000)

    def norm(g, n=1, max_norm=0.0, out=1 << 21, w=ws, nbytes=need):
        return lib.smo_grad_norm(g.ctypes.data, n, max_norm, out, w, nbytes, None)

    assert norm(g, n=-1) == 1 and norm(g, out=None) == 1 and norm(g, max_norm=float("nan")) == 1
    assert norm(g, out=2) == 2
    assert norm(g, w=None) == 3 and norm(g, nbytes=need - 1) == 3 and norm(g, w=ws + 8) == 3
    for field, value, want in [("grad", 0, 1), ("grad", 2, 2), ("n", -1, 1), ("dtype", 7, 1), ("reserved", 1, 1)]:
        t = g.copy()
        t[field] = value
        assert norm(t) == want, field


def test_host_scalars_agree():
    ext = _host_ext()
    for lr, b1, b2, eps, wd in [(1e-3, 0.9, 0.999, 1e-8, 0.01), (3e-4, 0.95, 0.98, 1e-6, 0.0), (0.0, 0.0, 0.0, 0.0, 0.3),
                                (1, 0.5, 0.75, 1e-12, 1)]:
        for step in (1, 2, 3, 10, 999, 12345, 10 ** 7):
            want = np.array([_host.adamw_scalars(lr, (b1, b2), eps, wd, step)], dtype=_lib.ADAMW_HYPER_DTYPE).tobytes()
            assert ext.adamw_hyper_bytes(lr, b1, b2, eps, wd, step) == want


def test_zero_cost_model():
    assert adamw_step_bytes((100, 100), False) == 28 * 10000
    assert adamw_step_bytes((100, 100), True) == 16 * 10000 + 16 * 79
    assert adamw_step_bytes((10, 10), True) == 28 * 100
    assert adamw_step_bytes((100, 100), False, elem=2, master=True) == 28 * 10000
    assert adamw_step_bytes((100, 100), False, elem=2) == 22 * 10000


@pytest.mark.parametrize("cls", [AdamW, AdamW8bit])
def test_step_hooks_and_schedulers(cls):
    """Hooks of one optimizer and of all, profiler records and a scheduler see every step."""
    p = _p()
    opt = cls([p], lr=0.5)
    seen = []
    handles = [opt.register_step_pre_hook(lambda o, args, kw: seen.append("pre")),
               opt.register_step_post_hook(lambda o, args, kw: seen.append("post")),
               register_optimizer_step_post_hook(lambda o, args, kw: seen.append("all"))]
    opt.step()
    assert seen == ["pre", "post", "all"] or sorted(seen) == ["all", "post", "pre"]
    for h in handles:
        h.remove()
    opt.step()
    assert len(seen) == 3
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        opt.step()
    assert any(f"Optimizer.step#{cls.__name__}.step" in e.key for e in prof.key_averages())
    assert opt.step(lambda: 3.0) == 3.0
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)
    opt.step()
    sched.step()
    assert opt.param_groups[0]["lr"] == 0.25


def test_schedules_are_validated():
    lib = _lib.load()
    t = np.zeros(1, dtype=_lib.SCHEDULE_DTYPE)
    assert _lib.SCHEDULE_DTYPE.itemsize == 56
    advance = lambda n=1, out=1 << 20: lib.smo_adamw_advance(t.ctypes.data, n, out, None)  # noqa: E731
    assert advance(n=0) == 0 and advance(n=-1) == 1 and advance() == 1   # no step count
    t["step"] = 1 << 21
    assert advance(out=None) == 1 and advance(out=2) == 2
    t["step"] = 2
    assert advance() == 2


def test_zero1_refuses_a_norm_of_one_ranks_gradients(monkeypatch):
    from smo_optimizer_b200 import zero

    monkeypatch.setattr(zero.dist, "is_initialized", lambda: True)
    monkeypatch.setattr(zero.dist, "get_world_size", lambda group=None: 2)
    monkeypatch.setattr(zero.dist, "get_rank", lambda group=None: 0)
    with pytest.raises(ValueError, match="max_grad_norm"):
        zero.Zero1([_p(), _p()], AdamW, max_grad_norm=1.0)
    z = zero.Zero1([_p(100), _p(200), _p(90)], AdamW8bit, min_8bit_numel=0, block_size=64)
    assert z.owner == [1, 0, 1] and z.costs[1] == adamw_step_bytes((200,), True, 64, 0)
