"""State dicts that AdamW and AdamW8bit load or refuse, on the CPU."""

import copy

import pytest
import torch

from smo_optimizer_b200 import AdamW, AdamW8bit

BOTH = pytest.mark.parametrize("cls", [AdamW, AdamW8bit])


def _p(n=10, dtype=torch.float32):
    return torch.nn.Parameter(torch.zeros(n, dtype=dtype))


def _saved(cls=torch.optim.AdamW, n=10, **options):
    """The state dict of a torch optimizer after one step."""
    p = _p(n)
    p.grad = torch.linspace(-1, 1, n)
    opt = cls([p], lr=1e-2, **options)
    opt.step()
    return opt.state_dict()


@BOTH
@pytest.mark.parametrize("options", [dict(maximize=True), dict(amsgrad=True), dict(maximize=True, amsgrad=True)], ids=str)
def test_options_that_change_the_step_are_refused(cls, options):
    p, q = _p(), _p()
    opt = cls([{"params": [p]}, {"params": [q], "lr": 0.5}], lr=0.25)
    before = copy.deepcopy(opt.state_dict())
    saved = _saved(**options)
    two = copy.deepcopy(saved)
    two["param_groups"].insert(0, dict(_saved()["param_groups"][0], params=[1]))
    for sd, o in ((two, opt), (saved, cls([p]))):
        with pytest.raises(ValueError, match="|".join(options)):
            o.load_state_dict(sd)
        assert not o.state
    assert opt.state_dict() == before
    with pytest.raises(ValueError, match="|".join(options)):
        cls([dict(params=[p], **options)])
    with pytest.raises(ValueError, match="|".join(options)):
        opt.add_param_group(dict(params=[_p()], **options))
    assert len(opt.param_groups) == 2


@BOTH
def test_decay_through_the_gradient_is_refused(cls):
    opt = cls([_p()])
    with pytest.raises(ValueError, match="decoupled_weight_decay"):
        opt.load_state_dict(_saved(torch.optim.Adam, weight_decay=0.1))
    with pytest.raises(ValueError, match="decoupled_weight_decay"):
        cls([dict(params=[_p()], decoupled_weight_decay=False)])  # the default decay
    with pytest.raises(TypeError):
        opt.add_param_group([_p()])
    assert not opt.state and len(opt.param_groups) == 1
    opt.load_state_dict(_saved(torch.optim.Adam))  # no decay at all: the same step
    assert len(opt.state) == 1 and opt.param_groups[0]["weight_decay"] == 0


@BOTH
def test_options_that_leave_the_step_as_it_is(cls):
    opt = cls([_p()])
    opt.load_state_dict(_saved(maximize=False, amsgrad=False, foreach=False))
    group = opt.param_groups[0]
    assert group["lr"] == 1e-2 and not group["maximize"] and not group["amsgrad"]
    assert set(opt.state[group["params"][0]]) == {"step", "exp_avg", "exp_avg_sq"}


def _coded(n, block):
    nb = -(-n // block)
    r = torch.Generator().manual_seed(n)
    return {"step": 3, "m_q": torch.randint(-127, 128, (nb, block), generator=r).to(torch.int8),
            "v_q": torch.randint(0, 256, (nb, block), generator=r).to(torch.uint8),
            "m_s": torch.rand((nb, 1), generator=r), "v_s": torch.rand((nb, 1), generator=r)}


def _floats(n, seed=0):
    r = torch.Generator().manual_seed(seed)
    return {"step": 2, "exp_avg": torch.randn(n, generator=r), "exp_avg_sq": torch.rand(n, generator=r)}


def _loaded(cls, dtype=torch.bfloat16):
    """An optimizer over three bf16 parameters with a loaded state each."""
    sizes = [30, 5000, 257]
    opt = cls([{"params": [_p(n, dtype) for n in sizes[:2]]}, {"params": [_p(sizes[2], dtype)], "lr": 0.5}], lr=0.25)
    sd = opt.state_dict()
    sd["state"] = {i: _floats(n, i) for i, n in enumerate(sizes)}
    if cls is AdamW8bit:
        sd["state"][1] = _coded(5000, 128)
    opt.load_state_dict(sd)
    return opt, copy.deepcopy(opt.state_dict())


def _same_state(a, b):
    assert a["param_groups"] == b["param_groups"] and a["state"].keys() == b["state"].keys()
    for i in a["state"]:
        assert a["state"][i].keys() == b["state"][i].keys()
        for k, t in a["state"][i].items():
            u = b["state"][i][k]
            assert (t.dtype == u.dtype and torch.equal(t, u)) if torch.is_tensor(t) else t == u, (i, k)


@BOTH
@pytest.mark.parametrize("spoil", [
    lambda sd: sd["state"][2].update(exp_avg=torch.zeros(256)), lambda sd: sd["state"][2].pop("exp_avg_sq"),
    lambda sd: sd["state"][0].update(step="many"), lambda sd: sd["state"][2].update(master=torch.zeros(1, 257)),
    lambda sd: sd["state"].update({1: dict(_coded(5000, 128), m_q=torch.zeros((39, 128), dtype=torch.int8))}),
    lambda sd: sd["param_groups"].pop(), lambda sd: sd["param_groups"][0]["params"].pop(),
    lambda sd: sd["param_groups"][1].update(maximize=True)])
def test_a_refused_load_changes_nothing(cls, spoil):
    opt, before = _loaded(cls)
    opt.master_weights = True
    held = [dict(opt.state[p]) for g in opt.param_groups for p in g["params"]]
    sd = copy.deepcopy(before)
    for g in sd["param_groups"]:
        g["lr"] = 7.0
    spoil(sd)
    with pytest.raises(ValueError):
        opt.load_state_dict(sd)
    _same_state(opt.state_dict(), before)
    now = [opt.state[p] for g in opt.param_groups for p in g["params"]]
    assert all(a[k] is b[k] for a, b in zip(now, held) for k in b)
    opt.load_state_dict(before)
    _same_state(opt.state_dict(), before)


@BOTH
def test_load_hooks_see_and_shape_what_is_loaded(cls):
    opt, before = _loaded(cls)
    seen = []

    def halve(o, sd):
        sd = copy.deepcopy(sd)
        sd["state"][0]["exp_avg"] *= 0.5
        sd["state"]["note"] = "kept"
        return sd

    opt.register_load_state_dict_pre_hook(halve)
    opt.register_load_state_dict_post_hook(lambda o: seen.append({k: v for k, v in o.state[o.param_groups[0]["params"][0]].items()}))
    opt.load_state_dict(before)
    p = opt.param_groups[0]["params"][0]
    assert opt.state[p]["exp_avg"].dtype == torch.float32
    assert torch.equal(opt.state[p]["exp_avg"], before["state"][0]["exp_avg"] * 0.5)
    assert seen[0]["exp_avg"] is opt.state[p]["exp_avg"] and opt.state["note"] == "kept"
    shared = before["state"][0]["exp_avg_sq"].data_ptr()
    assert opt.state[p]["exp_avg_sq"].data_ptr() != shared


@BOTH
def test_groups_without_an_option_take_the_optimizers(cls):
    opt, before = _loaded(cls)
    sd = copy.deepcopy(before)
    for key in ("eps", "block_size"):
        sd["param_groups"][0].pop(key, None)
    opt.load_state_dict(sd)
    _same_state(opt.state_dict(), before)


@BOTH
def test_capturable_loads_write_to_the_states_that_graphs_hold(cls):
    """A captured step holds the addresses of its states, step counts and learning rate: a load keeps them."""
    sizes = [30, 5000]
    opt = cls([_p(n, torch.bfloat16) for n in sizes], lr=torch.tensor(0.25), capturable=True, master_weights=True)
    sd = opt.state_dict()
    sd["state"] = {i: dict(_floats(n, i), master=torch.ones(n)) for i, n in enumerate(sizes)}
    if cls is AdamW8bit:
        sd["state"][1] = dict(_coded(5000, 128), master=torch.ones(5000))
    opt.load_state_dict(sd)
    params = opt.param_groups[0]["params"]
    held = [dict(opt.state[p]) for p in params]
    lr = opt.param_groups[0]["lr"]
    address = [{k: t.data_ptr() for k, t in st.items()} for st in held]
    opt._captured = True
    other = copy.deepcopy(opt.state_dict())
    for st in other["state"].values():
        for t in st.values():
            t.copy_(t.flip(0) if t.dim() else t + 5)
    other["param_groups"][0]["lr"] = torch.tensor(0.125)
    opt.load_state_dict(copy.deepcopy(other))
    for i, (p, st, at) in enumerate(zip(params, held, address)):
        assert opt.state[p].keys() == st.keys()
        for k, t in st.items():
            assert opt.state[p][k] is t and t.data_ptr() == at[k] and torch.equal(t, other["state"][i][k]), (i, k)
    assert opt.param_groups[0]["lr"] is lr and float(lr) == 0.125
    # a state that cannot stay where it is: the old one stays alive for the graphs
    gone = opt.state[params[0]]["exp_avg"]
    changed = copy.deepcopy(other)
    del changed["state"][0]["master"]
    opt.load_state_dict(changed)
    assert "master" not in opt.state[params[0]] and opt.state[params[0]]["exp_avg"] is not gone
    assert any(isinstance(kept, dict) and kept.get("exp_avg") is gone for kept in opt._kept)
    gone = opt.state[params[1]]
    del changed["state"][1]
    opt.load_state_dict(changed)
    assert not opt.state[params[1]] and any(kept is gone for kept in opt._kept)
    # nothing captured: a state dict taken before keeps its tensors
    plain = cls([_p(30)], capturable=True)
    plain.load_state_dict({"state": {0: _floats(30)}, "param_groups": plain.state_dict()["param_groups"]})
    before = plain.state_dict()
    plain.load_state_dict({"state": {0: _floats(30, 1)}, "param_groups": before["param_groups"]})
    assert torch.equal(before["state"][0]["exp_avg"], _floats(30)["exp_avg"]) and not plain._kept


@BOTH
def test_a_learning_rate_that_groups_share(cls):
    lr = torch.tensor(0.5)
    opt = cls([{"params": [_p(3)]}, {"params": [_p(4)]}, {"params": [_p(5)], "lr": 0.25}], lr=lr, capturable=True)
    opt._captured = True
    sd = copy.deepcopy(opt.state_dict())
    for g in sd["param_groups"][:2]:
        g["lr"] = torch.tensor(0.125)
    opt.load_state_dict(sd)
    assert [g["lr"] is lr for g in opt.param_groups] == [True, True, False] and float(lr) == 0.125
    assert opt.param_groups[2]["lr"] == 0.25
    sd["param_groups"][1]["lr"] = torch.tensor(2.0)
    opt.load_state_dict(sd)
    assert [float(g["lr"]) for g in opt.param_groups] == [0.125, 2.0, 0.25]
    assert any(kept is lr for kept in opt._kept)


@BOTH
def test_a_load_keeps_the_norm_that_graphs_write(cls):
    opt = cls([_p(3)], capturable=True, max_grad_norm=1.0)
    norm, scalars = torch.zeros(()), torch.zeros(1, 8)
    opt._workspace[0], opt._scalars[0], opt.last_grad_norm = (torch.zeros(8), norm), scalars, norm
    opt._captured = True
    opt.load_state_dict(opt.state_dict())
    assert opt.last_grad_norm is norm and opt._workspace[0][1] is norm and opt._scalars[0] is scalars
    opt._captured = False
    opt.load_state_dict(opt.state_dict())
    assert opt.last_grad_norm is None and not opt._workspace and any(kept is scalars for kept in opt._kept)
