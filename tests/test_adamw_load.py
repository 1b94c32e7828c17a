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
