"""Zero1 takes any callable that makes an optimizer, as long as it has a name."""

import torch

from smo_optimizer_b200 import zero


def test_a_function_that_makes_the_optimizer():
    def make(params, lr):
        return torch.optim.SGD(params, lr=lr)

    params = [torch.nn.Parameter(torch.ones(8, 8)), torch.nn.Parameter(torch.ones(3))]
    z = zero.Zero1(params, make, lr=0.5)
    # not one of this package's classes: the cost of float moments
    assert z.costs == [zero.step_bytes((8, 8), "make"), zero.step_bytes((3,), "make")]
    for p in params:
        p.grad = torch.ones_like(p)
    z.step()
    assert all(torch.equal(p.detach(), torch.full_like(p, 0.5)) for p in params)
