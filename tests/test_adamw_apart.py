"""Parameters that share memory would be written by two threads at once: AdamW and AdamW8bit refuse them."""

import pytest
import torch

from smo_optimizer_b200 import adamw


def _items(*tensors):
    return [(torch.nn.Parameter(t), None, None, None) for t in tensors]


def test_neighbours_and_views_that_interleave_are_apart():
    flat = torch.zeros(100)
    grid = torch.zeros(10, 10)
    adamw._check_apart("AdamW", _items(flat[:60], flat[60:], flat[:0], flat[50:50], torch.zeros(()), grid[:, :5], grid[:, 5:]))
    adamw._check_apart("AdamW", _items(grid.t(), flat.view(4, 25)[::2], flat.view(4, 25)[1::2]))


@pytest.mark.parametrize("views", [lambda f: (f, f), lambda f: (f[:60], f[59:]), lambda f: (f, f[40:50]),
                                   lambda f: (f.view(10, 10), torch.zeros(5), f[99:]), lambda f: (f[:50], f.half()[:0], f[49:50])])
def test_shared_elements_are_refused(views):
    made = views(torch.zeros(100))
    for order in (made, made[::-1]):
        with pytest.raises(ValueError, match="share memory"):
            adamw._check_apart("AdamW", _items(*order))


@pytest.mark.parametrize("p", [torch.zeros(1, 5).expand(4, 5), torch.zeros(()).expand(3), torch.zeros(20).as_strided((4, 4), (2, 1))])
def test_parameters_that_repeat_elements_are_refused(p):
    with pytest.raises(ValueError, match="share memory"):
        adamw._check_apart("AdamW", _items(torch.zeros(3), p))
