"""Compact-scene operators on the MI355X: calls at the edges of autograd, of their arguments and of the launch rules
(tests/test_gpu_compact.py has the values)."""
import pytest
import torch

from test_gpu_compact import DEV, both_routes, gen, model, scene

pytestmark = pytest.mark.gpu


def test_evict_of_groups_that_can_be_read_once():
    """Groups from an iterator (zip(begins, ends)): the same Gaussians as from a list."""
    a, b = model(), model()
    budgets = [500, 900]
    want, ranges = a.evict(budgets, recent=[100, 0], groups=[(0, 1000), (1000, 3000)])
    got, again = b.evict(budgets, recent=[100, 0], groups=zip([0, 1000], [1000, 3000]))
    assert again == ranges == [(0, 500), (500, 1400)] and b.num_points == 1400
    assert torch.equal(got, want) and torch.equal(a._arena.data, b._arena.data)
    c, d = model(), model()
    want, ranges = c.evict(700, groups=[(0, 1000), (1000, 3000)])
    got, again = d.evict(700, groups=iter([(0, 1000), (1000, 3000)]))  # one budget for all of them
    assert again == ranges and d.num_points == 1400 and torch.equal(got, want)


def test_evict_with_weights_of_another_number():
    m = model()
    m.contribution = torch.zeros(2999, 1, device=DEV)
    with pytest.raises(RuntimeError, match="contribution must hold 3000"):
        m.evict(100)
    assert m.num_points == 3000
