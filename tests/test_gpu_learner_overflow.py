"""GPU: gated recurrences whose products of neighbouring gates pass float32's range, behind a state or a gradient that is zero."""
import pytest
import torch

from test_gpu_learner_ops import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,N,D", [(8, 2, 5), (40, 3, 8), (300, 2, 7), (3000, 2, 40), (300, 600, 64), (3000, 40, 512)])
@pytest.mark.parametrize("gate", [1e10, -1e30, 3e38])
def test_zero_stays_zero_behind_gates_of_any_size(T, N, D, gate):
    """the window begins at zero and stays there until the last update; backwards the only gradient comes in at the first step.  With zero on the way nothing
    is multiplied that is not zero: h and every gradient are exact."""
    gates = torch.full((T, N, D), gate, device="cuda", requires_grad=True)
    update = torch.zeros((T, N, D), device="cuda")
    update[-1] = 3.0
    update.requires_grad_()
    h, last = ops().gated_recurrence(gates, update)
    assert (h[:-1] == 0).all() and (h[-1] == 3).all() and (last == 3).all()
    d_h = torch.zeros_like(h)
    d_h[0] = 2.0
    d_gate, d_update = torch.autograd.grad([h], [gates, update], [d_h])
    assert (d_update[0] == 2).all() and (d_update[1:] == 0).all() and (d_gate == 0).all()


@pytest.mark.parametrize("T", [40, 3000])
def test_a_cut_behind_such_gates_begins_anew(T):
    """the state is not zero, and what it grows to is not looked at behind the cut, nor does a gradient come through it"""
    gates = torch.full((T, 2, 6), 1e20, device="cuda", requires_grad=True)
    update = torch.ones((T, 2, 6), device="cuda", requires_grad=True)
    state = torch.ones((2, 6), device="cuda", requires_grad=True)
    first = torch.zeros((T, 2), dtype=torch.uint8, device="cuda")
    first[-1] = 1
    h, last = ops().gated_recurrence(gates, update, first, state)
    assert (h[-1] == 1).all() and (last == 1).all()
    d_gate, d_update, d_state = torch.autograd.grad([last], [gates, update, state], [torch.ones_like(last)])
    assert (d_update[-1] == 1).all() and (d_update[:-1] == 0).all() and (d_state == 0).all() and (d_gate[-1] == 0).all()
