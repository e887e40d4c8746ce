"""next_call raises its counter in sight of the graph engine."""
import pytest
import torch

from torchrl_amd import functional as F

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def test_a_backward_pass_behind_next_call_is_refused():
  """dropout on the counter itself, which next_call then raises: the backward pass would make another mask."""
  counter = torch.zeros(1, dtype=torch.int64, device=DEV)
  x = torch.randn(10, device=DEV, requires_grad=True)
  y = F.dropout(x, 0.5, 1, counter)
  F.next_call(counter)
  with pytest.raises(RuntimeError, match='modified by an inplace operation'):
    y.sum().backward()


def test_drawn_call_numbers_stay_good():
  counter = torch.zeros(1, dtype=torch.int64, device=DEV)
  x = torch.randn(100, device=DEV, requires_grad=True)
  calls = [F.next_call(counter) for _ in range(2)]
  ys = [F.dropout(x, 0.5, 1, c) for c in calls]
  F.next_call(counter)
  for i, y in enumerate(ys):
    g, = torch.autograd.grad(y.sum(), [x])
    assert torch.equal(g != 0, F.dropout(torch.ones(100, device=DEV), 0.5, 1, i) != 0)
  with torch.inference_mode():
    inner = torch.zeros(1, dtype=torch.int64, device=DEV)
    assert int(F.next_call(inner)) == 0 and int(F.next_call(counter)) == 3
  assert int(F.next_call(inner)) == 1
