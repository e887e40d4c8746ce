"""Dropout in a forward pass that is run again inside the backward pass: refused where the mask would be another one."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from torchrl_amd import functional as F


def test_no_call_number_is_drawn_inside_a_backward_pass():
  counter = torch.zeros(1, dtype=torch.int64)
  x = torch.randn(3, requires_grad=True)
  x.register_hook(lambda g: F.next_call(counter))
  with pytest.raises(RuntimeError, match='activation checkpointing'):
    x.sum().backward()
  with pytest.raises(RuntimeError, match='HIP device'):      # (outside: as ever)
    F.next_call(counter)


@pytest.mark.gpu
@pytest.mark.parametrize('reentrant', [False, True])
def test_dropout_layers_under_checkpointing(reentrant):
  from torchrl_amd.contrib.models import Dropout
  m = Dropout(0.5, seed=3).cuda()
  x = torch.randn(200, 16, device='cuda', requires_grad=True)
  y = checkpoint(lambda t: m(t * 1.5).square(), x, use_reentrant=reentrant)
  with pytest.raises(RuntimeError, match='activation checkpointing'):
    y.sum().backward()
  assert int(m.calls) == 1
  m.eval()      # (draws nothing)
  checkpoint(lambda t: m(t).square(), x, use_reentrant=reentrant).sum().backward()
  assert torch.equal(x.grad, 2 * x)


@pytest.mark.gpu
@pytest.mark.parametrize('reentrant', [False, True])
def test_a_call_number_from_outside_under_checkpointing(reentrant):
  counter = torch.zeros(1, dtype=torch.int64, device='cuda')
  x = torch.randn(200, 16, device='cuda', requires_grad=True)
  call = F.next_call(counter)
  fn = lambda t: F.dropout(t * 1.5, 0.5, 3, call).square()
  a, = torch.autograd.grad(fn(x).sum(), [x])
  checkpoint(fn, x, use_reentrant=reentrant).sum().backward()
  assert torch.equal(x.grad, a)
