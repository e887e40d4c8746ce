"""Layer norm, dropout and decay attention have no forward-mode derivatives: an input with a tangent is refused, where a
derivative of zero would be wrong."""
import pytest
import torch
from torch.autograd import forward_ad

from torchrl_amd import _lib
from torchrl_amd import functional as F


def _calls(dev, dual):
  """Every call with one of its inputs dual, by the node's name."""
  x, w, r = torch.randn(6, 8, device=dev), torch.randn(8, device=dev), torch.randn(6, 8, device=dev)
  q, S, lam = torch.randn(3, 2, 1, 8, device=dev), torch.randn(2, 1, 8, 8, device=dev), torch.full((1,), 0.9, device=dev)
  n = _lib.nodes()
  if dev == 'cpu':      # (the nodes themselves: the functions refuse the tensors before)
    norm = lambda x, w, b: n.layer_norm(x, w, b, 1e-5, 0, 0)
    drop = lambda x, r: n.dropout(x, r, 0.5, 1, 2, None, 0)
    attn = lambda q, k, v, S: n.decay_attention(q, k, v, S, lam, None, None, 0, 1.0, 0)
    step = lambda q, k, v, S: n.decay_step(q, k, v, lam, None, 0, S, None, 1.0, 0)
  else:
    norm, drop = F.layer_norm, lambda x, r: F.dropout(x, 0.5, 1, 2, residual=r)
    attn = lambda q, k, v, S: F.decay_attention(q, k, v, lam, state=S)
    step = lambda q, k, v, S: F.decay_attention_step(q, k, v, lam, S)
  for name, fn, args in (('layer_norm', norm, (x, w, w)), ('dropout', drop, (x, r)), ('decay_attention', attn, (q, q, q, S)),
                         ('decay_attention_step', step, (q[0], q[0], q[0], S))):
    for i in range(len(args)):
      yield name, fn, [dual(a) if i == j else a for j, a in enumerate(args)]


def _check(dev):
  for grad in (True, False):
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
      for name, fn, args in _calls(dev, lambda t: forward_ad.make_dual(t, torch.ones_like(t))):
        with pytest.raises(RuntimeError, match=name + ' has no forward-mode derivative'):
          fn(*args)


def test_nodes_refuse_tangents():
  _check('cpu')


@pytest.mark.gpu
def test_functions_refuse_tangents():
  _check('cuda')
  x = torch.randn(6, 8, device='cuda')
  with forward_ad.dual_level():      # (a tangent elsewhere is no matter)
    forward_ad.make_dual(torch.randn(3, device='cuda'), torch.ones(3, device='cuda'))
    assert torch.equal(F.layer_norm(x), F.layer_norm(x.clone()))


@pytest.mark.gpu
def test_the_module_refuses_tangents():
  from torchrl_amd.contrib.models import LayerNorm
  m = LayerNorm(8).cuda()
  x = torch.randn(6, 8, device='cuda')
  for p in m.parameters():
    p.requires_grad_(False)
  with forward_ad.dual_level(), pytest.raises(RuntimeError, match='forward-mode'):
    m(forward_ad.make_dual(x, torch.ones_like(x)))
