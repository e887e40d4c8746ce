"""An infinite state (or gradient of one) in decay attention: infinite where the recurrence keeps it so, and of its sign."""
import pytest
import torch

from tests import layer_reference as ref
from torchrl_amd import functional as F

pytestmark = pytest.mark.gpu
DEV = 'cuda'
INF = float('inf')


def _kinds(t):
  """0 finite, 1 and 2 the infinities, 3 NaN."""
  t = t.detach().double().cpu()
  return torch.where(t.isnan(), 3, torch.where(t == INF, 1, torch.where(t == -INF, 2, 0)))


def _inputs(T, N, D, dtype, decay, state, gstate):
  g = torch.Generator().manual_seed(T + D)
  H = len(decay)
  rn = lambda *s: torch.randn(*s, generator=g)
  a = dict(q=rn(T, N, H, D).to(dtype), k=rn(T, N, H, D).to(dtype), v=rn(T, N, H, D).to(dtype), decay=torch.tensor(decay),
           state=rn(N, H, D, D), gy=rn(T, N, H, D).to(dtype), gstate=rn(N, H, D, D))
  for n, on in (('state', state), ('gstate', gstate)):
    if on:
      a[n][0, :, 2, 5], a[n][-1, :, 3, 1] = INF, -INF
  return a


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('which', ['state', 'gstate'])
@pytest.mark.parametrize('T,D', [(1, 16), (5, 20), (16, 64), (40, 24), (100, 128), (700, 16), (4100, 16)])
def test_infinite_states_stay_infinite(T, D, which, dtype):
  """Powers of the decay that are exact, rounded up and rounded down, and below the smallest float; one chunk, many, and time in
  segments."""
  decay = [1.0, 0.5, 0.875, 0.9, 0.97, 1.0 - 2.0 ** -10, 1e-3, 1e-30]
  a = _inputs(T, 2, D, dtype, decay, which == 'state', which == 'gstate')
  want = ref.decay_attention(a['q'], a['k'], a['v'], a['decay'], state=a['state'], gy=a['gy'], gstate=a['gstate'])
  dev = {n: t.to(DEV) for n, t in a.items()}
  leaves = [dev[n].requires_grad_(True) for n in ('q', 'k', 'v', 'state')]
  out, last = F.decay_attention(dev['q'], dev['k'], dev['v'], dev['decay'], state=dev['state'])
  got = dict(zip(('dq', 'dk', 'dv', 'dstate'), torch.autograd.grad([out, last], leaves, [dev['gy'], dev['gstate']])),
             out=out, state=last)
  for n, t in got.items():
    kinds, expected = _kinds(t), _kinds(want[n])
    if dtype == torch.bfloat16 and n not in ('state', 'dstate'):      # (a product with it is a NaN there)
      kinds, expected = kinds > 0, expected > 0
    assert torch.equal(kinds, expected), n
  assert (_kinds(got['state' if which == 'state' else 'dstate']) == 1).any()


def test_infinite_states_end_at_a_start_and_agree_with_the_step():
  decay = [1.0, 0.5, 0.9, 0.97]
  a = _inputs(40, 2, 16, torch.float32, decay, True, False)
  a['start'] = torch.zeros(40, 2)
  a['start'][21, 0] = 1.0
  want = ref.decay_attention(a['q'], a['k'], a['v'], a['decay'], state=a['state'], start=a['start'])
  dev = {n: t.to(DEV) for n, t in a.items()}
  out, last = F.decay_attention(dev['q'], dev['k'], dev['v'], dev['decay'], state=dev['state'], start=dev['start'])
  st, outs = dev['state'], []
  for t in range(40):
    o, st = F.decay_attention_step(dev['q'][t], dev['k'][t], dev['v'][t], dev['decay'], st, start=dev['start'][t])
    outs.append(o)
  for got in ((out, last), (torch.stack(outs), st)):
    assert torch.equal(_kinds(got[0]), _kinds(want['out'])) and torch.equal(_kinds(got[1]), _kinds(want['state']))
