"""Decay attention with time cut into segments: as many as the workgroups join by themselves (up to 8) and one more, which a launch
of its own joins.  The number of segments is read off the workspace, so that a change of the rule shows here."""
import pytest
import torch

from tests import layer_reference as ref
from torchrl_amd import _lib
from torchrl_amd import functional as F

DEV = 'cuda'
LENGTHS = {1: 129, 3: 193, 7: 481, 8: 561, 9: 641}      # steps by the number of segments that they give here
SIZES = [(16, 16), (64, 64), (33, 40), (48, 80), (128, 128), (100, 68), (5, 3)]


def _segments(T, N, H, dk, dv):
  one, both = (_lib.lib().trl_decay_attention_workspace_bytes(T, N, H, dk, dv, b) for b in (0, 1))
  assert both == 2 * one
  return one / (4 * N * H * (dk * dv + 1)) if one else 1


@pytest.mark.parametrize('segs', LENGTHS)
@pytest.mark.parametrize('dk,dv', SIZES)
def test_the_lengths_here_have_the_segments_that_they_stand_for(dk, dv, segs):
  assert _segments(LENGTHS[segs], 3, 2, dk, dv) == segs


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('segs', LENGTHS)
@pytest.mark.parametrize('dk,dv', SIZES)
def test_segments_of_time(dk, dv, segs, dtype):
  """One env whole, one that ends inside the second segment, one that ends with a segment; starts in some segments, so that
  contributions are cut off; both gradients."""
  T, N, H = LENGTHS[segs], 3, 2
  g = torch.Generator().manual_seed(segs * 1000 + dk + dv)
  rn = lambda *s: torch.randn(*s, generator=g)
  a = dict(q=rn(T, N, H, dk).to(dtype), k=rn(T, N, H, dk).to(dtype), v=rn(T, N, H, dv).to(dtype),
           decay=torch.tensor([0.875, 0.998]))
  kw = dict(state=rn(N, H, dk, dv), start=torch.zeros(T, N), lengths=torch.tensor([T, 90, 160 if T >= 160 else 64]),
            gy=rn(T, N, H, dv).to(dtype), gstate=rn(N, H, dk, dv))
  kw['start'][[T // 2, T - 1], 0] = 1.0
  kw['start'][[0, 64], 2] = 1.0
  dev = {n: t.to(DEV) for n, t in (*a.items(), *kw.items())}
  leaves = [dev[n].requires_grad_(True) for n in ('q', 'k', 'v', 'state')]
  out, last = F.decay_attention(dev['q'], dev['k'], dev['v'], dev['decay'], state=dev['state'], start=dev['start'],
                                lengths=dev['lengths'])
  got = dict(zip(('dq', 'dk', 'dv', 'dstate'), torch.autograd.grad([out, last], leaves, [dev['gy'], dev['gstate']])),
             out=out, state=last)
  want = ref.decay_attention(a['q'], a['k'], a['v'], a['decay'], **kw)
  bound = ref.decay_bounds(a['q'], a['k'], a['v'], a['decay'], dtype, **kw)
  for n, t in got.items():
    ref.check(t, want[n], bound[n], n)
