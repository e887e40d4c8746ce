"""Decay attention multiplies what it computes (the state, the pair products, the weighed steps) with all 24 bits of a float32,
whatever the inputs' type: cases whose leading bits cancel, so that the result is the bits a shorter operand would not have.

Every product and sum in them is exact in float32, in any order, so the results are equal and not merely close."""
import pytest
import torch

from tests import layer_reference as ref
from torchrl_amd import functional as F

DEV = 'cuda'
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LONG, SHORT, LAST = 1 + 2.0 ** -9 + 2.0 ** -22, 1 + 2.0 ** -9, 2.0 ** -22      # LONG - SHORT = LAST
LAM = 0.5 + 2.0 ** -10 + 2.0 ** -24
SIZES = [(2, 2), (20, 33), (48, 80), (64, 64), (128, 128)]


def _bf16_parts(x, n):
  """The sum of the first n bf16 parts of a float32."""
  left, total = torch.tensor(x, dtype=torch.float32), 0.0
  for _ in range(n):
    part = left.bfloat16().float()
    total, left = total + float(part), left - part
  return total


def test_the_values_here_have_bits_that_two_bf16_parts_do_not_hold():
  for x in (LONG, LAM):
    assert _bf16_parts(x, 3) == x == float(torch.tensor(x, dtype=torch.float32))
    assert abs(_bf16_parts(x, 2) - x) >= 2.0 ** -24
  assert _bf16_parts(SHORT, 2) == SHORT
  for t in DTYPES:      # inputs and results that the types hold
    assert all(float(torch.tensor(x).to(t)) == x for x in (1.0, -1.0, 2.0 ** -9, LAST, 2 * LAST, 3 * LAST))


def _call(q, k, v, lam, dtype, **kw):
  H = q.shape[2]
  c = lambda t: None if t is None else t.to(DEV)
  return F.decay_attention(c(q.to(dtype)), c(k.to(dtype)), c(v.to(dtype)), torch.full((H,), lam, device=DEV), scale=1.0,
                           **{n: c(t) for n, t in kw.items()})


def _pick(*shape):
  """1 in the first place of the last dimension, -1 in the last."""
  t = torch.zeros(*shape)
  t[..., 0], t[..., -1] = 1.0, -1.0
  return t


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dk,dv', SIZES)
def test_the_state_in_the_output_and_in_dq(dk, dv, dtype):
  T, N, H = 40, 3, 2
  zk, zv = torch.zeros(T, N, H, dk), torch.zeros(T, N, H, dv)
  S = torch.full((N, H, dk, dv), SHORT)
  S[:, :, 0] = LONG
  out, last = _call(_pick(T, N, H, dk), zk, zv, 1.0, dtype, state=S)
  assert torch.equal(out.float().cpu(), torch.full_like(zv, LAST)) and torch.equal(last.cpu(), S)
  S = torch.full((N, H, dk, dv), SHORT)
  S[..., 0] = LONG
  q = torch.zeros(T, N, H, dk, dtype=dtype, device=DEV, requires_grad=True)
  out, _ = F.decay_attention(q, zk.to(dtype).to(DEV), zv.to(dtype).to(DEV), torch.ones(H, device=DEV), scale=1.0, state=S.to(DEV))
  dq, = torch.autograd.grad(out, [q], _pick(T, N, H, dv).to(dtype).to(DEV))
  assert torch.equal(dq.float().cpu(), torch.full_like(zk, LAST))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dk,dv', SIZES)
def test_the_gradient_of_the_state_in_dk_and_dv(dk, dv, dtype):
  T, N, H = 40, 3, 2
  zq = torch.zeros(T, N, H, dk, dtype=dtype, device=DEV)
  k = _pick(T, N, H, dk).to(dtype).to(DEV).requires_grad_(True)
  v = _pick(T, N, H, dv).to(dtype).to(DEV).requires_grad_(True)
  _, last = F.decay_attention(zq, k, v, torch.ones(H, device=DEV), scale=1.0)
  R = torch.full((N, H, dk, dv), SHORT)
  R[..., 0] = LONG
  dk_, = torch.autograd.grad(last, [k], R.to(DEV), retain_graph=True)
  assert torch.equal(dk_.float().cpu(), torch.full((T, N, H, dk), LAST))
  R = torch.full((N, H, dk, dv), SHORT)
  R[:, :, 0] = LONG
  dv_, = torch.autograd.grad(last, [v], R.to(DEV))
  assert torch.equal(dv_.float().cpu(), torch.full((T, N, H, dv), LAST))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dk,dv', [(3, 1), (20, 33), (48, 80), (64, 64), (128, 128)])
@pytest.mark.parametrize('starts', [False, True])
def test_the_pair_products(dk, dv, dtype, starts):
  """Two steps a chunk, v = 1 and -1, whose products with q are LONG and SHORT: every step sees LAST per pair before it."""
  T, N, H = 48, 2, 2
  q, k, v = torch.ones(T, N, H, dk), torch.zeros(T, N, H, dk), torch.zeros(T, N, H, dv)
  want = torch.zeros(T, N, H, dv)
  start = torch.zeros(T, N)
  for i, t in enumerate((3, 20, 37)):
    k[t:t + 2, ..., 0], k[t:t + 2, ..., 1], k[t, ..., 2] = 1.0, 2.0 ** -9, LAST
    v[t], v[t + 1] = 1.0, -1.0
    q[t] = 0.0
    want[t + 1:] = LAST * (1 if starts else i + 1)
    want[t] = 0.0
    if starts:
      start[t] = 1.0
  out, last = _call(q, k, v, 1.0, dtype, start=start)
  assert torch.equal(out.float().cpu(), want)
  S = torch.zeros(N, H, dk, dv)
  S[:, :, 2] = LAST * (1 if starts else 3)
  assert torch.equal(last.cpu(), S)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dk,dv', [(1, 1), (20, 33), (48, 80), (64, 64), (128, 128)])
@pytest.mark.parametrize('T', [2, 16, 32, 39])
def test_the_weighed_steps_in_the_state(dk, dv, T, dtype):
  N, H = 2, 2
  k, v = torch.zeros(T, N, H, dk), torch.zeros(T, N, H, dv)
  k[T - 2:], v[T - 2], v[T - 1] = 1.0, 1.0, -0.5
  _, last = _call(k, k, v, LAM, dtype)
  assert torch.equal(last.cpu(), torch.full((N, H, dk, dv), LAM - 0.5))
  # backward in time: lambda (q do - 1) with q do = 1
  S = torch.zeros(N, H, dk, dv, device=DEV, requires_grad=True)
  one = lambda d: torch.ones(1, N, H, d, dtype=dtype, device=DEV)
  out, last = F.decay_attention(one(dk), 0 * one(dk), 0 * one(dv), torch.full((H,), LAM, device=DEV), scale=1.0, state=S)
  ds, = torch.autograd.grad([out, last], [S], [one(dv), torch.full_like(last, -1.0)])
  assert not ds.any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_sixteen_bit_results_are_the_64_bit_ones_rounded(dtype):
  """All but the few whose exact value is next to a border between two values of the type.  A sum whose error has the size e
  crosses a border in a share e / step of the cases; e is 2^-23 of the results' size in float32 (some hundred roundings
  of 2^-25 each, added like random ones), and four times that is allowed."""
  g = torch.Generator().manual_seed(11)
  T, N, H, D = 1024, 1, 4, 64
  rn = lambda *s: torch.randn(*s, generator=g).to(dtype)
  a = dict(q=rn(T, N, H, D), k=rn(T, N, H, D), v=rn(T, N, H, D))
  decay = 1.0 - torch.exp2(-3.0 - torch.arange(H).float())
  gy = rn(T, N, H, D)
  want = ref.decay_attention(a['q'], a['k'], a['v'], decay, gy=gy)
  dev = {n: t.to(DEV).requires_grad_(True) for n, t in a.items()}
  out, _ = F.decay_attention(dev['q'], dev['k'], dev['v'], decay.to(DEV))
  got = dict(zip(('dq', 'dk', 'dv'), torch.autograd.grad(out, list(dev.values()), gy.to(DEV))), out=out.detach())
  if dtype == torch.float32:      # (itself the size of the errors)
    for n, t in got.items():
      w = want[n]
      assert float((t.cpu().double() - w).norm() / w.norm()) <= 2.0 ** -21, n
    return
  for n, t in got.items():
    w = want[n]
    step = torch.exp2(torch.floor(torch.log2(w.abs()))) * torch.finfo(dtype).eps
    share = float((t.cpu() != w.to(dtype)).double().mean())
    assert share <= float((2.0 ** -21 * w.square().mean().sqrt() / step).clamp_max(1.0).mean()), (n, share)
