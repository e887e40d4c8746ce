"""Layer norm and dropout on the device against plain 64-bit implementations (tests/layer_reference.py has the bounds)."""
import copy

import numpy as np
import pytest
import torch
from torch import nn

from tests import layer_reference as ref
from torchrl_amd import functional as F

pytestmark = pytest.mark.gpu
DEV = 'cuda'
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(seed):
  return torch.Generator().manual_seed(seed)


def _rows(rows, width, dtype, seed, mean=0.5):
  g = _gen(seed)
  x = torch.randn(rows, width, generator=g) * (0.5 + torch.rand(rows, 1, generator=g)) + mean * torch.randn(rows, 1, generator=g)
  return x.to(dtype).to(DEV)


def _norm_case(rows, width, dtype, relu, weight=True, bias=True, seed=0, mean=0.5):
  g = _gen(1000 + seed)
  x = _rows(rows, width, dtype, seed, mean).requires_grad_(True)
  w = (1 + 0.2 * torch.randn(width, generator=g)).to(DEV).requires_grad_(True) if weight else None
  b = (0.2 * torch.randn(width, generator=g)).to(DEV).requires_grad_(True) if bias else None
  gy = torch.randn(rows, width, generator=g).to(dtype).to(DEV)
  y = F.layer_norm(x, w, b, relu=relu)
  (ry, rx, rw, rb), (by, bx, bw, bb), nearest = ref.layer_norm(x, w, b, 1e-5, relu, gy)
  ref.check(y, ry, by, 'y')
  if relu and float(nearest) < float((by + 1e-7).max()):
    # a value that close to the border may lie on either side of it: it gets no gradient (those clipped further off do)
    z = _pre(x, w, b)
    gy = torch.where(z.abs().to(DEV) <= 4 * float(by.max()), torch.zeros_like(gy), gy)
    (_, rx, rw, rb), (_, bx, bw, bb), _ = ref.layer_norm(x, w, b, 1e-5, relu, gy)
  leaves = [t for t in (x, w, b) if t is not None]
  grads = dict(zip([n for n, t in (('x', x), ('w', w), ('b', b)) if t is not None], torch.autograd.grad(y, leaves, gy)))
  ref.check(grads['x'], rx, bx, 'dx')
  if weight:
    assert grads['w'].dtype == torch.float32
    ref.check(grads['w'], rw, bw, 'dw')
  if bias:
    ref.check(grads['b'], rb, bb, 'db')


def _pre(x, w, b):
  return ref.layer_norm(x, w, b, 1e-5, False)[0]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('width', [1, 2, 3, 4, 5, 7, 8, 9, 31, 33, 64, 65, 100, 128, 129, 255, 257, 511, 513])
def test_layer_norm_widths(width, dtype):
  _norm_case(37, width, dtype, relu=False, seed=width)


@pytest.mark.parametrize('dtype,width', [(torch.float32, 1000), (torch.float32, 1025), (torch.float32, 2049),
                                         (torch.float32, 4099), (torch.float32, 8192), (torch.float32, 8193),
                                         (torch.bfloat16, 1027), (torch.bfloat16, 2050), (torch.bfloat16, 4097),
                                         (torch.bfloat16, 8200), (torch.bfloat16, 16384), (torch.bfloat16, 16387),
                                         (torch.float16, 20001)])
def test_layer_norm_wide_rows(width, dtype):
  _norm_case(5, width, dtype, relu=False, seed=width)


@pytest.mark.parametrize('rows', [1, 2, 15, 16, 17, 255, 1000, 20011])
@pytest.mark.parametrize('width', [12, 64, 200])
def test_layer_norm_row_counts(rows, width):
  _norm_case(rows, width, torch.float32, relu=False, seed=rows)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,width', [(3, 1), (50, 64), (33, 129), (9, 700), (4, 8195)])
def test_layer_norm_relu(rows, width, dtype):
  _norm_case(rows, width, dtype, relu=True, seed=rows + width)


@pytest.mark.parametrize('weight,bias', [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize('relu', [False, True])
def test_layer_norm_without_parameters(weight, bias, relu):
  _norm_case(29, 77, torch.float32, relu, weight, bias, seed=5)
  _norm_case(3, 9001, torch.float32, relu, weight, bias, seed=6)


def test_layer_norm_rows_far_from_zero():
  """The second moment is taken about the mean: rows of mean 1,000 and spread 1 keep their digits."""
  g = _gen(3)
  x = (1000.0 + torch.randn(64, 256, generator=g)).to(DEV)
  y = F.layer_norm(x)
  want, bound = ref.layer_norm(x, None, None, 1e-5, False)
  ref.check(y, want, bound, 'y')
  assert float((y.double().cpu() - want).abs().max()) < 5e-4


def test_layer_norm_views_and_strides():
  g = _gen(4)
  base = torch.randn(40, 3, 66, generator=g).to(DEV)
  w, b = torch.randn(66, generator=g).to(DEV), torch.randn(66, generator=g).to(DEV)
  dense = F.layer_norm(base, w, b)
  # a transposed view, a slice that starts off the 16 B grid, an expanded input
  assert torch.equal(F.layer_norm(base.transpose(0, 1), w, b), dense.transpose(0, 1))
  flat = torch.empty(40 * 3 * 66 + 1, device=DEV)
  off = flat[1:].view(40, 3, 66).copy_(base)
  assert off.data_ptr() % 16 == 4 and torch.equal(F.layer_norm(off, w, b), dense)
  one = base[:1].clone().requires_grad_(True)
  y = F.layer_norm(one.expand(7, 3, 66), w, b)
  assert torch.equal(y, dense[:1].expand(7, 3, 66))
  gx, = torch.autograd.grad(y.sum(), [one])      # (an expanded gradient: stride 0)
  x2 = base[:1].clone().requires_grad_(True)
  g2, = torch.autograd.grad(F.layer_norm(x2, w, b), [x2], torch.ones(1, 3, 66, device=DEV))
  torch.testing.assert_close(gx, 7 * g2, rtol=1e-6, atol=1e-6)
  half = flat.to(torch.bfloat16)[1:1 + 66].view(1, 66)      # rows on a 2 B boundary
  ref.check(F.layer_norm(half, w, b), *ref.layer_norm(half, w, b, 1e-5, False), 'y')


def test_layer_norm_empty_and_partial_gradients():
  w = torch.ones(8, device=DEV, requires_grad=True)
  b = torch.zeros(8, device=DEV, requires_grad=True)
  x = torch.empty(0, 8, device=DEV, requires_grad=True)
  y = F.layer_norm(x, w, b)
  gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.empty(0, 8, device=DEV))
  assert y.shape == (0, 8) and gx.shape == (0, 8) and not gw.any() and not gb.any()
  x = _rows(19, 8, torch.float32, 1).requires_grad_(True)
  gy = torch.randn(19, 8, device=DEV)
  every = torch.autograd.grad(F.layer_norm(x, w, b), [x, w, b], gy)
  for i, t in enumerate((x, w, b)):
    frozen = [u.detach() if u is not t else u for u in (x, w, b)]
    assert torch.equal(torch.autograd.grad(F.layer_norm(*frozen), [t], gy)[0], every[i])
  assert not F.layer_norm(x.detach(), w.detach(), b.detach()).requires_grad


def test_layer_norm_values_that_are_not_finite_stay_in_their_row():
  x = _rows(9, 70, torch.float32, 2)
  clean = F.layer_norm(x)
  bad = x.clone()
  bad[2, 5], bad[6, 69] = float('nan'), float('inf')
  y = F.layer_norm(bad, relu=True)
  keep = [i for i in range(9) if i not in (2, 6)]
  assert torch.equal(y[keep], torch.relu(clean[keep])) and torch.isnan(y[2]).all() and torch.isnan(y[6]).any()


def test_layer_norm_gradient_against_differences():
  g = _gen(11)
  x = torch.randn(6, 33, generator=g).to(DEV).requires_grad_(True)
  w = torch.randn(33, generator=g).to(DEV).requires_grad_(True)
  b = torch.randn(33, generator=g).to(DEV).requires_grad_(True)
  gy = torch.randn(6, 33, generator=g).to(DEV)
  grads = torch.autograd.grad(F.layer_norm(x, w, b), [x, w, b], gy)
  value = lambda xx, ww, bb: float((ref.layer_norm(xx, ww, bb, 1e-5, False)[0] * gy.double().cpu()).sum())
  for i, t in enumerate((x, w, b)):
    d = torch.randn(t.shape, generator=g)
    h = 1e-4
    args = [u.detach().double().cpu() for u in (x, w, b)]
    up, dn = list(args), list(args)
    up[i], dn[i] = args[i] + h * d.double(), args[i] - h * d.double()
    num = (value(*up) - value(*dn)) / (2 * h)
    ana = float((grads[i].double().cpu() * d.double()).sum())
    assert abs(num - ana) <= 1e-5 * float((grads[i].double().cpu() * d.double()).abs().sum()) + 1e-6, (i, num, ana)


def test_layer_norm_same_bits_every_run():
  x = _rows(30011, 96, torch.bfloat16, 7).requires_grad_(True)
  w = torch.randn(96, generator=_gen(1)).to(DEV).requires_grad_(True)
  b = torch.randn(96, generator=_gen(2)).to(DEV).requires_grad_(True)
  gy = torch.randn(30011, 96, generator=_gen(3)).to(torch.bfloat16).to(DEV)
  runs = [torch.autograd.grad(F.layer_norm(x, w, b), [x, w, b], gy) for _ in range(3)]
  for r in runs[1:]:
    assert all(torch.equal(a, c) for a, c in zip(runs[0], r))


def test_layer_norm_half_parameters_get_their_own_type():
  w = torch.ones(16, device=DEV, dtype=torch.bfloat16, requires_grad=True)
  x = _rows(4, 16, torch.bfloat16, 1)
  gw, = torch.autograd.grad(F.layer_norm(x, w).sum(), [w])
  assert gw.dtype == torch.bfloat16


# ------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('n', [1, 3, 4, 5, 7, 8, 9, 1000, 4099, 70001])
@pytest.mark.parametrize('residual', [False, True])
def test_dropout_mask_and_values(n, dtype, residual):
  g = _gen(n)
  x = torch.randn(n, generator=g).to(dtype).to(DEV).requires_grad_(True)
  r = torch.randn(n, generator=g).to(dtype).to(DEV).requires_grad_(True) if residual else None
  gy = torch.randn(n, generator=g).to(dtype).to(DEV)
  for p, seed, call in ((0.1, 7, 0), (0.5, 2 ** 63 + 12345, 2 ** 40 + 3), (0.0, 1, 1), (0.999, 3, 2 ** 32 - 1)):
    y = F.dropout(x, p, seed, call, residual=r)
    keep = ref.kept((n,), p, seed, call)
    factor = keep.double() / (1 - p)
    want = x.detach().double().cpu() * factor + (r.detach().double().cpu() if residual else 0.0)
    # the scale and the product round once each, the sum once, the store once
    size = x.detach().double().cpu().abs() * factor + (r.detach().double().cpu().abs() if residual else 0.0)
    ref.check(y, want, 4 * ref.U32 * size + ref.half_step(dtype) * (want.abs() + 4 * ref.U32 * size) + 1e-7 * (dtype == torch.float16), 'y')
    if not residual:
      assert torch.equal(y.detach().cpu() == 0, ~keep | (x.detach().cpu() == 0))
    grads = torch.autograd.grad(y, [x, r] if residual else [x], gy)
    wantg = gy.double().cpu() * factor
    ref.check(grads[0], wantg, (2 * ref.U32 + ref.half_step(dtype)) * wantg.abs() * (1 + 1e-6) + 1e-7 * (dtype == torch.float16), 'dx')
    assert torch.equal(grads[0].cpu() == 0, ~keep | (gy.cpu() == 0))
    if residual:
      assert torch.equal(grads[1], gy)


def test_dropout_call_number_from_the_device_and_views():
  x = torch.randn(37, 11, generator=_gen(1)).to(DEV)
  by_value = F.dropout(x, 0.3, 5, 2 ** 33 + 9)
  assert torch.equal(F.dropout(x, 0.3, 5, torch.tensor([2 ** 33 + 9], device=DEV)), by_value)
  assert not torch.equal(F.dropout(x, 0.3, 5, 2 ** 33 + 10), by_value)
  assert not torch.equal(F.dropout(x, 0.3, 6, 2 ** 33 + 9), by_value)
  # the mask goes by the row-major index, wherever the memory lies
  off = torch.empty(37 * 11 + 1, device=DEV)[1:].view(37, 11).copy_(x)
  assert torch.equal(F.dropout(off, 0.3, 5, 2 ** 33 + 9), by_value)
  t = x.t().contiguous().t()
  assert not t.is_contiguous() and torch.equal(F.dropout(t, 0.3, 5, 2 ** 33 + 9), by_value)
  assert torch.equal(F.dropout(x.reshape(-1), 0.3, 5, 2 ** 33 + 9), by_value.reshape(-1))
  assert F.dropout(x[:0], 0.3, 5, 0).shape == (0, 11)


def test_dropout_drops_whatever_an_element_holds():
  keep = ref.kept((64,), 0.5, 3, 0)
  x = torch.ones(64)
  x[~keep] = float('nan')
  x[(~keep).nonzero()[0]] = float('inf')
  y = F.dropout(x.to(DEV), 0.5, 3, 0).cpu()
  assert torch.equal(y, torch.where(keep, 2.0, 0.0))


def test_dropout_keeps_its_share():
  """p of 2 M elements, and of every one of 64 residues of the index: within 6 standard deviations."""
  n, p = 1 << 21, 0.2
  y = F.dropout(torch.ones(n, device=DEV), p, 99, 4)
  dropped = (y == 0).double().cpu()
  assert abs(float(dropped.mean()) - p) < 6 * (p * (1 - p) / n) ** 0.5
  per = dropped.view(-1, 64).mean(0)
  assert float((per - p).abs().max()) < 6 * (p * (1 - p) / (n / 64)) ** 0.5


def test_dropout_refuses_a_backward_pass_behind_a_changed_call_number():
  call = torch.zeros(1, dtype=torch.int64, device=DEV)
  x = torch.randn(10, device=DEV, requires_grad=True)
  y = F.dropout(x, 0.5, 1, call)
  call.add_(1)
  with pytest.raises(RuntimeError, match='modified by an inplace operation'):
    y.sum().backward()


def test_next_call_counts():
  counter = torch.full((1,), 41, dtype=torch.int64, device=DEV)
  calls = [F.next_call(counter) for _ in range(3)]
  assert [int(c) for c in calls] == [41, 42, 43] and int(counter) == 44


# ------------------------------------------------------------------------------ captured, other streams
def test_captured_layers_replay():
  """LayerNorm and Dropout forward and backward in a graph: replays follow new inputs and draw new masks, with eager work
  in between."""
  from torchrl_amd.contrib.models import Dropout, LayerNorm
  norm, drop = LayerNorm(48).to(DEV), Dropout(0.4, seed=17).to(DEV)
  x = torch.randn(500, 48, device=DEV, requires_grad=True)
  gy = torch.randn(500, 48, device=DEV)

  def body():
    y = drop(norm(x, relu=True))
    return (y.detach(),) + torch.autograd.grad(y, [x, norm.weight, norm.bias], gy)      # (no graph outlives the body)

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    body()
  torch.cuda.current_stream().wait_stream(side)
  torch.cuda.synchronize()
  drop.calls.fill_(100)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    outs = body()
  start = int(drop.calls)
  assert start == 100      # (captured, not run)
  masks = []
  for i in range(4):
    with torch.no_grad():
      x.copy_(torch.randn(500, 48, generator=_gen(i)).to(DEV))
    graph.replay()
    got = [t.clone() for t in outs]
    torch.cuda.synchronize()
    xx = x.detach().clone().requires_grad_(True)
    h = F.layer_norm(xx, norm.weight, norm.bias, norm.eps, relu=True)
    y = F.dropout(h, 0.4, 17, 100 + i)
    want = (y,) + torch.autograd.grad(y, [xx, norm.weight, norm.bias], gy)
    for a, b in zip(got, want):
      assert torch.equal(a, b), i
    masks.append(got[0] == 0)
  assert int(drop.calls) == 104
  assert not torch.equal(masks[0], masks[1])


def test_two_graphs_and_two_streams_share_nothing():
  """Backward passes of two captured graphs replayed on two streams at once: each has its own partial sums."""
  params = [(torch.randn(64, device=DEV, requires_grad=True), torch.randn(64, device=DEV, requires_grad=True)) for _ in range(2)]
  xs = [torch.randn(60000, 64, device=DEV) for _ in range(2)]
  gy = torch.randn(60000, 64, device=DEV)
  run = lambda i: torch.autograd.grad(F.layer_norm(xs[i], *params[i]), list(params[i]), gy)
  want = [run(i) for i in range(2)]
  graphs, outs = [], []
  for i in range(2):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      run(i)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      outs.append(run(i))
    graphs.append(g)
  streams = [torch.cuda.Stream() for _ in range(2)]
  for _ in range(3):
    for i in range(2):
      streams[i].wait_stream(torch.cuda.current_stream())
      with torch.cuda.stream(streams[i]):
        graphs[i].replay()
        graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
      assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))


# ------------------------------------------------------------------------------ modules and controllers
@pytest.mark.parametrize('batch', [64, 3000, 9000])
def test_qnet_with_layer_norm_equals_torch_modules(batch):
  """The stack with its fused layers against plain torch modules in 64 bits holding the same parameters."""
  from torchrl_amd.contrib.models import QNet
  torch.manual_seed(0)
  net = QNet(9, 5, hidden=(64, 48), layer_norm=True).to(DEV)
  plain = nn.Sequential(nn.Linear(9, 64), nn.LayerNorm(64), nn.ReLU(), nn.Linear(64, 48), nn.LayerNorm(48), nn.ReLU(),
                        nn.Linear(48, 5)).double()
  plain.load_state_dict({k[len('net.'):]: v.double().cpu() for k, v in net.state_dict().items()})
  x = torch.randn(batch, 9, generator=_gen(1))
  g = torch.randn(batch, 5, generator=_gen(2))
  y = net(x.to(DEV))
  want = plain(x.double())
  # a value near zero in front of a ReLU may fall on either side: one of them moves a gradient by at most one row's share
  torch.testing.assert_close(y.double().cpu(), want, rtol=1e-4, atol=1e-4)
  y.backward(g.to(DEV))
  want.backward(g.double())
  for (n, p), q in zip(net.named_parameters(), plain.parameters()):
    scale = float(q.grad.abs().max())
    assert float((p.grad.double().cpu() - q.grad).abs().max()) <= 2e-3 * scale, n


def test_dropout_stack_modes():
  from torchrl_amd.contrib.models import QNet
  torch.manual_seed(1)
  net = QNet(6, 3, hidden=32, layer_norm=True, dropout=0.5).to(DEV)
  x = torch.randn(20, 6, device=DEV)
  net.train()
  a, b = net(x), net(x)
  assert not torch.equal(a, b)
  net.eval()
  assert torch.equal(net(x), net(x))
  calls = [int(v) for k, v in net.state_dict().items() if k.endswith('calls')]
  assert calls == [2, 2]
  drops = [m for m in net.net if type(m).__name__ == 'Dropout']
  assert drops[0]._rng.next()[0] != drops[1]._rng.next()[0]      # two layers never share a mask


@pytest.mark.parametrize('graph', [False, True])
def test_ddpg_controller_with_a_regularised_critic(graph):
  from torchrl_amd.contrib.controllers import DDPGController
  torch.manual_seed(0)
  np.random.seed(0)
  ctl = DDPGController(4, 2, -1.0, 1.0, device=DEV, hidden=64, layer_norm=True, dropout=0.01, graph=graph)
  assert ctl._fused is None and len([m for m in ctl.critic.net if type(m).__name__ == 'LayerNorm']) == 2
  before = ctl._critic.data.clone()
  g = _gen(0)
  for i in range(4):
    batch = [torch.randn(32, 4, generator=g), torch.rand(32, 2, generator=g), torch.randn(32, 1, generator=g),
             torch.randn(32, 4, generator=g), torch.zeros(32, 1)]
    info = ctl.learn(*(t.to(DEV) for t in batch))
    assert all(torch.isfinite(v).item() for v in info.values())
  assert not torch.equal(before, ctl._critic.data)
  # the critic ran on (s, actor(s)) and on (s, a) each step, the target's once
  assert [int(b) for b in ctl.critic.buffers()] == [8, 8] and [int(b) for b in ctl.target_critic.buffers()] == [4, 4]
  assert ctl.act(np.zeros((3, 4), np.float32)).shape == (3, 2)


@pytest.mark.parametrize('graph', [False, True])
def test_dqn_controller_with_a_regularised_network(graph):
  from torchrl_amd.contrib.controllers import DQNController
  torch.manual_seed(0)
  np.random.seed(0)
  ctl = DQNController(4, 3, device=DEV, hidden=32, layer_norm=True, dropout=0.1, double_dqn=True, graph=graph)
  assert ctl._fused is None
  g = _gen(0)
  for i in range(6):
    batch = [torch.randn(32, 4, generator=g), torch.randint(0, 3, (32, 1), generator=g).float(),
             torch.randn(32, 1, generator=g), torch.randn(32, 4, generator=g), torch.zeros(32, 1)]
    assert torch.isfinite(ctl.learn(*(t.to(DEV) for t in batch))['td_loss']).item()
    assert ctl.q_net.training
  obs = np.zeros((5, 4), np.float32)
  assert len(ctl.act(obs)) == 5 and not ctl.q_net.training
  assert ctl.act_device(torch.zeros(5, 4, device=DEV)).shape == (5,)


def test_fused_mlp_off_takes_torchs_layer_norm():
  from torchrl_amd import config
  from torchrl_amd.contrib.models import LayerNorm
  m = LayerNorm(24).to(DEV)
  x = torch.randn(6, 24, device=DEV)
  a = m(x, relu=True)
  config.fused_mlp = False
  try:
    b = m(x, relu=True)
  finally:
    config.fused_mlp = True
  torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)
  c = copy.deepcopy(m).cpu()(x.cpu(), relu=True)
  torch.testing.assert_close(a.cpu(), c, rtol=1e-5, atol=1e-6)


def test_rows_past_32_bits():
  """More than 2^31 elements: the last rows are those of a small call, and dropout's mask goes on by the element's number."""
  rows, width = (1 << 31) // 64 + 1000, 64
  x = torch.empty(rows, width, dtype=torch.bfloat16, device=DEV)
  x[:1000] = 1.0
  tail = torch.randn(500, width, generator=_gen(1)).bfloat16().to(DEV)
  x[-500:] = tail
  y = F.layer_norm(x)
  assert torch.equal(y[-500:], F.layer_norm(tail))
  y = F.dropout(x, 0.5, 11, 3)
  first = (rows - 500) * width
  words = ref.philox_words_from(first, 500 * width, 11, 3)
  keep = torch.from_numpy(words >= np.uint64(1 << 31)).view(500, width)
  assert torch.equal(y[-500:].cpu(), torch.where(keep, 2 * tail.cpu(), torch.zeros((), dtype=torch.bfloat16)))


def test_a_copied_dropout_layer_draws_its_own_masks():
  from torchrl_amd.contrib.models import Dropout
  a = Dropout(0.5).to(DEV)
  x = torch.randn(1000, device=DEV)
  a(x)
  b = copy.deepcopy(a)
  assert int(b.calls) == 1 and not torch.equal(a(x), b(x))
  c = Dropout(0.5, seed=9).to(DEV)
  assert torch.equal(c(x), copy.deepcopy(Dropout(0.5, seed=9)).to(DEV)(x))


def test_layer_norm_module_takes_other_types_through_torch():
  from torchrl_amd.contrib.models import LayerNorm
  m = LayerNorm(16).to(DEV).double()
  x = torch.randn(4, 16, device=DEV, dtype=torch.float64)
  torch.testing.assert_close(m(x), torch.nn.functional.layer_norm(x, (16,), m.weight, m.bias))


def test_one_tensor_in_two_roles():
  """dropout(x, residual=x) and layer_norm(x, w, w): the gradients of both roles add up."""
  x = torch.randn(300, 40, generator=_gen(0)).to(DEV).requires_grad_(True)
  gy = torch.randn(300, 40, generator=_gen(1)).to(DEV)
  y = F.dropout(x, 0.5, 3, 4, residual=x)
  keep = F.dropout(torch.ones_like(x), 0.5, 3, 4)      # 0 or 2
  assert torch.equal(y, x + keep * x)
  g, = torch.autograd.grad(y, [x], gy)
  assert torch.equal(g, gy + keep * gy)
  w = torch.randn(40, generator=_gen(2)).to(DEV).requires_grad_(True)
  u, v = w.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
  one, = torch.autograd.grad(F.layer_norm(x, w, w), [w], gy)
  two = torch.autograd.grad(F.layer_norm(x, u, v), [u, v], gy)
  assert torch.equal(one, two[0] + two[1])


def test_dropout_module_with_a_residual_of_another_type():
  """As under autocast: the branch in bfloat16, the residual in float32; training has the type that eval mode has."""
  from torchrl_amd.contrib.models import Dropout
  m = Dropout(0.5, seed=5).to(DEV)
  x = torch.randn(200, 16, generator=_gen(0)).bfloat16().to(DEV).requires_grad_(True)
  r = torch.randn(200, 16, generator=_gen(1)).to(DEV).requires_grad_(True)
  y = m(x, residual=r)
  assert y.dtype == m.eval()(x, residual=r).dtype == torch.float32
  assert torch.equal(y, F.dropout(x.float(), 0.5, 5, 0, residual=r))
  gx, gr = torch.autograd.grad(y.sum(), [x, r])
  assert gx.dtype == torch.bfloat16 and torch.equal(gr, torch.ones_like(r))
  y = m(r, residual=x)
  assert y.dtype == torch.float32
