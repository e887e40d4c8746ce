"""Decay attention on the device against the recurrence in 64 bits (tests/layer_reference.py has the bounds)."""
import pytest
import torch

from tests import layer_reference as ref
from torchrl_amd import functional as F

pytestmark = pytest.mark.gpu
DEV = 'cuda'
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(T, N, H, dk, dv, dtype=torch.float32, seed=0, cuts=0.0, ragged=False, state=True, decay=None):
  g = torch.Generator().manual_seed(seed * 7919 + T * 31 + N * 17 + H * 5 + dk + dv)
  rn = lambda *s: torch.randn(*s, generator=g)
  a = dict(q=rn(T, N, H, dk).to(dtype), k=rn(T, N, H, dk).to(dtype), v=rn(T, N, H, dv).to(dtype))
  a['decay'] = 1.0 - torch.exp2(-1.0 - 1.5 * torch.arange(H).float()) if decay is None else torch.tensor(decay)
  a['start'] = (torch.rand(T, N, generator=g) < cuts).float() if cuts else None
  a['lengths'] = torch.randint(0, T + 1, (N,), generator=g, dtype=torch.int32) if ragged else None
  a['state'] = rn(N, H, dk, dv) if state else None
  a['gy'], a['gstate'] = rn(T, N, H, dv).to(dtype), rn(N, H, dk, dv)
  return a


def _run(a, grads=True, scale=None, use=('out', 'state')):
  """Results of the framework's call on the case's inputs, by name."""
  dev = {n: (t.to(DEV) if t is not None else None) for n, t in a.items()}
  leaves = [n for n in ('q', 'k', 'v', 'state') if dev[n] is not None]
  if grads:
    for n in leaves:
      dev[n].requires_grad_(True)
  out, last = F.decay_attention(dev['q'], dev['k'], dev['v'], dev['decay'], scale=scale, start=dev['start'],
                                lengths=dev['lengths'], state=dev['state'])
  res = dict(out=out, state=last)
  if grads:
    pairs = [(out, dev['gy'])] * ('out' in use) + [(last, dev['gstate'])] * ('state' in use)
    gr = torch.autograd.grad([p[0] for p in pairs], [dev[n] for n in leaves], [p[1] for p in pairs])
    res.update({'d' + n: t for n, t in zip(leaves, gr)})
  return res


def _check(a, grads=True, scale=None, use=('out', 'state')):
  got = _run(a, grads, scale, use)
  kw = dict(scale=scale, start=a['start'], lengths=a['lengths'], state=a['state'])
  if grads:
    kw.update(gy=a['gy'] if 'out' in use else None, gstate=a['gstate'] if 'state' in use else None)
  want = ref.decay_attention(a['q'], a['k'], a['v'], a['decay'], **kw)
  bound = ref.decay_bounds(a['q'], a['k'], a['v'], a['decay'], a['q'].dtype, **kw)
  for n, t in got.items():
    ref.check(t, want[n], bound[n], n)
  return got, want


SHAPES = [(1, 1, 1, 1, 1), (1, 3, 2, 64, 64), (2, 2, 1, 5, 3), (15, 2, 2, 16, 16), (16, 1, 3, 32, 32), (17, 2, 1, 33, 64),
          (31, 3, 2, 64, 17), (33, 2, 3, 48, 80), (47, 1, 2, 128, 128), (50, 5, 1, 100, 128), (64, 3, 1, 17, 5),
          (70, 2, 2, 65, 66), (100, 2, 2, 127, 31), (40, 3, 2, 8, 120), (20, 2, 1, 1, 128), (20, 2, 1, 128, 1),
          (24, 1, 1, 96, 112)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_decay_attention_shapes(shape, dtype):
  _check(_inputs(*shape, dtype=dtype))
  _check(_inputs(*shape, dtype=dtype, seed=1, cuts=0.15, ragged=True))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', [(600, 1, 2, 64, 64), (1000, 2, 1, 33, 40), (130, 1, 1, 16, 128), (333, 3, 3, 48, 80),
                                   (1025, 1, 1, 128, 64), (129, 2, 2, 20, 20)])
def test_decay_attention_in_segments_of_time(shape, dtype):
  """Few heads and many steps: the pass is cut into segments and joined."""
  _check(_inputs(*shape, dtype=dtype))
  _check(_inputs(*shape, dtype=dtype, seed=1, cuts=0.01))
  _check(_inputs(*shape, dtype=dtype, seed=2, cuts=0.01, ragged=True))


def test_decay_attention_many_heads_in_wide_tiles():
  """Enough heads that a wave carries several column tiles."""
  _check(_inputs(20, 600, 4, 24, 64, cuts=0.05, ragged=True))
  _check(_inputs(18, 530, 4, 70, 33, dtype=torch.bfloat16, cuts=0.05))
  _check(_inputs(18, 300, 4, 64, 40, cuts=0.05))


@pytest.mark.parametrize('use', [('out',), ('state',)])
def test_decay_attention_one_gradient_alone(use):
  _check(_inputs(40, 2, 2, 32, 16, cuts=0.05), use=use)
  _check(_inputs(500, 1, 1, 32, 16, cuts=0.01), use=use)


def test_decay_attention_without_state_flags_or_scale():
  _check(_inputs(37, 2, 2, 20, 24, state=False))
  _check(_inputs(37, 2, 2, 20, 24, state=False), scale=0.7)
  _check(_inputs(37, 2, 2, 20, 24), scale=-1.3)
  _check(_inputs(37, 2, 2, 20, 24), grads=False)


@pytest.mark.parametrize('decay', [[0.0, 1.0], [1.0, 1.0], [0.0, 0.0], [1e-30, 0.999999]])
def test_decay_attention_extreme_decays(decay):
  _check(_inputs(50, 2, 2, 16, 16, decay=decay, cuts=0.05))
  _check(_inputs(400, 1, 2, 16, 16, decay=decay, cuts=0.01))


def test_decay_attention_starts_everywhere_lengths_zero_and_one():
  a = _inputs(35, 4, 2, 24, 24, cuts=0.1)
  a['start'] = torch.ones(35, 4)
  _check(a)
  a = _inputs(35, 4, 2, 24, 24, cuts=0.1)
  a['lengths'] = torch.tensor([0, 1, 35, 16], dtype=torch.int32)
  got, _ = _check(a)
  assert not got['out'][:, 0].any() and torch.equal(got['state'][0].detach().cpu(), a['state'][0])
  assert not got['dq'][:, 0].any() and not got['dv'][1:, 1].any()
  assert torch.equal(got['dstate'][0].cpu(), a['gstate'][0])
  # lengths beyond the rollout are its own
  a['lengths'] = torch.tensor([-3, 1, 99, 16], dtype=torch.int32)
  again = _run(a)
  for n in got:
    assert torch.equal(got[n], again[n]), n
  a['lengths'] = torch.tensor([-3, 1, 2 ** 40, 16], dtype=torch.int64)
  again = _run(a)
  for n in got:
    assert torch.equal(got[n], again[n]), n


def test_decay_attention_empty_rollouts():
  a = _inputs(0, 3, 2, 8, 8)
  got = _run(a)
  assert got['out'].shape == (0, 3, 2, 8) and torch.equal(got['state'].detach().cpu(), a['state'])
  assert torch.equal(got['dstate'].cpu(), a['gstate'])
  got = _run(_inputs(5, 0, 2, 8, 8))
  assert got['out'].shape == (5, 0, 2, 8) and got['dstate'].shape == (0, 2, 8, 8)


def test_decay_attention_start_types():
  a = _inputs(60, 3, 2, 16, 16, cuts=0.1)
  base = _run(a)
  for s in (a['start'].bool(), a['start'].to(torch.uint8) * 7, a['start'] * -0.25, a['start'].t().contiguous().t()):
    got = _run(dict(a, start=s))
    for n in base:
      assert torch.equal(base[n], got[n]), n


def test_decay_attention_reads_through_strides():
  """Slices of one projection, env-major memory, rows off the 16 B grid: the same bits as dense copies."""
  a = _inputs(45, 3, 2, 20, 20, cuts=0.05)
  base = _run(a)
  qkv = torch.stack([a['q'], a['k'], a['v']], 2).to(DEV)                       # [T, N, 3, H, D]
  env = [t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1) for t in (a['q'], a['k'], a['v'])]
  off = [torch.empty(t.numel() + 1, device=DEV)[1:].view(t.shape).copy_(t) for t in (a['q'], a['k'], a['v'])]
  wide = [torch.randn(45, 3, 2, 40, device=DEV)[..., 7:27].copy_(t) for t in (a['q'], a['k'], a['v'])]
  last = [t.to(DEV).transpose(2, 3).contiguous().transpose(2, 3) for t in (a['q'], a['k'], a['v'])]
  for q, k, v in (qkv.unbind(2), env, off, wide, last):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    st = a['state'].to(DEV).requires_grad_(True)
    out, s = F.decay_attention(q, k, v, a['decay'].to(DEV), start=a['start'].to(DEV), state=st)
    gr = torch.autograd.grad([out, s], [q, k, v, st], [a['gy'].to(DEV), a['gstate'].to(DEV)])
    for n, t in zip(('out', 'state', 'dq', 'dk', 'dv', 'dstate'), (out, s) + gr):
      assert torch.equal(base[n], t), n


def test_decay_attention_shared_heads_and_broadcast_inputs():
  """Keys and values of one head expanded to all: read in place, their gradients added up over the heads."""
  a = _inputs(30, 2, 4, 16, 24, cuts=0.05)
  q = a['q'].to(DEV).requires_grad_(True)
  k1, v1 = (a[n][:, :, :1].to(DEV).requires_grad_(True) for n in ('k', 'v'))
  out, _ = F.decay_attention(q, k1.expand(-1, -1, 4, -1), v1.expand(-1, -1, 4, -1), a['decay'].to(DEV),
                             start=a['start'].to(DEV), state=a['state'][:1].to(DEV).expand(2, -1, -1, -1))
  gq, gk, gv = torch.autograd.grad(out, [q, k1, v1], a['gy'].to(DEV))
  full = dict(a, k=a['k'][:, :, :1].expand(-1, -1, 4, -1).contiguous(), v=a['v'][:, :, :1].expand(-1, -1, 4, -1).contiguous(),
              state=a['state'][:1].expand(2, -1, -1, -1).contiguous())
  got = _run(full, use=('out',))
  assert torch.equal(out, got['out']) and torch.equal(gq, got['dq'])
  torch.testing.assert_close(gk[:, :, 0], got['dk'].sum(2), rtol=1e-5, atol=1e-5)
  torch.testing.assert_close(gv[:, :, 0], got['dv'].sum(2), rtol=1e-5, atol=1e-5)


def test_decay_attention_carries_on_where_it_stopped():
  a = _inputs(100, 2, 2, 32, 32, cuts=0.03)
  whole = _run(a, grads=False)
  dev = {n: (t.to(DEV) if t is not None else None) for n, t in a.items()}
  state, outs = dev['state'], []
  for lo, hi in ((0, 1), (1, 30), (30, 47), (47, 100)):
    o, state = F.decay_attention(dev['q'][lo:hi], dev['k'][lo:hi], dev['v'][lo:hi], dev['decay'], start=dev['start'][lo:hi],
                                 state=state)
    outs.append(o)
  kw = dict(start=a['start'], state=a['state'])
  bound = ref.decay_bounds(a['q'], a['k'], a['v'], a['decay'], torch.float32, **kw)
  assert bool(((torch.cat(outs) - whole['out']).abs().double().cpu() <= 2 * bound['out']).all())
  assert bool(((state - whole['state']).abs().double().cpu() <= 2 * bound['state']).all())


# ------------------------------------------------------------------------------ values that are not finite
def _same_pattern(got, want, bound, what):
  """Finite where the recurrence is finite (and right there), not finite where it is not."""
  got = got.detach().double().cpu()
  fine = torch.isfinite(want)
  assert torch.equal(torch.isfinite(got), fine), what
  over = ((got - want).abs() - bound)[fine]
  assert over.numel() == 0 or float(over.max()) <= 0, what


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('value', [float('nan'), float('inf'), -float('inf')])
@pytest.mark.parametrize('T,where', [(60, 21), (700, 333)])
@pytest.mark.parametrize('name', ['q', 'k', 'v'])
def test_decay_attention_not_finite_steps_reach_only_what_they_touch(name, T, where, value, dtype):
  """A value that is not finite changes the steps of its own episode from its own on, in its env and head, and nothing else:
  not the steps before it (which share its chunk), not those behind the next start."""
  a = _inputs(T, 2, 2, 20, 24, dtype=dtype)
  a['start'] = torch.zeros(T, 2)
  a['start'][[where - 8, where + 9], 0] = 1.0
  clean = dict(a)
  a = dict(a, **{name: a[name].clone()})
  a[name][where, 0, 1, 3] = value
  kw = dict(start=a['start'], state=a['state'])
  want = ref.decay_attention(a['q'], a['k'], a['v'], a['decay'], **kw)
  bound = ref.decay_bounds(clean['q'], clean['k'], clean['v'], clean['decay'], dtype, **kw)
  got = _run(a, grads=False)
  for n in ('out', 'state'):
    _same_pattern(got[n], want[n], bound[n], n)
  assert torch.isfinite(want['out'][:, 1]).all() and torch.isfinite(want['out'][where + 9:]).all()
  assert not torch.isfinite(want['out'][where, 0, 1]).all()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('T,where', [(60, 21), (700, 333)])
@pytest.mark.parametrize('name', ['q', 'k', 'v', 'gy'])
def test_decay_attention_gradients_of_not_finite_steps(name, T, where, dtype):
  a = _inputs(T, 2, 2, 20, 24, dtype=dtype)
  a['start'] = torch.zeros(T, 2)
  a['start'][[where - 8, where + 9], 0] = 1.0
  kw = dict(start=a['start'], state=a['state'], gy=a['gy'], gstate=a['gstate'])
  bound = ref.decay_bounds(a['q'], a['k'], a['v'], a['decay'], dtype, **kw)
  a = dict(a, **{name: a[name].clone()})
  a[name][where, 0, 1, 3] = float('nan')
  kw['gy'] = a['gy']
  want = ref.decay_attention(a['q'], a['k'], a['v'], a['decay'], **kw)
  got = _run(a)
  for n in ('dq', 'dk', 'dv', 'dstate'):
    _same_pattern(got[n], want[n], bound[n], n)


def test_decay_attention_state_that_is_not_finite_ends_at_a_start():
  a = _inputs(50, 2, 1, 16, 16)
  a['start'] = torch.zeros(50, 2)
  a['start'][20, 0] = 1
  bound = ref.decay_bounds(a['q'], a['k'], a['v'], a['decay'], torch.float32, start=a['start'], state=a['state'])
  a['state'] = a['state'].clone()
  a['state'][0, 0, 2, 5] = float('nan')
  want = ref.decay_attention(a['q'], a['k'], a['v'], a['decay'], start=a['start'], state=a['state'])
  got = _run(a, grads=False)
  for n in ('out', 'state'):
    _same_pattern(got[n], want[n], bound[n], n)
  assert torch.isfinite(got['state']).all()


def test_decay_attention_does_not_read_behind_the_lengths():
  a = _inputs(90, 4, 2, 24, 16, cuts=0.05)
  a['lengths'] = torch.tensor([90, 33, 1, 0], dtype=torch.int32)
  base = _run(a)
  b = dict(a)
  for n in ('q', 'k', 'v', 'gy'):
    b[n] = a[n].clone()
    for i, length in enumerate(a['lengths']):
      b[n][int(length):, i] = float('nan')
  b['start'] = a['start'].clone()
  for i, length in enumerate(a['lengths']):
    b['start'][int(length):, i] = float('nan')
  got = _run(b)
  for n in base:
    assert torch.equal(base[n], got[n]), n


# ------------------------------------------------------------------------------ gradients, runs, graphs
def test_decay_attention_gradients_against_differences():
  a = _inputs(21, 2, 2, 6, 5, cuts=0.1, ragged=True)
  got = _run(a)
  g = torch.Generator().manual_seed(1)

  def value(**over):
    r = ref.decay_attention(**{n: over.get(n, a[n]) for n in ('q', 'k', 'v', 'decay', 'start', 'lengths', 'state')})
    return float((r['out'] * a['gy'].double()).sum() + (r['state'] * a['gstate'].double()).sum())

  for n in ('q', 'k', 'v', 'state'):
    d = torch.randn(a[n].shape, generator=g, dtype=torch.float64)
    h = 1e-4
    num = (value(**{n: a[n].double() + h * d}) - value(**{n: a[n].double() - h * d})) / (2 * h)
    prod = got['d' + n].double().cpu() * d
    assert abs(num - float(prod.sum())) <= 1e-5 * float(prod.abs().sum()), n


@pytest.mark.parametrize('shape', [(40, 3, 2, 32, 48), (900, 1, 2, 64, 64)])
def test_decay_attention_same_bits_every_run(shape):
  a = _inputs(*shape, cuts=0.02)
  runs = [_run(a) for _ in range(3)]
  for r in runs[1:]:
    for n in r:
      assert torch.equal(runs[0][n], r[n]), n


@pytest.mark.parametrize('D', [32, 128])
def test_decay_attention_captured_and_on_other_streams(D):
  a = _inputs(700, 1, 2, D, D, cuts=0.01)      # (in segments: the captured passes bring workspaces of their own)
  dev = {n: (t.to(DEV) if t is not None else None) for n, t in a.items()}
  for n in ('q', 'k', 'v'):
    dev[n].requires_grad_(True)

  def body():
    out, s = F.decay_attention(dev['q'], dev['k'], dev['v'], dev['decay'], start=dev['start'], state=dev['state'])
    # (no graph outlives the body)
    return (out.detach(), s.detach()) + torch.autograd.grad(out, [dev['q'], dev['k'], dev['v']], dev['gy'])

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    body()
  torch.cuda.current_stream().wait_stream(side)
  torch.cuda.synchronize()
  graphs, outs = [], []
  for _ in range(2):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      outs.append(body())
    graphs.append(g)
  streams = [torch.cuda.Stream() for _ in range(2)]
  for i in range(3):
    with torch.no_grad():
      dev['q'].copy_(torch.randn(dev['q'].shape, generator=torch.Generator().manual_seed(i)).to(DEV))
    for st, g in zip(streams, graphs):
      st.wait_stream(torch.cuda.current_stream())
      with torch.cuda.stream(st):
        g.replay()
    torch.cuda.synchronize()
    want = body()
    for o in outs:
      assert all(torch.equal(x, y) for x, y in zip(o, want)), i


# ------------------------------------------------------------------------------ the single-step form
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('N,H,dk,dv', [(1, 1, 1, 1), (1, 4, 64, 64), (3, 2, 33, 17), (5, 1, 128, 128), (2, 3, 48, 80),
                                       (70, 2, 16, 32), (4, 2, 7, 65), (2, 1, 128, 3)])
def test_decay_step(N, H, dk, dv, dtype):
  a = _inputs(1, N, H, dk, dv, dtype=dtype)
  a['start'] = (torch.arange(N) % 3 == 2).float().view(1, N)
  want = ref.decay_attention(a['q'], a['k'], a['v'], a['decay'], start=a['start'], state=a['state'])
  bound = ref.decay_bounds(a['q'], a['k'], a['v'], a['decay'], dtype, start=a['start'], state=a['state'])
  q, k, v, st = (a[n].to(DEV) for n in ('q', 'k', 'v', 'state'))
  for start in (a['start'][0].to(DEV), a['start'][0].bool().to(DEV)):
    kept = st.clone()
    out, new = F.decay_attention_step(q[0], k[0], v[0], a['decay'].to(DEV), st, start=start)
    assert torch.equal(st, kept) and out.dtype == dtype
    ref.check(out, want['out'][0], bound['out'][0], 'out')
    ref.check(new, want['state'], bound['state'], 'state')
    o2, s2 = F.decay_attention_step(q[0], k[0], v[0], a['decay'].to(DEV), kept, start=start, out_state=kept)
    assert s2 is kept and torch.equal(s2, new) and torch.equal(o2, out)


def test_decay_step_follows_the_sequence_form():
  """Acting step by step, states in place, envs reset on the way: the sequence form's outputs and state."""
  a = _inputs(120, 5, 2, 24, 40, cuts=0.05)
  dev = {n: t.to(DEV) for n, t in a.items() if t is not None}
  whole = _run(a, grads=False)
  state, outs = dev['state'].clone(), []
  for t in range(120):
    o, state = F.decay_attention_step(dev['q'][t], dev['k'][t], dev['v'][t], dev['decay'], state, start=dev['start'][t],
                                      out_state=state)
    outs.append(o)
  bound = ref.decay_bounds(a['q'], a['k'], a['v'], a['decay'], torch.float32, start=a['start'], state=a['state'])
  assert bool(((torch.stack(outs) - whole['out']).abs().double().cpu() <= 2 * bound['out']).all())
  assert bool(((state - whole['state']).abs().double().cpu() <= 2 * bound['state']).all())


def test_decay_step_captured_in_place_and_not_finite_states():
  a = _inputs(8, 3, 2, 16, 16)
  dev = {n: t.to(DEV) for n, t in a.items() if t is not None}
  q, k, v = (dev[n][0].clone() for n in ('q', 'k', 'v'))
  start = torch.zeros(3, device=DEV)
  state = dev['state'].clone()
  graph = torch.cuda.CUDAGraph()
  F.decay_attention_step(q, k, v, dev['decay'], state.clone())
  torch.cuda.synchronize()
  with torch.cuda.graph(graph):
    out, _ = F.decay_attention_step(q, k, v, dev['decay'], state, start=start, out_state=state)
  eager = dev['state'].clone()
  state.copy_(dev['state'])
  for t in range(8):
    q.copy_(dev['q'][t])
    k.copy_(dev['k'][t])
    v.copy_(dev['v'][t])
    if t == 5:
      start.copy_(torch.tensor([0.0, 1.0, 0.0]))
      state[1] = float('nan')
      eager[1] = float('nan')
    graph.replay()
    torch.cuda.synchronize()
    o, eager = F.decay_attention_step(dev['q'][t], dev['k'][t], dev['v'][t], dev['decay'], eager, start=start)
    assert torch.equal(o, out) and torch.equal(eager, state), t
    if t == 5:
      start.zero_()
  assert torch.isfinite(state).all()


def test_decay_step_refusals_on_the_device():
  a = _inputs(1, 2, 1, 8, 8)
  q, k, v, st = (a[n].to(DEV) for n in ('q', 'k', 'v', 'state'))
  dec = a['decay'].to(DEV)
  step = lambda **kw: F.decay_attention_step(**{**dict(q=q[0], k=k[0], v=v[0], decay=dec, state=st), **kw})
  with pytest.raises(ValueError, match='no gradient'):
    step(q=q[0].clone().requires_grad_(True))
  with pytest.raises(ValueError, match='overlaps'):
    buf = torch.zeros(2 * 64 + 16, device=DEV)
    step(state=buf[:128].view(2, 1, 8, 8), out_state=buf[16:].view(2, 1, 8, 8))
  with pytest.raises(ValueError, match='contiguous'):
    step(out_state=torch.zeros(2, 1, 8, 16, device=DEV)[..., ::2])
  with pytest.raises(ValueError, match='shares memory'):
    one = torch.zeros(1, 1, 8, 8, device=DEV)
    step(q=q[0, :1], k=k[0, :1], v=v[0, :1], state=one.transpose(2, 3), out_state=one)


# ------------------------------------------------------------------------------ the block that uses all of them
def _block(seed=0, dropout=0.0):
  from torchrl_amd.contrib.models import MemoryBlock
  torch.manual_seed(seed)
  return MemoryBlock(48, heads=3, head_size=20, dropout=dropout).to(DEV)


def _block64(m, x, start):
  """The block from its definition in 64 bits."""
  p = {n: t.detach().double().cpu().requires_grad_(n != 'decay') for n, t in list(m.named_parameters()) + list(m.named_buffers())
       if t.dtype == torch.float32}
  T, N, W = x.shape
  h = torch.nn.functional.layer_norm(x, (W,), p['norm.weight'], p['norm.bias'], m.norm.eps)
  qkv = torch.nn.functional.linear(h, p['qkv.weight'], p['qkv.bias']).view(T, N, 3, m.heads, m.head_size)
  S, outs = torch.zeros(N, m.heads, m.head_size, m.head_size, dtype=torch.float64), []
  for t in range(T):
    q, k, v = qkv[t].unbind(1)
    S = torch.where(start[t].view(N, 1, 1, 1) != 0, 0.0, p['decay'].view(1, -1, 1, 1) * S) + k.unsqueeze(-1) * v.unsqueeze(-2)
    outs.append((q.unsqueeze(-1) * S).sum(-2) * m.head_size ** -0.5)
  y = x + torch.nn.functional.linear(torch.stack(outs).flatten(-2), p['out.weight'], p['out.bias'])
  return y, S, p


def test_memory_block_forward_gradients_and_steps():
  m = _block()
  g = torch.Generator().manual_seed(0)
  x = torch.randn(70, 4, 48, generator=g)
  start = (torch.rand(70, 4, generator=g) < 0.05).float()
  gy = torch.randn(70, 4, 48, generator=g)
  xd = x.to(DEV).requires_grad_(True)
  y, state = m(xd, start=start.to(DEV))
  x64 = x.double().requires_grad_(True)
  want, S, p = _block64(m, x64, start)
  torch.testing.assert_close(y.double().cpu(), want, rtol=2e-5, atol=2e-5)
  torch.testing.assert_close(state.double().cpu(), S, rtol=2e-5, atol=2e-5)
  y.backward(gy.to(DEV))
  want.backward(gy.double())
  for n, t in m.named_parameters():
    assert float((t.grad.double().cpu() - p[n].grad).abs().max()) <= 2e-5 * float(p[n].grad.abs().max()) + 2e-5, n
  torch.testing.assert_close(xd.grad.double().cpu(), x64.grad, rtol=5e-5, atol=5e-5)
  # acting: the same function a step at a time, the state in place
  st, outs = m.initial_state(4), []
  for t in range(70):
    o, st = m.step(x[t].to(DEV), st, start=start[t].to(DEV), out_state=st)
    outs.append(o)
  torch.testing.assert_close(torch.stack(outs), y.detach(), rtol=2e-5, atol=2e-5)
  torch.testing.assert_close(st, state.detach(), rtol=2e-5, atol=2e-5)


def test_memory_block_dropout_and_bf16():
  m = _block(dropout=0.25)
  x = torch.randn(20, 3, 48, device=DEV)
  m.train()
  a, _ = m(x)
  b, _ = m(x)
  share = float((a == x).float().mean())
  assert not torch.equal(a, b) and abs(share - 0.25) < 0.05
  m.eval()
  c, _ = m(x)
  assert torch.equal(c, m(x)[0])
  h = _block(dropout=0.25).bfloat16().train()
  assert torch.equal(h.decay, m.decay)      # (kept in float32: 1 - 2^-10 is 1 in bfloat16)
  y, s = h(x.bfloat16().requires_grad_(True))
  y.float().sum().backward()
  assert y.dtype == torch.bfloat16 and s.dtype == torch.float32
  assert all(torch.isfinite(p.grad).all() for p in h.parameters())


def test_second_derivatives_are_refused_and_library_errors_keep_their_class():
  from torchrl_amd import _lib
  x = torch.randn(4, 8, device=DEV, requires_grad=True)
  for y in (F.layer_norm(x), F.dropout(x, 0.5, 1, 2),
            F.decay_attention(x.view(4, 1, 1, 8), x.view(4, 1, 1, 8), x.view(4, 1, 1, 8), torch.ones(1, device=DEV))[0]):
    g, = torch.autograd.grad(y.square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match='differentiate twice'):
      g.sum().backward()
  q = torch.empty(1, 1 << 22, 1, 1, device=DEV)
  with pytest.raises(_lib.TrlError, match='too many'):
    F.decay_attention(q, q, q, torch.ones(1, device=DEV))


def test_decay_attention_offsets_past_32_bits():
  """Steps 60 M elements apart: the last ones lie past 2^31 elements and 2^32 bytes."""
  T, N, H, D = 40, 2, 2, 32
  a = _inputs(T, N, H, D, D, dtype=torch.bfloat16, cuts=0.05)
  base = _run(a)
  stride = 60_000_000
  far = {}
  for n in ('q', 'k', 'v'):
    buf = torch.empty((T - 1) * stride + N * H * D, dtype=torch.bfloat16, device=DEV)
    far[n] = buf.as_strided((T, N, H, D), (stride, H * D, D, 1)).copy_(a[n].to(DEV)).requires_grad_(True)
  out, s = F.decay_attention(far['q'], far['k'], far['v'], a['decay'].to(DEV), start=a['start'].to(DEV),
                             state=a['state'].to(DEV))
  gr = torch.autograd.grad([out, s], [far[n] for n in ('q', 'k', 'v')], [a['gy'].to(DEV), a['gstate'].to(DEV)])
  for n, t in zip(('out', 'state', 'dq', 'dk', 'dv'), (out, s) + gr):
    assert torch.equal(base[n], t), n


def test_decay_attention_on_one_thread_and_with_a_state_written_since():
  """The engine's single-threaded mode; a step that writes a saved state in place is noticed."""
  a = _inputs(40, 2, 2, 16, 16)
  base = _run(a)
  with torch.autograd.set_multithreading_enabled(False):
    got = _run(a)
  for n in base:
    assert torch.equal(base[n], got[n]), n
  dev = {n: (t.to(DEV) if t is not None else None) for n, t in a.items()}
  q = dev['q'].requires_grad_(True)
  out, _ = F.decay_attention(q, dev['k'], dev['v'], dev['decay'], state=dev['state'])
  with torch.no_grad():
    F.decay_attention_step(q[0], dev['k'][0], dev['v'][0], dev['decay'], dev['state'], out_state=dev['state'])
  with pytest.raises(RuntimeError, match='modified by an inplace operation'):
    out.sum().backward()


def test_decay_attention_of_one_tensor_in_three_roles():
  """q, k and v the same tensor: its gradient is the sum of the three."""
  g = torch.Generator().manual_seed(3)
  x = torch.randn(200, 3, 2, 24, generator=g).to(DEV).requires_grad_(True)
  gy = torch.randn(200, 3, 2, 24, generator=g).to(DEV)
  decay = torch.tensor([0.9, 0.99], device=DEV)
  one, = torch.autograd.grad(F.decay_attention(x, x, x, decay)[0], [x], gy)
  three = [x.detach().clone().requires_grad_(True) for _ in range(3)]
  q, k, v = torch.autograd.grad(F.decay_attention(*three, decay)[0], three, gy)
  # (two additions in float32, in an order that is the engine's)
  assert torch.all((one - (q + k + v)).abs() <= 2 * torch.finfo(torch.float32).eps * (q.abs() + k.abs() + v.abs()))


def test_memory_block_under_autocast():
  m = _block(dropout=0.25).train()
  x = torch.randn(40, 3, 48, device=DEV, requires_grad=True)
  with torch.autocast('cuda', torch.bfloat16):
    y, s = m(x)
    m.eval()
    z, _ = m(x)
  assert y.dtype == z.dtype == torch.float32 and s.dtype == torch.float32
  y.sum().backward()
  assert torch.isfinite(x.grad).all() and all(torch.isfinite(p.grad).all() for p in m.parameters())


def test_decay_attention_in_inference_mode():
  q = torch.randn(30, 2, 1, 8, device=DEV)
  decay = torch.full((1,), 0.95, device=DEV)
  want, last = F.decay_attention(q, q, q, decay)
  with torch.inference_mode():
    out, state = F.decay_attention(q, q, q, decay)
    assert torch.equal(out, want) and torch.equal(state, last)
    st = torch.zeros(2, 1, 8, 8, device=DEV)
    for t in range(30):
      o, st = F.decay_attention_step(q[t], q[t], q[t], decay, st, out_state=st)
  torch.testing.assert_close(st, last, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('dk,dv', [(16, 16), (33, 40), (64, 64), (128, 100)])
def test_decay_attention_flags_of_long_sequences(dk, dv, dtype):
  """More steps than a workgroup takes flags of at once, and enough heads that time is not cut (but for the smallest ones); some
  envs against the reference, uint8 flags bit for bit against float32 ones."""
  a = _inputs(530, 257, 1, dk, dv, dtype=dtype, cuts=0.02, ragged=True, decay=[0.97])
  a['lengths'][:3] = torch.tensor([530, 529, 513], dtype=torch.int32)
  a['start'][[0, 63, 64, 128, 192, 255, 256, 512, 529]] = 1.0
  a['start'][:, 1] *= -0.0      # (-0 is no start)
  got = _run(a)
  some = [0, 1, 2, 100, 256]
  part = {n: t if n == 'decay' else t[some] if n in ('lengths', 'state', 'gstate') else t[:, some] for n, t in a.items()}
  kw = {n: part[n] for n in ('start', 'lengths', 'state', 'gy', 'gstate')}
  want = ref.decay_attention(part['q'], part['k'], part['v'], part['decay'], **kw)
  bound = ref.decay_bounds(part['q'], part['k'], part['v'], part['decay'], dtype, **kw)
  for n, t in got.items():
    ref.check(t[some] if n in ('state', 'dstate') else t[:, some], want[n], bound[n], n)
  b = _run(dict(a, start=(a['start'] != 0).to(torch.uint8)))
  assert all(torch.equal(got[n], b[n]) for n in got)


def test_decay_attention_a_not_finite_step_between_flags():
  """An infinity in the first step of a block of flags, a start behind it: nothing of it after the start."""
  a = _inputs(200, 257, 1, 16, 16, decay=[0.97])
  a['start'] = torch.zeros(200, 257)
  a['start'][[65, 130]] = 1.0
  clean = _run(a, grads=False)['out']
  a['k'][64] = float('inf')
  out = _run(a, grads=False)['out']
  assert torch.equal(out[:64], clean[:64]) and not torch.isfinite(out[64]).any()
  # (its chunk's later steps are taken one by one: the same sums in another order, of up to 65 terms and 16 products each)
  terms = 4 * (65 + 16) * torch.finfo(torch.float32).eps
  size = ref.decay_attention(a['q'].abs()[65:], _inputs(200, 257, 1, 16, 16, decay=[0.97])['k'].abs()[65:], a['v'].abs()[65:],
                             a['decay'], start=a['start'][65:])['out']
  assert torch.all((out[65:] - clean[65:]).abs().double().cpu() <= terms * size)


def test_decay_attention_flags_of_long_sequences_in_one_wave():
  """As above with workgroups of one wave, whose blocks of flags are 64 steps: heads enough that time is not cut."""
  for dtype in (torch.float32, torch.bfloat16):
    a = _inputs(330, 900, 1, 16, 12, dtype=dtype, cuts=0.02, ragged=True, decay=[0.97])
    a['lengths'][:2] = torch.tensor([330, 321], dtype=torch.int32)
    a['start'][[0, 63, 64, 128, 192, 255, 256, 320, 329]] = 1.0
    got = _run(a)
    some = [0, 1, 100, 899]
    part = {n: t if n == 'decay' else t[some] if n in ('lengths', 'state', 'gstate') else t[:, some] for n, t in a.items()}
    kw = {n: part[n] for n in ('start', 'lengths', 'state', 'gy', 'gstate')}
    want = ref.decay_attention(part['q'], part['k'], part['v'], part['decay'], **kw)
    bound = ref.decay_bounds(part['q'], part['k'], part['v'], part['decay'], dtype, **kw)
    for n, t in got.items():
      ref.check(t[some] if n in ('state', 'dstate') else t[:, some], want[n], bound[n], n)


@pytest.mark.parametrize('T,N,H,D', [(4100, 1, 1, 8), (700, 30, 4, 16), (1000, 40, 2, 32), (900, 3, 2, 128)])
def test_decay_attention_many_segments_of_small_heads(T, N, H, D):
  """Segments by the number of waves: more than the workgroups join themselves, and as many as they do."""
  _check(_inputs(T, N, H, D, D, cuts=0.003, ragged=True))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('dk,dv', [(128, 64), (64, 128), (112, 32), (128, 65), (97, 128), (128, 1), (100, 68)])
def test_decay_attention_wide_heads_in_column_groups(dk, dv, dtype):
  """Heads of more than 96 are split by columns over workgroups: whole, ragged and missing second groups, with and without
  segments, and a value that is not finite in one group's columns only."""
  _check(_inputs(40, 3, 2, dk, dv, dtype=dtype, cuts=0.05, ragged=True))
  _check(_inputs(260, 1, 2, dk, dv, dtype=dtype, cuts=0.01))
  a = _inputs(40, 2, 1, dk, dv, dtype=dtype, state=False)
  clean = _run(a, grads=False)['out']
  a['v'][20, :, :, dv - 1] = float('inf')
  out = _run(a, grads=False)['out']
  assert torch.equal(out[:16], clean[:16]) and not torch.isfinite(out[20:, ..., dv - 1]).any()
  if dv > 1:      # (the other columns: the same sums, some of them step by step)
    size = ref.decay_attention(*(torch.nan_to_num(a[n].float(), posinf=0.0).abs() for n in ('q', 'k', 'v')), a['decay'])['out']
    bound = 8 * (40 + dk) * torch.finfo(torch.float32).eps + torch.finfo(dtype).eps
    assert torch.all((out - clean)[..., :dv - 1].abs().double().cpu() <= bound * size[..., :dv - 1])
