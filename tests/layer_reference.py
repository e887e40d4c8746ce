"""Plain 64-bit implementations of layer norm, dropout and decay attention, and bounds of what 32-bit sums may be off.

A bound counts roundings: a sum of n terms added in any order, each a product of a few rounded factors, is off by at most
about n * 2^-24 times the sum of the terms' absolute values; storing it adds half a step of the output's type."""
import numpy as np
import torch

U32 = 2.0 ** -24


def half_step(dtype):
  return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------ layer norm
def layer_norm(x, w, b, eps, relu, gy=None):
  """(y, dx, dw, db) in 64 bits from the inputs' own values, and the bounds of the four."""
  dt = x.dtype
  x = x.detach().double().cpu()
  D = x.shape[-1]
  w64 = torch.ones(D).double() if w is None else w.detach().double().cpu()
  b64 = torch.zeros(D).double() if b is None else b.detach().double().cpu()
  m = x.mean(-1, keepdim=True)
  var = ((x - m) ** 2).mean(-1, keepdim=True)
  r = 1.0 / torch.sqrt(var + eps)
  n = (x - m) * r
  z = n * w64 + b64
  y = z.clamp_min(0.0) if relu else z
  # adds in a row's sum: up to 8 slots of 8 elements a lane and 8 exchanges, more per lane in rows past 8,192 elements
  K = 80 + D / 256
  dm = K * U32 * x.abs().mean(-1, keepdim=True)
  dn = r * (dm + 2 * U32 * x.abs()) + n.abs() * (K + 8) * U32 + n.abs() * (r * dm) ** 2
  dz = dn * w64.abs() + 4 * U32 * (n.abs() * w64.abs() + b64.abs())
  by = dz + half_step(dt) * (y.abs() + dz)
  if gy is None:
    return y, by
  g = gy.detach().double().cpu()
  if relu:
    g = torch.where(z <= 0, 0.0, g)
  h = g * w64
  a, c = h.mean(-1, keepdim=True), (h * n).mean(-1, keepdim=True)
  dx = r * (h - a - n * c)
  da = K * U32 * h.abs().mean(-1, keepdim=True)
  dc = K * U32 * (h * n).abs().mean(-1, keepdim=True) + (h.abs() * dn).mean(-1, keepdim=True)
  ddx = r * (da + n.abs() * dc + dn * c.abs() + 8 * U32 * (h.abs() + a.abs() + (n * c).abs())) + dx.abs() * (K + 8) * U32
  bx = ddx + half_step(dt) * (dx.abs() + ddx)
  flat = lambda t: t.reshape(-1, D)
  dw, db = flat(g * n).sum(0), flat(g).sum(0)
  rows = flat(x).shape[0]
  Kr = 64 + rows / 16
  bw = Kr * U32 * flat((g * n).abs()).sum(0) + flat(g.abs() * dn).sum(0)
  bb = Kr * U32 * flat(g.abs()).sum(0)
  return (y, dx, dw, db), (by, bx, bw, bb), z.abs().amin() if z.numel() else 1.0


# ------------------------------------------------------------------------------ dropout
def philox_words(n, seed, call):
  """Word i % 4 of Philox-4x32-10, key = seed, counter = (call, i // 4 with its top bit set), for i < n."""
  return philox_words_from(0, n, seed, call)


def philox_words_from(first, n, seed, call):
  """The same for first <= i < first + n, first a multiple of 4."""
  low = 0xFFFFFFFF
  groups = np.arange((n + 3) // 4, dtype=np.uint64) + np.uint64(first // 4)
  c = [np.full_like(groups, call & low), np.full_like(groups, call >> 32), groups & np.uint64(low),
       (groups >> np.uint64(32)) | np.uint64(1 << 31)]
  k = [seed & low, seed >> 32]
  for _ in range(10):
    a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
    c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & np.uint64(low),
         (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & np.uint64(low)]
    k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
  return np.stack(c, 1).reshape(-1)[:n]


def kept(shape, p, seed, call):
  n = int(np.prod(shape))
  return torch.from_numpy(philox_words(n, seed, call) >= np.uint64(min(2 ** 32 - 1, int(p * 2 ** 32 + 0.5)))).view(shape)


# ------------------------------------------------------------------------------ decay attention
def decay_attention(q, k, v, decay, scale=None, start=None, lengths=None, state=None, gy=None, gstate=None):
  """The recurrence step by step in 64 bits, selections where the definition says "not read": dict of out, state and, with
  gy or gstate, dq, dk, dv, dstate."""
  q, k, v, decay = (t.detach().double().cpu() for t in (q, k, v, decay))
  T, N, H, dk = q.shape
  dv = v.shape[3]
  scale = dk ** -0.5 if scale is None else scale
  lam = decay.view(1, H, 1, 1)
  S0 = torch.zeros(N, H, dk, dv, dtype=torch.float64) if state is None else state.detach().double().cpu()
  L = [T] * N if lengths is None else [min(max(int(x), 0), T) for x in lengths]
  live = torch.tensor([[t < L[n] for n in range(N)] for t in range(T)], dtype=torch.bool).view(T, N)
  cut = torch.zeros(T, N, dtype=torch.bool) if start is None else start.detach().cpu() != 0
  zero = torch.zeros((), dtype=torch.float64)
  S, out = S0.clone(), torch.zeros(T, N, H, dv, dtype=torch.float64)
  want = gy is not None or gstate is not None
  G = torch.zeros_like(out) if gy is None else gy.detach().double().cpu()
  dq, dk_, dv_ = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
  for t in range(T):
    on, c = live[t].view(N, 1, 1, 1), cut[t].view(N, 1, 1, 1)
    new = torch.where(c, zero, lam * S) + k[t].unsqueeze(-1) * v[t].unsqueeze(-2)
    S = torch.where(on, new, S)
    out[t] = torch.where(on[..., 0], scale * (q[t].unsqueeze(-1) * S).sum(-2), zero)
    if want:
      dq[t] = torch.where(on[..., 0], scale * (S * G[t].unsqueeze(-2)).sum(-1), zero)
  res = dict(out=out, state=S)
  if not want:
    return res
  R = torch.zeros_like(S) if gstate is None else gstate.detach().double().cpu()
  for t in reversed(range(T)):
    on, c = live[t].view(N, 1, 1, 1), cut[t].view(N, 1, 1, 1)
    R1 = R + scale * q[t].unsqueeze(-1) * G[t].unsqueeze(-2)
    dk_[t] = torch.where(on[..., 0], (R1 * v[t].unsqueeze(-2)).sum(-1), zero)
    dv_[t] = torch.where(on[..., 0], (R1 * k[t].unsqueeze(-1)).sum(-2), zero)
    R = torch.where(on, torch.where(c, zero, lam * R1), R)
  res.update(dq=dq, dk=dk_, dv=dv_, dstate=R)
  return res


def decay_bounds(q, k, v, decay, dtype, **kw):
  """Bounds of decay_attention's results: the recurrence on absolute values has every term of a result; a term meets at most
  T / 16 scalings of the state, T additions to it, dk (dv) additions of a row and a few roundings of its own."""
  scale = kw.pop('scale', None)
  absd = {n: (t.abs() if torch.is_tensor(t) and n in ('state', 'gy', 'gstate') else t) for n, t in kw.items()}
  scale = (q.shape[3] ** -0.5 if scale is None else abs(scale))
  a = decay_attention(q.abs(), k.abs(), v.abs(), decay, scale=scale, **absd)
  terms = (2 * q.shape[0] + max(q.shape[3], v.shape[3]) + 32) * U32
  return {n: terms * t + (0.0 if n in ('state', 'dstate') else half_step(dtype) * t) + 1e-40 for n, t in a.items()}


def check(got, want, bound, what):
  got = got.detach().double().cpu()
  assert got.shape == want.shape, (what, tuple(got.shape), tuple(want.shape))
  assert torch.isfinite(got).all(), what
  over = (got - want).abs() - bound
  worst = float(over.max()) if over.numel() else -1.0
  assert worst <= 0, '%s: over its bound by %g (largest error %g, largest value %g)' % (
      what, worst, float((got - want).abs().max()), float(want.abs().max()))
