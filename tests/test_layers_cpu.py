"""Layer norm, dropout and decay attention without a device: refusals, the C entry points' checks, module construction."""
import ctypes as C

import pytest
import torch

from tests import layer_reference as ref
from torchrl_amd import _lib
from torchrl_amd import functional as F


def test_cpu_tensors_are_refused():
  x = torch.randn(3, 4)
  q = torch.randn(2, 3, 1, 4)
  for call in (lambda: F.layer_norm(x), lambda: F.dropout(x, 0.5, 0, 0), lambda: F.next_call(torch.zeros(1, dtype=torch.int64)),
               lambda: F.decay_attention(q, q, q, torch.ones(1)),
               lambda: F.decay_attention_step(q[0], q[0], q[0], torch.ones(1), torch.zeros(3, 1, 4, 4))):
    with pytest.raises(_lib.TrlError, match='HIP device'):
      call()


def _refused(rc, text):
  assert rc == -1 and text in _lib.lib().trl_last_error().decode(), (rc, _lib.lib().trl_last_error())


def test_layer_norm_entry_checks():
  lib = _lib.lib()
  p = 4096      # (never read: every call below ends before a launch)
  _refused(lib.trl_layer_norm_fwd(p, p, p, 4, 4, 1, 1e-5, 0, p, p, p, None), 'dtype')
  _refused(lib.trl_layer_norm_fwd(p, p, p, -1, 4, 0, 1e-5, 0, p, p, p, None), 'shape')
  _refused(lib.trl_layer_norm_fwd(p, p, p, 4, 0, 0, 1e-5, 0, p, p, p, None), 'shape')
  _refused(lib.trl_layer_norm_fwd(p, p, p, 4, 1 << 24, 0, 1e-5, 0, p, p, p, None), 'shape')
  _refused(lib.trl_layer_norm_fwd(p, p, p, 1 << 39, 4, 0, 1e-5, 0, p, p, p, None), 'too many')
  _refused(lib.trl_layer_norm_fwd(p, p, p, 4, 4, 0, 0.0, 0, p, p, p, None), 'eps')
  _refused(lib.trl_layer_norm_fwd(p, p, p, 4, 4, 0, float('nan'), 0, p, p, p, None), 'eps')
  _refused(lib.trl_layer_norm_fwd(p, p, p, 4, 4, 0, 1e-5, 2, p, p, p, None), 'act')
  _refused(lib.trl_layer_norm_fwd(None, p, p, 4, 4, 0, 1e-5, 0, p, p, p, None), 'null')
  assert lib.trl_layer_norm_fwd(None, None, None, 0, 4, 0, 1e-5, 0, None, None, None, None) == 0
  _refused(lib.trl_layer_norm_bwd(p, p, p, p, p, p, 4, 4, 0, 0, p, p, p, None, None), 'workspace')
  _refused(lib.trl_layer_norm_bwd(p, p, p, p, None, p, 4, 4, 0, 0, p, p, p, p, None), 'null')
  assert lib.trl_layer_norm_bwd(p, p, p, p, p, p, 4, 4, 0, 0, None, None, None, None, None) == 0
  assert lib.trl_layer_norm_bwd_workspace_bytes(4, 4, 1) < 0
  for rows, width, dt in ((0, 1, 0), (1, 1, 2), (1 << 20, 64, 0), (1 << 20, 64, 2), (7, 100000, 3)):
    assert lib.trl_layer_norm_bwd_workspace_bytes(rows, width, dt) >= 8 * width


def test_dropout_entry_checks():
  lib = _lib.lib()
  p = 4096
  _refused(lib.trl_dropout(p, None, 4, 1, 0.5, 0, 0, None, p, None), 'dtype')
  _refused(lib.trl_dropout(p, None, -4, 0, 0.5, 0, 0, None, p, None), 'length')
  _refused(lib.trl_dropout(p, None, 1 << 40, 0, 0.5, 0, 0, None, p, None), 'length')
  for bad in (-0.1, 1.0, 1.5, float('nan')):
    _refused(lib.trl_dropout(p, None, 4, 0, bad, 0, 0, None, p, None), 'p must be')
  _refused(lib.trl_dropout(None, None, 4, 0, 0.5, 0, 0, None, p, None), 'null')
  assert lib.trl_dropout(None, None, 0, 0, 0.5, 0, 0, None, None, None) == 0
  _refused(lib.trl_next_call(p, p, None), 'one buffer')


def test_decay_attention_entry_checks():
  lib = _lib.lib()
  p = 4096
  st = (C.c_int64 * 9)(*([1] * 9))

  def fwd(T=4, N=2, H=1, dk=8, dv=8, dt=0, q=p, start_dtype=0, start=None, state_out=p, ws=None, decay=p):
    return lib.trl_decay_attention_fwd(q, p, p, st, decay, start, start_dtype, None, None, T, N, H, dk, dv, dt, 1.0, p,
                                       state_out, ws, None)

  def bwd(T=4, N=2, H=1, dk=8, dv=8, dt=0, q=p, dq=p, ws=None):
    return lib.trl_decay_attention_bwd(p, None, q, p, p, st, p, None, 0, None, None, T, N, H, dk, dv, dt, 1.0, dq, p, p, None,
                                       ws, None)

  def step(N=2, H=1, dk=8, dv=8, dt=0, state=p):
    return lib.trl_decay_attention_step(p, p, p, p, None, 0, state, N, H, dk, dv, dt, 1.0, p, p, None)

  for call in (fwd, bwd, step):
    _refused(call(dt=1), 'dtype')
    _refused(call(N=-1), 'bad shape')
    _refused(call(H=0), 'bad shape')
    _refused(call(dk=0), 'head sizes')
    _refused(call(dk=129), 'head sizes')
    _refused(call(dv=129), 'head sizes')
    _refused(call(N=1 << 22), 'too many')
    assert call(N=0) == 0
  for call in (fwd, bwd):
    _refused(call(T=-1), 'bad shape')
    _refused(call(T=1 << 30), 'too many')
    _refused(call(q=None), 'null')
    _refused(call(T=4096, N=1), 'workspace')
  _refused(fwd(start=p, start_dtype=2), 'start')
  _refused(fwd(state_out=None), 'null')
  _refused(fwd(decay=None), 'null')
  _refused(bwd(dq=None), 'null')
  _refused(step(state=None), 'null')
  ws = lib.trl_decay_attention_workspace_bytes
  assert ws(4, 2, 1, 8, 8, 0) == 0 and ws(16, 5000, 4, 64, 64, 1) == 0
  assert ws(8192, 1, 8, 64, 64, 0) > 0 and ws(8192, 1, 8, 64, 64, 1) == 2 * ws(8192, 1, 8, 64, 64, 0)
  assert ws(4, 2, 1, 8, 129, 0) < 0


def test_models_keep_the_reference_initialisation_without_the_new_layers():
  """Default networks have the parameters, names and draws that they had; with the layers, Linear weights keep theirs."""
  from torchrl_amd.contrib.models import DDPGCriticNet, QNet
  torch.manual_seed(3)
  a = QNet(4, 2)
  assert list(a.state_dict()) == ['net.%d.%s' % (i, n) for i in (0, 2, 4) for n in ('weight', 'bias')]
  torch.manual_seed(3)
  b = QNet(4, 2, layer_norm=True, dropout=0.1)
  assert torch.equal(a.net[0].weight, b.net[0].weight) and torch.equal(a.net[4].weight, b.net[8].weight)
  torch.manual_seed(3)
  c = DDPGCriticNet(4, 2, 16, layer_norm=True)
  assert [type(m).__name__ for m in c.net] == ['SkinnyLinear', 'LayerNorm', 'ReLU'] * 2 + ['SkinnyLinear']
  c.eval()
  assert c(torch.randn(5, 4), torch.randn(5, 2)).shape == (5, 1)


def test_controllers_act_on_the_cpu_with_the_new_layers():
  import numpy as np
  from torchrl_amd.contrib.controllers import DQNController
  ctl = DQNController(4, 2, device='cpu', hidden=16, layer_norm=True, dropout=0.2)
  assert len(ctl.act(np.zeros((3, 4), np.float32))) == 3
  with pytest.raises(_lib.TrlError):
    ctl.q_net.train()
    ctl.q_net(torch.zeros(3, 4))      # (training through dropout needs the device)


def test_module_arguments():
  from torchrl_amd.contrib.models import Dropout, MemoryBlock
  for bad in (-0.1, 1.0):
    with pytest.raises(ValueError):
      Dropout(bad)
  m = MemoryBlock(32, heads=4, head_size=16)
  assert m.decay.shape == (4,) and abs(float(m.decay[0]) - 0.875) < 1e-6 and m.initial_state(3).shape == (3, 4, 16, 16)
  assert sorted(m.state_dict()) == sorted(['norm.weight', 'norm.bias', 'qkv.weight', 'qkv.bias', 'out.weight', 'out.bias',
                                           'drop.calls', 'decay'])
  for bad in ([0.5], [0.5, 0.5, 0.5, 1.5], [0.5, 0.5, 0.5, float('nan')]):
    with pytest.raises(ValueError):
      MemoryBlock(32, heads=4, decay=bad)
  d = Dropout(0.5).eval()
  x = torch.randn(3)
  assert d(x) is x and torch.equal(d(x, residual=x), 2 * x)


def test_reference_generator_is_the_published_one():
  """Philox-4x32-10's known answers (Salmon et al., Parallel random numbers: as easy as 1, 2, 3, the counter-based
  generators' test vectors), through the bit that keeps dropout's counters apart."""
  import numpy as np

  def rounds(ctr, key):
    c, k = [np.array([v], dtype=np.uint64) for v in ctr], list(key)
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
      a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
      c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
      k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return [int(v[0]) for v in c]

  assert rounds([0] * 4, [0] * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
  assert rounds([0xffffffff] * 4, [0xffffffff] * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
  seed, call = 0x123456789abcdef0, 0x0fedcba987654321
  words = ref.philox_words(9, seed, call)
  for g in range(2):
    assert [int(w) for w in words[4 * g:4 * g + 4]] == rounds([0x87654321, 0x0fedcba9, g, 0x80000000], [0x9abcdef0, 0x12345678])


def test_memory_block_from_the_meta_device():
  import torch
  from torchrl_amd.contrib.models import MemoryBlock
  m = MemoryBlock(32, heads=4, head_size=16)
  values = {k: v.clone() for k, v in m.state_dict().items()}
  m = m.to('meta').to_empty(device='cpu')
  m.load_state_dict(values)
  assert m.decay.dtype == torch.float32 and torch.equal(m.decay, values['decay'])
