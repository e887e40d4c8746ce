"""Layer norm at the ends of its range of values: rows far from zero in the lanes that a row does not fill."""
import pytest
import torch

from torchrl_amd import functional as F

pytestmark = pytest.mark.gpu
DEV = 'cuda'


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('relu', [False, True])
@pytest.mark.parametrize('width', [1, 3, 7, 9, 40, 65, 200, 257, 520, 1030, 2100, 4104, 20000])
@pytest.mark.parametrize('value,eps', [(2.0 ** 100, 1.2e-38), (-2.0 ** 120, 1e-5)])
def test_large_equal_values_have_finite_gradients(width, value, eps, relu, dtype):
  """x = value everywhere: (x - mean) = 0, y = b, dx = r (h - mean(h)) with r = eps^-1/2 -- while (0 - value) r is not finite.
  Every sum of a row's values that the kernel may make is a small multiple of a power of two, so the mean is the value."""
  g = torch.Generator().manual_seed(width)
  rows = 9
  if width * abs(value) > 2.0 ** 127:
    value = value / 2.0 ** 14
    eps = max(eps / 2.0 ** 28, 1.2e-38)
  x = torch.full((rows, width), value).to(dtype).to(DEV).requires_grad_(True)
  w, b = torch.randn(width, generator=g), torch.randn(width, generator=g)
  gy = torch.randn(rows, width, generator=g).to(dtype)
  wd, bd = w.to(DEV).requires_grad_(True), b.to(DEV).requires_grad_(True)
  y = F.layer_norm(x, wd, bd, eps=eps, relu=relu)
  assert torch.equal(y.float().cpu(), (b.clamp_min(0) if relu else b).to(dtype).float().expand(rows, width))
  dx, dw, db = torch.autograd.grad(y, [x, wd, bd], gy.to(DEV))
  r = float(torch.tensor(eps, dtype=torch.float32).double()) ** -0.5
  t = gy.double() * ((b > 0) if relu else torch.ones(width, dtype=torch.bool))
  h = t * w.double()
  want = r * (h - h.mean(1, keepdim=True))
  size = h.abs() + h.abs().mean(1, keepdim=True)
  # a row's sum has up to 80 + width / 256 additions, r and the products a few roundings; then the result's own
  bound = (80 + width / 256 + 8) * 2.0 ** -24 * r * size + torch.finfo(dtype).eps / 2 * want.abs()
  assert bool(((dx.double().cpu() - want).abs() <= bound).all())
  assert not dw.any()
  assert bool(((db.double().cpu() - t.sum(0)).abs() <= rows * 2.0 ** -24 * t.abs().sum(0)).all())
