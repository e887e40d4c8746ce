"""Dropout's probability at the end of its range: kept words are those of at least round(p 2^32), and above 1 - 2^-33 that is no
32-bit word any more (one value too many would be kept, and scaled by 1 / (1 - p))."""
import numpy as np
import pytest
import torch

from tests import layer_reference as ref
from torchrl_amd import _lib
from torchrl_amd import functional as F

TOP = 1.0 - 2.0 ** -33


def test_probabilities_that_no_word_stands_for_are_refused():
  from torchrl_amd.contrib.models import Dropout
  lib = _lib.lib()
  for p in (TOP, 1.0 - 1e-12, float(np.nextafter(1.0, 0.0)), 1.0):
    assert lib.trl_dropout(4096, None, 4, 0, p, 0, 0, None, 4096, None) == -1
    assert b'p must be' in lib.trl_last_error()
    with pytest.raises(ValueError, match='p must be'):
      Dropout(p)
  assert lib.trl_dropout(None, None, 0, 0, float(np.nextafter(TOP, 0.0)), 0, 0, None, None, None) == 0
  assert Dropout(1.0 - 2.0 ** -32).p < TOP


@pytest.mark.gpu
def test_the_highest_probability():
  """Its threshold is 2^32 - 1: of 2^22 elements none, or the few words of that value are kept, as the generator has them."""
  n, p = 1 << 22, 1.0 - 2.0 ** -32
  x = torch.ones(n, device='cuda')
  with pytest.raises(ValueError, match='p must be'):
    F.dropout(x, TOP, 5, 9)
  words = ref.philox_words(n, 5, 9)
  assert torch.equal(F.dropout(x, p, 5, 9).cpu(), torch.from_numpy(words == 2 ** 32 - 1).float() * 2.0 ** 32)
  # a threshold that the generator's first words lie on both sides of, and on
  t = int(np.sort(words)[n // 2])
  kept = F.dropout(x, t / 2 ** 32, 5, 9).cpu() != 0
  assert torch.equal(kept, torch.from_numpy(words >= t))
