"""YaRN's frequencies where its ramp ends behind the last pair: long original lengths, or a large number of turns for its lower end."""
import math

import pytest
import torch


def published(rot, theta, factor, length, low, high):
  """The method as published, index by index: the ramp runs from the floor to the ceiling of the indices that turn `high` and `low` times,
  kept within 0 and the number of dimensions less 1; the share kept falls along it."""

  def index_of(turns):
    return rot * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(theta))

  first, last = max(math.floor(index_of(high)), 0), min(math.ceil(index_of(low)), rot - 1)
  out = []
  for i in range(rot // 2):
    ramp = min(max((i - first) / (last - first), 0.0), 1.0)
    f = theta**(-2 * i / rot)
    out.append(f / factor * ramp + f * (1 - ramp))
  return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("rot,theta,factor,length,low,high",
                         [(128, 1e4, 4.0, 4096, 1.0, 32.0), (128, 5e5, 8.0, 8192, 1.0, 32.0), (128, 1e4, 4.0, 65536, 1.0, 32.0),
                          (64, 1e4, 16.0, 1 << 20, 1.0, 32.0), (128, 1e4, 4.0, 4096, 0.01, 0.5), (20, 1e4, 2.0, 131072, 1.0, 32.0)])
def test_yarn_is_the_published_ramp(rot, theta, factor, length, low, high):
  from cache_dit_amd import ops
  got, scale = ops.rotary_frequencies(rot, theta, scaling="yarn", factor=factor, original_length=length, low=low, high=high, device="cpu")
  assert torch.allclose(got, published(rot, theta, factor, length, low, high), rtol=1e-13, atol=0)
  assert scale == 0.1 * math.log(factor) + 1
