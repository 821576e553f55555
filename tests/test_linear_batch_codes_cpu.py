"""linear_batch and precompute_stage handed an activation that is in FP8 already, as float8_per_row Linears take it: one by one."""
import pytest
import torch
from torch import nn

from cache_dit_amd import nn as quantized
from cache_dit_amd import ops


@pytest.fixture
def pair(monkeypatch):
  seen = []

  def mm(codes, scales, *args, **kwargs):
    seen.append((codes, scales))
    return torch.zeros(2, 8)

  monkeypatch.setattr(ops, "float8_inference_scaled_mm", mm)
  pair = torch.zeros(2, 16).to(torch.float8_e4m3fn), torch.ones(2, 1)
  yield pair, seen


def linear():
  lin = nn.Linear(16, 8, dtype=torch.bfloat16)
  lin.__class__ = quantized.Fp8DynamicLinear
  lin.register_buffer("weight_scale", torch.ones(8, 1))
  lin.epilogue, lin._scale_mode_id = 0, 0
  return lin


def test_a_batch(pair):
  pair, seen = pair
  outs = quantized.linear_batch([(pair, [linear(), linear()]), (pair, [linear()])])
  assert [len(o) for o in outs] == [2, 1] and len(seen) == 3 and all(s[0] is pair[0] and s[1] is pair[1] for s in seen)


def test_a_stage_is_not_computed_ahead(pair):
  pair, seen = pair
  lin = linear()
  assert quantized.precompute_stage([(pair, [lin])]) is False and not seen and lin._precomputed is None
