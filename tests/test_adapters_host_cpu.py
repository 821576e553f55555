"""A converted Linear without adapters does not look for any: its call is bound by the host."""
import pytest
import torch
from torch import nn

from cache_dit_amd import mxfp4, ops
from cache_dit_amd import nn as quantized


@pytest.fixture
def calls(monkeypatch):
  """The operators' stand-ins; looking for adapters is an error."""
  out = torch.zeros(2, 8)

  def stand_in(*args, **kwargs):
    return out

  for module, names in ((ops, ("linear_w8a8_op", "w8a16_mm_op", "float8_inference_scaled_mm", "linear_w8a8_cat2_op")),
                        (mxfp4, ("mxfp4_linear_op", "w4a16_mm_op", "mxfp4_mm"))):
    for name in names:
      monkeypatch.setattr(module, name, stand_in)

  def looked(self, *args):
    raise AssertionError("looked for adapters")

  for name in ("_adapters", "_own_epilogue", "_with_adapters"):
    monkeypatch.setattr(quantized._Fp8LinearBase, name, looked)
  monkeypatch.setattr(quantized._Fp8LinearBase, "_check_input", lambda self, x: None)
  return out


@pytest.mark.parametrize("cls", ["Fp8DynamicLinear", "Fp8DynamicLinearPerTensor", "Fp8WeightOnlyLinear", "Mxfp4Linear", "Mxfp4WeightOnlyLinear"])
def test_no_adapters_cost_nothing(calls, cls):
  lin = nn.Linear(16, 8, dtype=torch.bfloat16)
  lin.__class__ = getattr(quantized, cls)
  lin.register_buffer("weight_scale", torch.ones(8, 1))
  lin.epilogue, lin._scale_mode_id = 0, 0
  assert lin(torch.zeros(2, 16)) is calls
  if cls in ("Fp8DynamicLinear", "Mxfp4Linear"):
    assert lin((torch.zeros(2, 16), torch.ones(2, 1))) is calls
