"""linear_on_cat on a source that has FP8 codes only: there are no values to concatenate."""
import pytest
import torch
from torch import nn

from test_gpu_adapters import BF16, bank, cd, linear, no_grad  # noqa: F401
from test_gpu_adapters_codes import activation

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [True, False])
def test_a_source_without_values_is_refused(cd, first):  # noqa: F811
  y, _ = activation(cd)
  other = torch.randn(2, 21, 128, device="cuda").to(BF16)
  xs = [y, other] if first else [other, y]
  lin = linear("float8_per_row", K=384)
  with pytest.raises(RuntimeError, match="materialize=True"):
    cd.linear_on_cat(lin, xs)
  cd.attach_lora_(lin, bank(cd, K=384))
  cd.set_lora_ids(lin, 0)
  for module in (lin, linear("float8_weight_only", K=384), nn.Linear(384, 32, dtype=BF16, device="cuda")):
    with pytest.raises(RuntimeError, match="materialize=True"):
      cd.linear_on_cat(module, xs)
