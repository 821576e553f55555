"""Adapters beside Linears whose activation has FP8 codes only (ln_modulate_quant(materialize=False))."""
import pytest
import torch
from torch import nn

from test_gpu_adapters import BF16, bank, cd, linear, no_grad  # noqa: F401

pytestmark = pytest.mark.gpu


def activation(cd, seed=3):  # noqa: F811
  """The activation without values, and its codes and scales."""
  g = torch.Generator().manual_seed(seed)
  x, shift, scale = (torch.randn(*s, 256, generator=g).to(BF16).cuda() for s in ((2, 21), (2, 1), (2, 1)))
  y = cd.ops.ln_modulate_quant(x, shift, scale, materialize=False)
  assert cd.ops.is_codes_only(y)
  return y, cd.ops.fp8_rowwise_quant(cd.ops.ln_modulate_quant(x, shift, scale))


def test_adapters_take_the_codes_too(cd):  # noqa: F811
  """One by one, as siblings, in a batch and in a stage: what the Linears give on the codes themselves."""
  lins = [linear("float8_per_row", seed=i, gelu=i == 1) for i in range(3)]
  for i, lin in enumerate(lins):
    cd.attach_lora_(lin, bank(cd, seed=i))
    cd.set_lora_ids(lin, torch.tensor([1, 0]).cuda())
  holder = nn.ModuleList(lins)
  _, codes = activation(cd)
  want = [lin(codes) for lin in lins]
  cd.share_activation_quant_(holder)

  def same(got):
    assert all(torch.equal(g, w) for g, w in zip(got, want))

  y, _ = activation(cd)
  same([lin(y) for lin in lins])
  same([lin(y.view(42, 256).view(2, 21, 256)) for lin in lins])
  y, _ = activation(cd)
  same(cd.linear_batch([(y, lins)])[0])
  same(cd.linear_batch([(codes, lins)])[0])
  y, _ = activation(cd)
  assert cd.precompute_stage([(y, lins)])
  same([lin(y) for lin in lins])
  plain = torch.randn(2, 21, 256, device="cuda").to(BF16)
  assert cd.group_sibling_linears_(holder, run=lambda: [lin(plain) for lin in lins]) == 1
  y, _ = activation(cd)
  same([lin(y) for lin in lins])


def test_without_the_codes_it_is_refused(cd):  # noqa: F811
  lin = linear("float8_per_row")
  cd.attach_lora_(lin, bank(cd))
  cd.set_lora_ids(lin, 0)
  y, _ = activation(cd)
  with pytest.raises(RuntimeError, match="materialize=True"):
    lin(y)  # shares no codes
