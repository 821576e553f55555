"""Adapters that come, change and go beside Linears of a compiled graph."""
import pytest
import torch
from torch import nn

from test_gpu_adapters import BF16, TYPES, bank, cd, linear, no_grad  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant_type", TYPES)
def test_attached_and_taken_away_behind_compilation(cd, quant_type):  # noqa: F811
  class Net(nn.Module):

    def __init__(self):
      super().__init__()
      self.lin = linear(quant_type, gelu=True)

    def forward(self, x):
      return self.lin(x) + 1

  torch._dynamo.reset()
  net = Net()
  compiled = torch.compile(net, fullgraph=True, backend="eager")
  x = torch.randn(3, 7, 256, device="cuda").to(BF16)
  own = net(x)
  assert torch.equal(compiled(x), own)
  cd.attach_lora_(net.lin, bank(cd))
  assert torch.equal(compiled(x), own)
  ids = torch.tensor([1, -1, 0], dtype=torch.int32).cuda()
  cd.set_lora_ids(net, ids)
  with_adapters = net(x)
  assert torch.equal(compiled(x), with_adapters) and not torch.equal(with_adapters, own)
  ids.copy_(ids.flip(0))
  assert torch.equal(compiled(x), net(x)) and not torch.equal(compiled(x), with_adapters)
  cd.set_lora_ids(net, None)
  assert torch.equal(compiled(x), own)
  cd.set_lora_ids(net, 1)
  assert torch.equal(compiled(x), net(x)) and not torch.equal(compiled(x), own)
  assert cd.detach_lora_(net) == 1
  assert torch.equal(compiled(x), own)
