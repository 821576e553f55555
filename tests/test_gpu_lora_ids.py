"""lora_add with one number for all rows, or one request, on what is not laid out as the kernels take it."""
import pytest
import torch
from torch import nn

from test_gpu_lora import BF16, make, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ids", [torch.tensor(1), torch.tensor([1, 0]), torch.tensor(1, dtype=torch.int16), torch.tensor([0, 1], dtype=torch.int8)])
@pytest.mark.parametrize("S", [9, 1500])
def test_ids_with_parts_of_a_joint_sequence(ops, S, ids):  # noqa: F811
  a, _ = make(2 * S, 40, 64, [16, 5], seed=S)
  d = {n: None if t is None else t.cuda() for n, t in a.items()}
  base, x, ids = d["base"].view(2, S, 40), d["x"].view(2, S, 64), ids.cuda()
  want = ops.lora_add(base, x, d["down"], d["up"], ids.int(), scale=d["scale"], rank=d["rank"])
  joint_x, joint = torch.cat((x, x), 1), torch.cat((base, base), 1)
  for b, v, scale in ((base, joint_x[:, S:], d["scale"]), (joint[:, :S], x, d["scale"]), (joint[:, S:], joint_x[:, :S], d["scale"]),
                      (base, x, d["scale"].double())):
    assert torch.equal(ops.lora_add(b, v, d["down"], d["up"], ids, scale=scale, rank=d["rank"]), want)
  one = ops.lora_add(joint[:1, S:], joint_x[:1, S:, :], d["down"], d["up"], ids.reshape(-1)[:1].clone(), scale=d["scale"], rank=d["rank"])
  assert torch.equal(one[0], ops.lora_add(base[0], x[0], d["down"], d["up"], ids.reshape(-1)[0].int(), scale=d["scale"], rank=d["rank"]))


def test_one_adapter_for_a_whole_model(ops):  # noqa: F811
  """set_lora_ids(module, number), then a slice of a joint sequence."""
  import cache_dit_amd as cd
  from cache_dit_amd.nn import convert_linear_
  torch.manual_seed(0)
  lin = convert_linear_(nn.Linear(64, 48, dtype=BF16, device="cuda"), "float8_per_row")
  cd.attach_lora_(lin, cd.LoraAdapters([(torch.randn(4, 64).cuda(), torch.randn(48, 4).cuda())]))
  cd.set_lora_ids(lin, 0)
  joint = torch.randn(2, 20, 64, device="cuda").to(BF16)
  with torch.no_grad():
    assert torch.equal(lin(joint[:, 5:]), lin(joint[:, 5:].contiguous()))
