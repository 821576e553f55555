"""A row's result of lora_add does not depend on which adapters the rows beside it name, whichever kernel takes them."""
import pytest
import torch

from test_gpu_lora import make, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ranks", [[16, 16], [48, 20], [64, 64], [128, 70], [256, 200]])
@pytest.mark.parametrize("N,K", [(264, 256), (131, 257)])
@pytest.mark.parametrize("M,fp8", [(40, False), (900, True), (5000, False), (5000, True)])
def test_neighbours_with_other_adapters(ops, M, fp8, N, K, ranks):  # noqa: F811
  a, g = make(M, N, K, ranks, fp8, seed=N)
  a["base"] = a["base"] * 0.01  # (what base adds must not hide the sums' last bits)
  d = {n: None if t is None else t.cuda() for n, t in a.items()}

  def run(ids):
    return ops.lora_add(d["base"], d["x"], d["down"], d["up"], ids.cuda(), scale=d["scale"], rank=d["rank"], x_scale=d["x_scale"])

  alone = run(torch.zeros(M, dtype=torch.int32))
  for ids in (torch.arange(M, dtype=torch.int32) % 7 == 3, torch.arange(M, dtype=torch.int32) // 40 % 2 == 1, torch.rand(M, generator=g) < 0.5):
    for other in (1, -1):
      mixed = torch.where(ids, other, 0)
      same = (~ids).cuda()
      assert torch.equal(run(mixed)[same], alone[same])
