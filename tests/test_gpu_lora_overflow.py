"""lora_add where x down^T leaves fp32: an infinity of one rank is an infinity in the result, in that row alone."""
import pytest
import torch

from test_gpu_lora import make, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [20, 2500])
@pytest.mark.parametrize("N", [136, 131])
@pytest.mark.parametrize("R", [16, 32, 48, 80, 144, 176])
@pytest.mark.parametrize("mixed", [False, True])
def test_one_rank_overflows(ops, M, N, R, mixed):  # noqa: F811
  """Row 3 has 6e38 for the last rank, which fp32 does not hold; its results are infinities of up's sign."""
  a, g = make(M, N, 64, [R, R], seed=R)
  a["x"][3], a["x"][3, 0] = 0, 2.0
  a["down"][:, R - 1, 0], a["scale"] = 3e38, torch.ones(2)
  others = torch.arange(M) != 3
  a["x"][others, 0] = 0
  sign = torch.where(torch.arange(N) % 3 == 0, -1.0, 1.0)
  a["up"][:, :, R - 1] = sign * a["up"][:, :, R - 1].abs().clamp(min=0.01)
  d = {n: None if t is None else t.cuda() for n, t in a.items()}
  ids = torch.arange(M) % 2 if mixed else torch.ones(M)
  got = ops.lora_add(d["base"], d["x"], d["down"], d["up"], ids.int().cuda(), scale=d["scale"], rank=d["rank"]).cpu()
  assert torch.equal(got[3].float(), sign * float("inf")) and got[others].isfinite().all()
