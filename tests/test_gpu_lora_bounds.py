"""lora_add where a tile's buffers end early: last tiles of one row, columns that end just behind a tile, ranks of one row, codes whose last
step is mostly behind their row. What lies next to the tensors is NaN and must not come in."""
import pytest
import torch

from oracle import block_oracle as bo
from test_gpu_lora import BF16, check, make, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def inside(t, dev="cuda"):
  """t with NaN in front of it and behind it."""
  pad = 64 * 1024
  wide = torch.full((t.numel() + 2 * pad, ), float("nan"), dtype=torch.float32).to(t.dtype).to(dev)
  wide[pad:pad + t.numel()] = t.reshape(-1).to(dev)
  return wide[pad:pad + t.numel()].view(t.shape)


@pytest.mark.parametrize("ranks", [[1], [65, 1], [129, 1]])
@pytest.mark.parametrize("K,fp8", [(144, True), (160, True), (176, True), (136, False)])
@pytest.mark.parametrize("N", [129, 130, 131, 136])
@pytest.mark.parametrize("requests,rows", [(1, 2049), (33, 65), (17, 129)])
def test_tiles_that_end_early(ops, requests, rows, N, K, fp8, ranks):  # noqa: F811
  M = requests * rows
  a, g = make(M, N, K, ranks, fp8, seed=M + N + K)
  ids = torch.randint(0, len(ranks), (requests, ), generator=g)
  d = {n: None if t is None else inside(t) if n in ("base", "x", "down", "up") else t.cuda() for n, t in a.items()}
  got = ops.lora_add(d["base"].view(requests, rows, N), d["x"].view(requests, rows, K), d["down"], d["up"], ids.cuda(), scale=d["scale"],
                     rank=d["rank"], x_scale=d["x_scale"]).view(M, N)
  pick = torch.cat((torch.arange(0, M, 61), torch.arange(rows - 1, M, rows)))
  want, mag = bo.lora(a["base"][pick], a["x"][pick], a["down"], a["up"], ids.repeat_interleave(rows)[pick], a["scale"], a["rank"],
                      a["x_scale"][pick] if fp8 else None)
  check(got[pick.cuda()], want, mag, K, a["down"].shape[1])
  assert got.isfinite().all()
