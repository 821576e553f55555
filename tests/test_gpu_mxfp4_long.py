"""The 4-bit products for few rows at the longest K they take: sizes of all of K that pass 32 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what,M,K", [("w4a16", 16, 140000032), ("w4a4", 16, 250000032), ("codes", 16, 268435424)])
def test_long_k(what, M, K):
  """Whole numbers under powers of two: partial sums are multiples of 1/8, a random walk of a few thousand (under 2^21, so fp32
  holds each of them), and the result has to be equal."""
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  from cache_dit_amd import ops
  N = 16
  g = torch.Generator(device="cuda").manual_seed(K)
  # 0, .5, 1, -.5, -1 under scales of 2^-2 to 1
  table = torch.tensor([0, 1, 2, 9, 10], dtype=torch.uint8, device="cuda")
  codes = torch.empty(N, K // 2, dtype=torch.uint8, device="cuda")
  scales = torch.full((N, 4 * -(-K // 128)), 127, dtype=torch.uint8, device="cuda")
  x = torch.empty(M, K, dtype=torch.bfloat16, device="cuda")
  want = torch.zeros(M, N, dtype=torch.float64, device="cuda")
  value = torch.tensor([0, .5, 1, 0, 0, 0, 0, 0, 0, -.5, -1], dtype=torch.float64, device="cuda")
  step = 1 << 22
  for at in range(0, K, step):
    n = min(step, K - at)
    pick = table[torch.randint(0, 5, (N, n), generator=g, device="cuda", dtype=torch.int32)]
    codes[:, at // 2:(at + n) // 2] = pick[:, 0::2] | (pick[:, 1::2] << 4)
    e = torch.randint(125, 128, (N, n // 32), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    scales[:, at // 32:(at + n) // 32] = e
    x[:, at:at + n] = torch.randint(-1, 2, (M, n), generator=g, device="cuda", dtype=torch.int8)
    w = (value[pick.int()].view(N, n // 32, 32) * torch.exp2(e.double() - 127)[..., None]).view(N, n)
    want += x[:, at:at + n].double() @ w.t()
  bias = torch.arange(N, device="cuda").to(torch.bfloat16)
  want += bias.double()
  if what == "w4a16":
    assert torch.equal(ops.w4a16_mm(x, codes, scales, bias), want.to(torch.bfloat16))
  elif what == "w4a4":
    assert torch.equal(ops.mxfp4_linear(x, codes, scales, bias), want.to(torch.bfloat16))
  else:
    assert torch.equal(ops.mxfp4_mm(*ops.mxfp4_quant(x), codes, scales, torch.float32, bias.float()), want.float())
