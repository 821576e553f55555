"""The 4-bit products' tiles where a workgroup takes several of them, one after the other: every output of every tile, bit for bit.

Operands are small whole numbers under powers of two (0, .5, 1 and signs under 2^-2 to 1): partial sums are multiples of 1/64 and
below 2^11 in magnitude, which fp32 holds in any order of addition."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  from cache_dit_amd import ops
  return ops


@pytest.fixture
def variant(ops):
  from cache_dit_amd import _native
  yield _native.set_gemm_variant
  _native.set_gemm_variant(-1)


def draw(R, K, g):
  """(codes, scales, values in fp32)"""
  table = torch.tensor([0, 1, 2, 8, 9, 10], dtype=torch.uint8, device="cuda")
  c = table[torch.randint(0, 6, (R, K), generator=g, device="cuda")]
  s = torch.full((R, 4 * -(-K // 128)), 127, dtype=torch.uint8, device="cuda")
  s[:, :K // 32] = torch.randint(125, 128, (R, K // 32), generator=g, device="cuda").to(torch.uint8)
  value = torch.tensor([0, .5, 1, 0, 0, 0, 0, 0, 0, -.5, -1], device="cuda")
  v = value[c.int()].view(R, K // 32, 32) * torch.exp2(s[:, :K // 32].float() - 127)[..., None]
  return c[:, 0::2] | (c[:, 1::2] << 4), s, v.view(R, K)


#: variant: rows and columns of its tile, workgroups a CU holds, M and N that give more tiles than that on 256 CUs, no whole
#: multiple of it, the last row and column of tiles ragged (N odd for one of them)
TILES = {1: (256, 256, 1, 4200, 4500), 5: (128, 256, 1, 4200, 2300), 6: (256, 128, 1, 2300, 4203), 2: (128, 128, 2, 3000, 2901),
         3: (64, 128, 2, 1500, 2900), 7: (128, 64, 2, 3000, 1470), 4: (64, 64, 2, 1500, 4400), 8: (32, 64, 3, 900, 1801)}


@pytest.mark.parametrize("v", sorted(TILES))
@pytest.mark.parametrize("K", [96, 992, 1024, 1248, 1696])  # fewer steps of 256 than a tile's least; 4, part of one and whole; 5; 7
def test_every_output_of_several_tiles_a_workgroup(ops, variant, v, K):
  bm, bn, per_cu, M, N = TILES[v]
  cus = torch.cuda.get_device_properties(0).multi_processor_count
  tiles = -(-M // bm) * -(-N // bn)
  assert cus > 256 or (tiles > cus * per_cu and tiles % (cus * per_cu))
  g = torch.Generator(device="cuda").manual_seed(1000 * v + K)
  a, a_s, av = draw(M, K, g)
  w, w_s, wv = draw(N, K, g)
  bias = torch.randint(-32, 33, (N, ), generator=g, device="cuda").float()
  want = av @ wv.t() + bias
  assert want.abs().max() < 2**11
  variant(v)
  for out in (F32, BF16, F16):
    got = ops.mxfp4_mm(a, a_s, w, w_s, out, bias=bias.to(out))
    assert torch.equal(got, want.to(out)), out
  x = av.to(BF16)
  assert torch.equal(x.float(), av)
  assert torch.equal(ops.w4a16_mm(x, w, w_s, bias.to(BF16)), want.to(BF16))


@pytest.mark.parametrize("M,N,K", [(8200, 4500, 352), (16400, 1000, 672), (4608, 5120, 1312)])
def test_the_automatic_choice_of_several_rounds(ops, M, N, K):
  g = torch.Generator(device="cuda").manual_seed(K)
  a, a_s, av = draw(M, K, g)
  w, w_s, wv = draw(N, K, g)
  want = (av @ wv.t()).to(BF16)
  assert torch.equal(ops.mxfp4_mm(a, a_s, w, w_s, BF16), want)
  assert torch.equal(ops.w4a16_mm(av.to(BF16), w, w_s), want)
