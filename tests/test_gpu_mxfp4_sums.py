"""What the w4a4 products' sums in fp32 keep: small products next to a large bias, a large running sum, a large product."""
import pytest
import torch

from oracle import mxfp4_oracle as mo

pytestmark = pytest.mark.gpu
F32 = torch.float32
VARIANTS = [-1, 0, 1, 2, 3, 4, 5, 6, 7, 8, 100]


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


def matrix(R, K, codes, scales=()):
  """R equal rows: codes at some k, scale bytes of some blocks, zeros under 1 elsewhere."""
  c = torch.zeros(R, K, dtype=torch.uint8)
  for k, v in codes:
    c[:, k] = v
  s = torch.full((R, mo.scale_bytes(K)), 127, dtype=torch.uint8)
  for b, v in scales:
    s[:, b] = v
  return (c[:, 0::2] | (c[:, 1::2] << 4)).cuda(), s.cuda()


@pytest.mark.parametrize("v", VARIANTS)
@pytest.mark.parametrize("M", [9, 300])
def test_small_products_next_to_large_addends(ops, variant, v, M):
  """2^22 and 1.5: fp32 holds the sum. Beside the bias, in a step before and behind, and in the same instruction."""
  N, one, three_halves = 200, 2, 3
  variant(v)
  want = 2.0**22 + 1.5

  def product(a, w, bias=None):
    got = ops.mxfp4_mm(*a, *w, F32, bias=bias)
    assert (got == want).all(), torch.unique(got)[:4].tolist()

  large = 127 + 11  # 2^11 on either side
  product(matrix(M, 128, [(0, one)]), matrix(N, 128, [(0, three_halves)]), torch.full((N, ), 2.0**22, device="cuda"))
  product(matrix(M, 1024, [(0, one), (900, one)], [(0, large)]), matrix(N, 1024, [(0, one), (900, three_halves)], [(0, large)]))
  product(matrix(M, 1024, [(0, one), (900, one)], [(28, large)]), matrix(N, 1024, [(0, three_halves), (900, one)], [(28, large)]))
  product(matrix(M, 64, [(0, one), (33, one)], [(0, large)]), matrix(N, 64, [(0, one), (33, three_halves)], [(0, large)]))
  # 96 products of 1/64, 28 places below the largest
  small = [(k, 1) for k in range(32, 128)]
  scales = [(0, large)] + [(b, 125) for b in (1, 2, 3)]
  product(matrix(M, 128, [(0, one)] + small, scales), matrix(N, 128, [(0, one)] + small, scales))


@pytest.mark.parametrize("v", VARIANTS)
@pytest.mark.parametrize("M,N,K", [(7, 130, 2208), (300, 260, 128), (300, 260, 2208), (300, 260, 5120)])
def test_sums_of_very_different_products(ops, variant, v, M, N, K):
  """Blocks 2^24 apart, in fp32. An instruction sums 64 (or 128) products and the sum so far. It keeps what lies 28 places below
  the largest of them (the test above), so each of the 65 (129) addends loses less than 2^-28 of it, and rounds to fp32, at most
  2^-23 of it: per 64 products (65 / 2^28 + 2^-23) = 3.7e-7 of the largest, which the sum of all magnitudes bounds. Joining the
  partial sums of up to eight wavefronts, two each, and the bias: 17 roundings of 2^-24."""
  g = torch.Generator().manual_seed(M + N + K)

  def wide(R):
    return torch.randn(R, K, generator=g) * torch.exp2(torch.randint(-12, 13, (R, K // 32, 1), generator=g).float()).expand(
        -1, -1, 32).reshape(R, K)

  a, w = mo.quantize(wide(M)), mo.quantize(wide(N))
  bias = torch.randn(N, generator=g) * 100
  want, sums = mo.product(mo.dequantize(*a).cuda(), mo.dequantize(*w).cuda(), bias.cuda())
  variant(v)
  got = ops.mxfp4_mm(*(t.cuda() for t in (*a, *w)), F32, bias=bias.cuda())
  limit = (-(-K // 64) * 3.7e-7 + 17 * 2.0**-24) * (sums + bias.cuda().abs())
  err = (got.double() - want).abs()
  assert (err <= limit).all(), float((err / limit).max())
