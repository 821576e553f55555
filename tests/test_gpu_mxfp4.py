"""MXFP4 on the GPU: quantizer and inverse bit for bit, both products against 64 bits."""
import pytest
import torch

from oracle import mxfp4_oracle as mo

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  from cache_dit_amd import ops
  return ops


def rows(M, K, dtype, seed=0):
  """Blocks of very different size, with rows of the values that matter to a rounding."""
  g = torch.Generator().manual_seed(seed)
  x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-12, 13, (M, K // 32, 1), generator=g).float()
                                                    ).expand(-1, -1, 32).reshape(M, K)
  special = torch.tensor([0.0, -0.0, .25, -.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.9, 7.0, -7.0, 4.0, 0.125])
  if M > 1:
    x[1] = special.repeat(K // 16) * 2.0**-3  # ties of the grid, block maxima of 7/8 and around
  if M > 2:
    x[2] = 0
    x[2, :32] = torch.finfo(dtype).tiny / 4  # subnormal in every type
    x[2, -32:] = torch.finfo(dtype).max
  return x.to(dtype)


def same(got, want):
  codes, scales = (t.cpu() for t in got)
  assert torch.equal(scales, want[1])
  assert torch.equal(codes, want[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 32), (3, 96), (5, 160), (77, 4096), (513, 32), (7, 2048), (3, 8192), (3, 16416)])
def test_quantizer_is_exact(ops, dtype, M, K):
  x = rows(M, K, dtype)
  codes, scales = ops.mxfp4_quant(x.cuda())
  assert codes.shape == (M, K // 2) and scales.shape == (M, mo.scale_bytes(K))
  want = mo.quantize(x)
  same((codes, scales), want)
  v = mo.dequantize(*want)
  for out in DTYPES:
    assert torch.equal(ops.mxfp4_dequant(codes, scales, out).cpu(), v.to(out)), out


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_not_finite(ops, dtype):
  x = rows(4, 128, dtype)
  x[0, 5], x[1, 40], x[3, 127] = float("inf"), float("nan"), float("-inf")
  codes, scales = ops.mxfp4_quant(x.cuda())
  same((codes, scales), mo.quantize(x))
  assert scales.cpu()[0, 0] == 255 and scales.cpu()[1, 1] == 255 and scales.cpu()[3, 3] == 255
  v = ops.mxfp4_dequant(codes, scales, torch.float32).cpu()  # (fp16's largest block is beyond fp16)
  assert v[0, :32].isnan().all() and v[1, 32:64].isnan().all() and v[3, 96:].isnan().all()
  assert v[0, 32:].isfinite().all() and v[2].isfinite().all()


def test_every_code_and_scale(ops):
  """All pairs of codes under every scale byte, in fp32 and bf16 (2^-127 times half is the smallest)."""
  codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)  # K = 512
  scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16)
  v = mo.dequantize(codes, scales)
  for out in (torch.float32, torch.bfloat16):
    got = ops.mxfp4_dequant(codes.cuda(), scales.cuda(), out).cpu()
    assert torch.equal(got.nan_to_num(7e7), v.to(out).nan_to_num(7e7)), out


def test_layouts_of_the_quantizer(ops):
  x = rows(24, 256, torch.bfloat16).cuda()
  want = mo.quantize(x.cpu())
  wide = torch.zeros(24, 320, dtype=torch.bfloat16, device="cuda")
  wide[:, 64:] = x
  same(ops.mxfp4_quant(wide[:, 64:]), want)  # a row stride
  odd = torch.zeros(24 * 256 + 1, dtype=torch.bfloat16, device="cuda")
  odd[1:] = x.reshape(-1)
  same(ops.mxfp4_quant(odd[1:].view(24, 256)), want)  # rows off 16 bytes
  same(ops.mxfp4_quant(x.t().contiguous().t()), want)  # a last stride that is not 1
  c, s = ops.mxfp4_quant(torch.cat((x, x)).view(2, 24, 256)[:, 8:])  # a slice of each batch entry
  assert c.shape == (2, 16, 128) and s.shape == (2, 16, 8)
  same((c[1], s[1]), (want[0][8:], want[1][8:]))
  c, s = ops.mxfp4_quant(x[3])
  assert c.shape == (128, ) and s.shape == (8, )
  same((c[None], s[None]), (want[0][3:4], want[1][3:4]))
  padded = torch.zeros(24, 64 * 3, dtype=torch.uint8, device="cuda")
  padded[:, 4:132] = want[0].cuda()
  got = ops.mxfp4_dequant(padded[:, 4:132], want[1].cuda())
  assert torch.equal(got.cpu(), mo.dequantize(*want).to(torch.bfloat16))
  for shape in ((0, 64), (2, 0, 64), (3, 0)):
    c, s = ops.mxfp4_quant(torch.empty(shape, dtype=torch.bfloat16, device="cuda"))
    assert c.shape == (*shape[:-1], shape[-1] // 2) and s.shape == (*shape[:-1], mo.scale_bytes(shape[-1]))
    assert ops.mxfp4_dequant(c, s).shape == shape


# ------------------------------------------------------------------------------------ products

#: M, N, K: one row to many, N odd and whole, K of whole steps and not, tiles' edges
SHAPES = [(1, 16, 32), (1, 1, 128), (1, 5120, 4096), (2, 33, 96), (15, 200, 1312), (16, 1024, 2048), (17, 48, 256),
          (33, 127, 544), (64, 256, 512), (77, 640, 1024), (129, 257, 160), (255, 384, 2208), (256, 256, 256),
          (300, 1001, 4128), (512, 768, 768), (1000, 2000, 1056), (2049, 520, 5120), (4608, 2560, 640)]


def operands(M, N, K, seed=0):
  g = torch.Generator().manual_seed(seed + M + 3 * N + 7 * K)
  x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))
  x[:, torch.randint(0, K, (max(1, K // 500), ), generator=g)] *= 20
  w = torch.randn(N, K, generator=g) * 0.05 * torch.exp(torch.randn(N, 1, generator=g))
  bias = torch.randn(N, generator=g) * 0.1
  return x.to(torch.bfloat16), mo.quantize(w), bias.to(torch.bfloat16)


def check(got, want, sums, dtype, gelu=False):
  """One rounding to the type (half a step, eps/2 relative) and the sum's own error. The matrix instruction for 4- and
  8-bit operands drops bits of an addend 13 places below the largest product of its sum, i.e. at most 2^-13 of
  it, and an instruction sums 128 and the sum so far; the largest products of all instructions are at most the sum of the
  magnitudes, so 2^-12 of that holds for addends that err to either side (64 of one sign in the mean: 2^-13 * 129 / 64). GELU has
  slopes up to 1.13."""
  got, want, sums = got.double().cpu(), want.cpu(), sums.cpu()
  limit = torch.finfo(dtype).eps / 2 * want.abs() + 1.2 * 2.0**-12 * sums + 1e-6
  if gelu:
    limit = limit + 2e-6 * want.abs()  # hardware exp2 and reciprocal, an ulp of fp32 each, and the folded constants
  bad = (got - want).abs() > limit
  assert not bad.any(), (int(bad.sum()), float((got - want).abs().max()), bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_against_64_bits(ops, M, N, K):
  x, w, bias = operands(M, N, K)
  got = ops.mxfp4_linear(x.cuda(), w[0].cuda(), w[1].cuda(), bias.cuda())
  assert got.shape == (M, N) and got.dtype == torch.bfloat16
  a = mo.dequantize(*mo.quantize(x)).cuda()
  check(got, *mo.product(a, mo.dequantize(*w).cuda(), bias.cuda()), torch.bfloat16)


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_weight_only_against_64_bits(ops, M, N, K):
  x, w, bias = operands(M, N, K)
  got = ops.w4a16_mm(x.cuda(), w[0].cuda(), w[1].cuda(), bias.cuda())
  assert got.shape == (M, N) and got.dtype == torch.bfloat16
  want, sums = mo.product(x.double().cuda(), mo.dequantize(*w).cuda(), bias.cuda())
  # bf16 operands: exact products, fp32 sums in any order, 2^-24 of the magnitudes' sum for each of K additions at most
  limit = 2.0**-8 * want.abs() + K * 2.0**-24 * sums + 1e-6
  assert ((got.double() - want).abs() <= limit).all()


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 77, 256), (40, 129, 480), (300, 640, 1024), (600, 1024, 2560)])
@pytest.mark.parametrize("gelu", [False, True])
def test_product_of_codes(ops, out, M, N, K, gelu):
  x, w, bias = operands(M, N, K, 5)
  a = ops.mxfp4_quant(x.cuda())
  w = [t.cuda() for t in w]
  for b in (bias.cuda(), None):
    got = ops.mxfp4_mm(*a, *w, out, bias=b, epilogue=int(gelu))
    assert got.dtype == out
    check(got, *mo.product(mo.dequantize(*mo.quantize(x)).cuda(), mo.dequantize(*[t.cpu() for t in w]).cuda(), b, gelu), out, gelu)


@pytest.mark.parametrize("M", [1, 2, 9, 16, 17, 40, 64, 200, 700])
@pytest.mark.parametrize("N,K", [(16, 32), (80, 288), (512, 512), (1024, 640), (515, 1024)])
def test_every_k_and_scale_is_where_it_belongs(ops, M, N, K):
  """Small whole numbers under powers of two: every partial sum is exact (multiples of 1/64, at most 8 K in magnitude, under
  24 bits; addends at most 2^9 apart), so the result has to be equal, bit for bit."""
  g = torch.Generator().manual_seed(M * N + K)
  def draw(R):
    c = torch.randint(0, 3, (R, K), generator=g) + 8 * torch.randint(0, 2, (R, K), generator=g)  # 0, .5, 1 and signs
    c = c.to(torch.uint8)
    s = torch.full((R, mo.scale_bytes(K)), 127, dtype=torch.uint8)
    s[:, :K // 32] = torch.randint(125, 128, (R, K // 32), generator=g).to(torch.uint8)
    return c[:, 0::2] | (c[:, 1::2] << 4), s
  a, w = draw(M), draw(N)
  av, wv = mo.dequantize(*a), mo.dequantize(*w)
  want = av @ wv.t()
  got = ops.mxfp4_mm(*[t.cuda() for t in a], *[t.cuda() for t in w], torch.float32)
  assert torch.equal(got.cpu().double(), want)
  got = ops.w4a16_mm(av.to(torch.bfloat16).cuda(), *[t.cuda() for t in w])
  assert torch.equal(got.cpu(), want.to(torch.bfloat16))


@pytest.mark.parametrize("M", [1, 3, 40, 300])
def test_a_nan_stays_in_its_row_and_column(ops, M):
  x, w, bias = operands(M, 200, 320, 9)
  x[0, 7] = float("nan")
  w[1][5, 3] = 255
  for f in (ops.mxfp4_linear, ops.w4a16_mm):
    got = f(x.cuda(), w[0].cuda(), w[1].cuda(), bias.cuda()).cpu()
    want = torch.zeros(M, 200, dtype=torch.bool)
    want[0], want[:, 5] = True, True
    assert torch.equal(got.isnan(), want)


@pytest.mark.parametrize("M", [1, 30, 500])
def test_layouts_of_the_products(ops, M):
  """Row strides, slices, rows off their alignment, leading dimensions, a bias off its own."""
  N, K = 264, 512
  x, w, bias = operands(M, N, K, 3)
  x, w, bias = x.cuda(), [t.cuda() for t in w], bias.cuda()
  for f in (ops.mxfp4_linear, ops.w4a16_mm):
    want = f(x, *w, bias)
    wide = torch.full((M, K + 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, :K] = x
    assert torch.equal(f(wide[:, :K], *w, bias), want)
    assert torch.equal(f(x.t().contiguous().t(), *w, bias), want)
    odd = torch.zeros(M * K + 1, dtype=torch.bfloat16, device="cuda")
    odd[1:] = x.reshape(-1)
    assert torch.equal(f(odd[1:].view(M, K), *w, bias), want)
    wcodes = torch.full((N, K // 2 + 48), 0x77, dtype=torch.uint8, device="cuda")
    wcodes[:, :K // 2] = w[0]
    wscale = torch.full((N, 20), 255, dtype=torch.uint8, device="cuda")
    wscale[:, 4:] = w[1]
    assert torch.equal(f(x, wcodes[:, :K // 2], wscale[:, 4:], bias), want)
    b1 = torch.zeros(N + 1, dtype=torch.bfloat16, device="cuda")
    b1[1:] = bias
    assert torch.equal(f(x, *w, b1[1:]), want)
    assert torch.equal(f(x[:, None], *w, bias), want[:, None])
    assert f(x[0], *w, bias).shape == (N, )
    assert f(x[:0], *w, bias).shape == (0, N)


def test_products_without_a_sum(ops):
  bias = torch.tensor([1.0, -2.0, 0.5], dtype=torch.bfloat16, device="cuda")
  x = torch.empty(4, 0, dtype=torch.bfloat16, device="cuda")
  w = torch.empty(3, 0, dtype=torch.uint8, device="cuda")
  for f in (ops.mxfp4_linear, ops.w4a16_mm):
    assert torch.equal(f(x, w, w, bias), bias.expand(4, 3))
    assert torch.equal(f(x, w, w, bias, 1), torch.nn.functional.gelu(bias.float(), approximate="tanh").to(bias.dtype).expand(4, 3))


def test_refusals(ops):
  x, w, bias = (t for t in operands(4, 32, 64))
  x, w, bias = x.cuda(), [t.cuda() for t in w], bias.cuda()
  with pytest.raises(ValueError, match="multiple of 32"):
    ops.mxfp4_quant(x[:, :40])
  with pytest.raises(ValueError, match="float16, bfloat16 or float32"):
    ops.mxfp4_quant(x.double())
  with pytest.raises(RuntimeError, match="no CPU path"):
    ops.mxfp4_quant(x.cpu())
  with pytest.raises(ValueError, match="bfloat16"):
    ops.mxfp4_linear(x.half(), *w)
  with pytest.raises(ValueError, match="bfloat16"):
    ops.w4a16_mm(x.float(), *w)
  with pytest.raises(ValueError, match="shape mismatch"):
    ops.mxfp4_linear(x[:, :32], *w)
  with pytest.raises(ValueError, match="scale bytes"):
    ops.w4a16_mm(x, w[0], w[1][:, :2])
  with pytest.raises(ValueError, match="leading dimensions"):
    ops.mxfp4_dequant(w[0][:3], w[1])
  with pytest.raises(ValueError, match="uint8"):
    ops.mxfp4_linear(x, w[0].view(torch.int8), w[1])
  with pytest.raises(ValueError, match="bias must have"):
    ops.mxfp4_linear(x, *w, bias[:5])
  with pytest.raises(ValueError, match="output dtype"):
    ops.mxfp4_dequant(*w, torch.float64)
  from cache_dit_amd import _native
  with pytest.raises(_native.CditNativeError, match="epilogue"):
    ops.mxfp4_linear(x, *w, bias, 4)
