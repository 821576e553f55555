"""gate_residual_norm, the quantizer and its inverse where what is read once goes past the caches (non-temporal accesses, above 64
MB): the results are those of the same rows in calls below that size, bit for bit; and rows off their alignment, whose lanes hold
the same pieces as those of aligned rows."""
import pytest
import torch

from oracle import mxfp4_oracle as mo

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  from cache_dit_amd import ops
  return ops


def rand(shape, dtype, seed, std=1.0):
  return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").mul_(std).to(dtype)


def slices(t, at, n):
  """Tokens at .. at + n - 1 of each batch entry; vectors of an entry, or of all, as they are."""
  return t if t is None or t.dim() < 3 or t.shape[1] == 1 else t[:, at:at + n]


@pytest.mark.parametrize("dtype,stream", [(BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("B,S,K", [(3, 2200, 5120), (2, 9000, 2048), (3, 1399, 8192), (2, 1300, 15360)])
@pytest.mark.parametrize("mod", ["batch", "token"])
@pytest.mark.parametrize("post,codes", [(None, False), ("rms", True)])
def test_norm_past_the_caches(ops, dtype, stream, B, S, K, mod, post, codes):
  """One piece of a row a lane and two; a workgroup's run of rows crosses the batch entries."""
  assert 2 * B * S * K >= 64 << 20
  x, branch = rand((B, S, K), stream, 1), rand((B, S, K), dtype, 2)
  gate, shift, scale = (rand((B, S if mod == "token" else 1, K), dtype, 3 + i, 0.3) for i in range(3))
  kw = dict(norm="layer" if post else "rms", post_norm=post, quant_type="mxfp4" if codes else None)
  if post:
    kw["post_weight"] = rand((K, ), dtype, 7)
  else:
    kw["norm_weight"] = rand((K, ), dtype, 8)
  got = ops.gate_residual_norm(x, branch, gate, shift, scale, **kw)
  n = (32 << 20) // (2 * B * K)  # half of the size above
  for at in range(0, S, n):
    part = [slices(t, at, n) for t in (x, branch, gate, shift, scale)]
    for a, b in zip(got, ops.gate_residual_norm(*part, **kw)):
      assert torch.equal(a[:, at:at + n], b)
  # and a few rows against 64 bits: the statistics' roundings (K / 64 and some of 2^-24 of terms of order 10) and one of the type
  pick = torch.tensor([0, S // 2, S - 1], device="cuda")
  few = [t if t.shape[1] == 1 else t[:, pick] for t in (x, branch, gate, shift, scale)]
  want_h, want_y = mo.gate_residual_norm(*(t.cpu() for t in few), norm_kind=kw["norm"], post_norm=post,
                                         norm_weight=kw["norm_weight"].cpu() if not post else None,
                                         post_weight=kw["post_weight"].cpu() if post else None)
  small = 10 * (64 + K / 64) * 2.0**-24
  h = got[0][:, pick].double().cpu()
  assert ((h - want_h).abs() <= torch.finfo(stream).eps / 2 * want_h.abs() + small).all()
  if not codes:
    y = got[1][:, pick].double().cpu()
    assert ((y - want_y).abs() <= torch.finfo(dtype).eps / 2 * want_y.abs() + 4 * small).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,K", [(9001, 4096), (2500, 13824), (1100000, 32)])
def test_quantizer_past_the_caches(ops, dtype, M, K):
  assert 2 * M * K > 64 << 20
  x = rand((M, K), dtype, 1) * torch.exp2(torch.randint(-8, 5, (M, 1), device="cuda").float()).to(dtype)
  x[5, 7], x[M - 1, 31] = float("inf"), float("nan")
  codes, scales = ops.mxfp4_quant(x)
  v = ops.mxfp4_dequant(codes, scales, dtype)
  n = (32 << 20) // (2 * K)
  for at in range(0, M, n):
    c, s = ops.mxfp4_quant(x[at:at + n])
    assert torch.equal(codes[at:at + n], c) and torch.equal(scales[at:at + n], s)
    assert torch.equal(v[at:at + n].view(torch.int16), ops.mxfp4_dequant(c, s, dtype).view(torch.int16))
  for rows in (slice(0, 40), slice(M - 40, M)):
    want = mo.quantize(x[rows].cpu())
    assert torch.equal(codes[rows].cpu(), want[0]) and torch.equal(scales[rows].cpu(), want[1])


@pytest.mark.parametrize("dtype,stream", [(BF16, BF16), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("K", [96, 768, 1000, 2048, 5120, 8192])
def test_rows_off_their_alignment_are_equal(ops, dtype, stream, K):
  """Lane l of a row's wavefronts has piece l either way, and wavefronts without a piece add zeros: nothing differs."""
  M = 37
  x, branch, gate = rand((M, K), stream, 1), rand((M, K), dtype, 2), rand((K, ), dtype, 3)
  odd = torch.zeros(M * K + 1, dtype=dtype, device="cuda")
  odd[1:] = branch.reshape(-1)
  apart = torch.full((M, K + 3), float("nan"), dtype=stream, device="cuda")
  apart[:, :K] = x
  for kw in (dict(norm="rms"), dict(norm="layer", post_norm="layer", shift=rand((K, ), dtype, 4))):
    want = ops.gate_residual_norm(x, branch, gate, **kw)
    for got in (ops.gate_residual_norm(x, odd[1:].view(M, K), gate, **kw), ops.gate_residual_norm(apart[:, :K], branch, gate, **kw)):
      assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
