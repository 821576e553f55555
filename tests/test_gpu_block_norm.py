"""gate_residual_norm on the GPU against 64 bits."""
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


def check(name, got, want, terms, K):
  """One rounding (eps/2 relative) and fp32 arithmetic: `terms` is what the steps' magnitudes add up to (cancellation between
  them is not divided out). A mean of K values in fp32 is off by at most K 2^-24 of their mean magnitude added in a row, by
  about log2 K of it in the trees used; 64 + K / 64 roundings of 2^-24 hold for both statistics and the steps behind them."""
  eps = torch.finfo(got.dtype).eps / 2
  tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # fp16's results may be subnormal
  err = (got.double().cpu() - want).abs()
  limit = eps * want.abs() + terms * (64 + K / 64) * 2.0**-24 * (1 + eps) + tiny
  assert (err <= limit).all(), (name, float((err / limit).max()), float(err.max()))


def run_case(ops, shape, K, dtype, stream, norm, post, mod, residual_scale=1.0, seed=0, eps=1e-6):
  g = torch.Generator().manual_seed(seed)
  full = (*shape, K)
  x = (torch.randn(full, generator=g) * 3 + torch.randn(*shape, 1, generator=g)).to(stream)
  b = torch.randn(full, generator=g).to(dtype)
  kw, names = {}, ("gate", "shift", "scale")
  if mod == "one":
    v = {n: torch.randn(K, generator=g) * 0.3 for n in names}
  elif mod == "batch":
    v = {n: torch.randn(shape[0], *([1] * (len(shape) - 1)), K, generator=g) * 0.3 for n in names}
  elif mod == "token":
    v = {n: torch.randn(full, generator=g) * 0.3 for n in names}
  else:
    v = {}
    if "gate" in mod:
      v["gate"] = torch.randn(K, generator=g)
    if "weight" in mod:
      kw["norm_weight"] = (1 + 0.1 * torch.randn(K, generator=g)).to(dtype)
    if "shift" in mod:
      v["shift"] = torch.randn(K, generator=g)
  kw.update({n: t.to(dtype) for n, t in v.items()})
  if post:
    kw["post_norm"] = post.split("-")[0]
    if post.endswith("-w"):
      kw["post_weight"] = (1 + 0.1 * torch.randn(K, generator=g)).to(dtype)
  want_h, want_y = mo.gate_residual_norm(x, b, norm_kind=norm, residual_scale=residual_scale, eps=eps, **kw)
  h, y = ops.gate_residual_norm(x.cuda(), b.cuda(), norm=norm, residual_scale=residual_scale, eps=eps,
                                **{n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in kw.items()})
  assert h.dtype == stream and y.dtype == dtype and h.shape == x.shape == y.shape
  # magnitudes that the sums go through
  t = b.double().abs() if not post else mo.norm(b.double(), kw["post_norm"], eps).abs() + 1
  if "post_weight" in kw:
    t = t * kw["post_weight"].double().abs()
  hm = abs(residual_scale) * x.double().abs() + t * (kw["gate"].double().abs() if "gate" in kw else 1)
  check("h", h, want_h, hm, K)
  var = (want_h - (want_h.mean(-1, keepdim=True) if norm == "layer" else 0)).square().mean(-1, keepdim=True)
  rstd = 1 / torch.sqrt(var + eps)
  # an error of h moves y by rstd of it, directly, through the mean and through the variance
  ym = (hm + hm.mean(-1, keepdim=True)) * rstd + mo.norm(want_h, norm, eps).abs() * (1 + (hm.square().mean(-1, keepdim=True)).sqrt() * rstd)
  for n, f in (("norm_weight", lambda w: w.abs()), ("scale", lambda w: (1 + w).abs() + 1)):
    if n in kw:
      ym = ym * f(kw[n].double())
  if "shift" in kw:
    ym = ym + kw["shift"].double().abs()
  check("y", y, want_y, ym, K)


TYPES = [(BF16, BF16), (F16, F16), (F32, F32), (BF16, F32), (F16, F32)]


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("norm,post,mod", [("layer", None, "batch"), ("rms", "rms-w", "weight"), ("layer", "layer", "token"),
                                           ("rms", "rms", "one"), ("rms", None, "none")])
@pytest.mark.parametrize("shape,K", [((2, 5), 256), ((1, 3), 5120)])
def test_types_and_forms(ops, dtype, stream, norm, post, mod, shape, K):
  run_case(ops, shape, K, dtype, stream, norm, post, mod)


@pytest.mark.parametrize("K", [1, 7, 8, 40, 63, 64, 100, 512, 513, 1000, 1536, 2048, 2560, 4104, 6144, 8192, 8200, 12288, 15360,
                               16384, 16392, 20000])
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_widths(ops, K, norm):
  # (one element: a LayerNorm of it is 0 whatever it is, and eps decides; eps of 1e-2 keeps rstd small there)
  run_case(ops, (2, 3), K, BF16, BF16, norm, "rms-w" if K % 3 else None, "batch", eps=1e-6 if K > 1 else 1e-2)


@pytest.mark.parametrize("K", [8, 9, 15, 17, 71, 505, 519, 1025, 2047, 4097, 6151, 8193, 15001, 16383, 16385])
@pytest.mark.parametrize("dtype,stream", TYPES)
def test_rows_of_any_length(ops, K, dtype, stream):
  """Pieces of 8 that end with the row; every lane's, wavefront's and register's edge."""
  run_case(ops, (2, 3), K, dtype, stream, "layer", "layer", "batch", seed=K)
  run_case(ops, (1, 4), K, dtype, stream, "rms", None, "token", seed=K + 1)


@pytest.mark.parametrize("shape", [(1, 1), (1, ), (3, ), (1, 700), (5, 401), (2, 3, 4)])
def test_rows(ops, shape):
  run_case(ops, shape, 1280, BF16, F32, "layer", "rms-w", "batch" if len(shape) > 1 else "one")


@pytest.mark.parametrize("mod", ["gate", "weight", "shift", "gate weight shift"])
def test_what_is_none_is_left_out(ops, mod):
  run_case(ops, (2, 4), 640, BF16, BF16, "layer", None, mod, residual_scale=0.5)


def test_rows_far_from_zero_and_constant_rows(ops):
  """A mean 1000 times the deviation: squares of the values less the mean. A constant row: y is the shift."""
  g = torch.Generator().manual_seed(1)
  x = 1000 + torch.randn(4, 4096, generator=g)
  b = torch.randn(4, 4096, generator=g)
  x[3], b[3] = 5.0, 0.0
  shift = torch.randn(4096, generator=g)
  want_h, want_y = mo.gate_residual_norm(x, b, shift=shift)
  h, y = ops.gate_residual_norm(x.cuda(), b.cuda(), shift=shift.cuda())
  check("h", h, want_h, x.double().abs() + b.double().abs(), 4096)
  # h is off by half a step of 1000 (3.1e-5), the mean by less; both over a deviation of 1.41
  assert ((y.double().cpu() - want_y).abs()[:3] <= 1e-4).all()
  assert torch.equal(y[3].cpu(), shift)


def test_not_finite_values_stay_in_their_rows(ops):
  x = torch.randn(6, 512).to(BF16)
  b = torch.randn(6, 512).to(BF16)
  x[1, 3], b[4, 500] = float("nan"), float("inf")
  h, y = (t.cpu() for t in ops.gate_residual_norm(x.cuda(), b.cuda(), norm="rms"))
  bad = torch.tensor([1, 4])
  good = torch.tensor([0, 2, 3, 5])
  assert y[1].isnan().all() and y[4, 500].isnan()
  assert y[good].isfinite().all() and h[good].isfinite().all() and h[bad].isfinite().sum() == 2 * 511


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("K", [32, 96, 1280, 5120, 16384, 16416])
def test_codes_are_those_of_the_rounded_result(ops, dtype, stream, K):
  g = torch.Generator().manual_seed(K)
  x, b = torch.randn(2, 9, K, generator=g).to(stream).cuda(), torch.randn(2, 9, K, generator=g).to(dtype).cuda()
  kw = dict(gate=torch.randn(2, 1, K, generator=g).to(dtype).cuda(), scale=torch.randn(2, 1, K, generator=g).to(dtype).cuda(),
            post_norm="rms", post_weight=torch.randn(K, generator=g).to(dtype).cuda())
  h, y = ops.gate_residual_norm(x, b, **kw)
  h2, codes, scales = ops.gate_residual_norm(x, b, **kw, quant_type="mxfp4")
  want = ops.mxfp4_quant(y)
  assert torch.equal(h, h2) and torch.equal(codes, want[0]) and torch.equal(scales, want[1])


def test_layouts(ops):
  """Row strides, slices of a joint sequence, chunks of a modulation, a mix of types, off their alignment."""
  B, S, K = 2, 10, 768
  g = torch.Generator().manual_seed(2)
  x, b = (torch.randn(B, S, K, generator=g).to(BF16).cuda() for _ in range(2))
  mod = torch.randn(B, 1, 3 * K, generator=g).to(BF16).cuda()
  gate, shift, scale = mod.chunk(3, dim=-1)
  want = ops.gate_residual_norm(x, b, gate.contiguous(), shift.contiguous(), scale.contiguous())

  def equal(got, part=slice(None)):
    assert torch.equal(got[0], want[0][part]) and torch.equal(got[1], want[1][part])

  equal(ops.gate_residual_norm(x, b, gate, shift, scale))
  equal(ops.gate_residual_norm(x, b, gate[:, 0], shift, scale.expand(B, S, K)))
  equal(ops.gate_residual_norm(x, b, gate.float(), shift, scale))
  equal(ops.gate_residual_norm(x, b, gate.float(), shift.float(), scale.float()))
  joint = torch.cat((torch.full((B, 3, K), float("nan"), dtype=BF16, device="cuda"), b), 1)
  equal(ops.gate_residual_norm(x, joint[:, 3:], gate, shift, scale))
  one = ops.gate_residual_norm(x[:1], joint[:1, 3:], gate[:1], shift[:1], scale[:1])
  equal(one, slice(0, 1))
  odd = torch.zeros(B * S * K + 1, dtype=BF16, device="cuda")
  odd[1:] = b.reshape(-1)
  got = ops.gate_residual_norm(x, odd[1:].view(B, S, K), gate, shift, scale)
  # (another order of additions: an ulp of bf16 here and there)
  assert (got[1].float() - want[1].float()).abs().max() <= 2.0**-7 * want[1].float().abs().max()
  tokens = mod.expand(B, S, 3 * K).contiguous()
  equal(ops.gate_residual_norm(x, b, *tokens.chunk(3, dim=-1)))
  assert all(t.shape == (0, 4, K) for t in ops.gate_residual_norm(x[:0, :4], b[:0, :4]))


def test_refusals(ops):
  x = torch.randn(2, 3, 64, device="cuda").to(BF16)
  v = torch.ones(64, device="cuda", dtype=BF16)
  f = ops.gate_residual_norm
  with pytest.raises(ValueError, match="norm must be"):
    f(x, x, norm="batch")
  with pytest.raises(ValueError, match="without post_norm"):
    f(x, x, post_weight=v)
  with pytest.raises(ValueError, match="quant_type"):
    f(x, x, quant_type="int8")
  with pytest.raises(ValueError, match="one shape"):
    f(x, x[:1])
  with pytest.raises(ValueError, match="of its type or float32"):
    f(x, x.float())
  with pytest.raises(ValueError, match="vectors of K"):
    f(x, x, gate=v[:32])
  with pytest.raises(ValueError, match="one per index"):
    f(x, x, gate=v.expand(3, 64))
  with pytest.raises(ValueError, match="expected one vector"):
    f(x, x, norm_weight=v.expand(2, 64))
  with pytest.raises(ValueError, match="multiple of 32"):
    f(x[..., :40], x[..., :40], quant_type="mxfp4")
  with pytest.raises(RuntimeError, match="no CPU path"):
    f(x, x.cpu())
  with pytest.raises(RuntimeError, match="no backward"):
    f(x.float().requires_grad_(), x.float())
  with torch.no_grad():
    f(x.float().requires_grad_(), x.float())
