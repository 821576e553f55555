"""MXFP4 as it is used: quantized modules, a block's operators one after the other, captured graphs, other streams,
torch.compile; every kernel variant; operands beyond 32-bit offsets."""
import copy

import pytest
import torch
from torch import nn

from oracle import mxfp4_oracle as mo

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
TYPES = ["mxfp4", "mxfp4_weight_only"]


@pytest.fixture(scope="module")
def cd():
  if not torch.cuda.is_available():
    pytest.skip("no GPU")
  import cache_dit_amd
  return cache_dit_amd


def rand(*shape, seed=0, std=1.0):
  return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).mul_(std).to(BF16).cuda()


class Block(nn.Module):

  def __init__(self, d):
    super().__init__()
    self.to_q = nn.Linear(d, d)
    self.proj_mlp = nn.Linear(d, 4 * d)
    self.act_mlp = nn.GELU(approximate="tanh")
    self.proj_out = nn.Linear(4 * d, d, bias=False)
    self.mod = nn.Linear(d, d)

  def forward(self, x):
    return x + self.proj_out(self.act_mlp(self.proj_mlp(self.to_q(x) + self.mod(x))))


class Net(nn.Module):
  _repeated_blocks = ["Block"]

  def __init__(self, d=288):
    super().__init__()
    self.blocks = nn.ModuleList([Block(d), Block(d)])

  def forward(self, x):
    for b in self.blocks:
      x = b(x)
    return x


def product_limit(want, sums, K, codes):
  """bf16's half step, and the sum's own error: as in the tests of the operators (codes: the 4-bit instruction's
  alignment of addends, 2^-12; else fp32 additions)."""
  return 2.0**-8 * want.abs() + (1.2 * 2.0**-12 if codes else K * 2.0**-24) * sums + 1e-6


def check_product(got, x, w, scale, bias, qt, gelu=False):
  """`got` for bf16 x [M, K] against 64 bits."""
  a = mo.dequantize(*mo.quantize(x.cpu())).cuda() if qt == "mxfp4" else x.double()
  v = mo.dequantize(w.cpu(), scale.cpu()).cuda()
  want, sums = mo.product(a, v, bias, gelu)
  # (GELU has slopes up to 1.13)
  limit = product_limit(want, sums * (1.13 if gelu else 1.0), x.shape[-1], qt == "mxfp4") + (2e-6 * want.abs() if gelu else 0)
  err = (got.double() - want).abs()
  assert (err <= limit).all(), (float((err / limit).max()), float(err.max()))


# ------------------------------------------------------------------------------------ modules


@pytest.mark.parametrize("qt", TYPES)
@pytest.mark.parametrize("where", ["gpu", "cpu_then_gpu"])
def test_quantize_a_module(cd, qt, where):
  torch.manual_seed(0)
  net = Net().to(BF16)
  ref = copy.deepcopy(net)
  net = net.cuda() if where == "gpu" else net
  assert cd.quantize(net, cd.QuantizeConfig(quant_type=qt)) is net
  net = net.cuda()
  cls = cd.Mxfp4Linear if qt == "mxfp4" else cd.Mxfp4WeightOnlyLinear
  for blk, rblk in zip(net.blocks, ref.blocks):
    assert type(blk.mod) is nn.Linear  # excluded
    for name in ("to_q", "proj_mlp", "proj_out"):
      lin, rlin = getattr(blk, name), getattr(rblk, name)
      assert type(lin) is cls and isinstance(lin, nn.Linear) and not lin.weight.requires_grad
      codes, scales = mo.quantize(rlin.weight.detach())
      assert torch.equal(lin.weight.cpu(), codes) and torch.equal(lin.weight_scale.cpu(), scales)
      from cache_dit_amd.nn import dequantize_weight
      assert torch.equal(dequantize_weight(lin).cpu(), mo.dequantize(codes, scales).to(BF16))
      for x in (rand(3, lin.in_features, seed=1), rand(130, lin.in_features, seed=2)):
        check_product(lin(x), x, lin.weight, lin.weight_scale, lin.bias, qt)
  x = rand(2, 50, 288, seed=3)
  y = net(x)
  assert y.shape == x.shape and y.dtype == BF16 and y.isfinite().all()
  assert "quant_type=" + qt in repr(net.blocks[0].to_q)
  # saved and loaded
  other = Net().to(BF16).cuda()
  cd.quantize(other, cd.QuantizeConfig(quant_type=qt))
  other.load_state_dict(net.state_dict())
  assert torch.equal(other(x), y)


@pytest.mark.parametrize("qt", TYPES)
def test_fused_gelu(cd, qt):
  torch.manual_seed(1)
  lin, act = nn.Linear(160, 264, dtype=BF16).cuda(), nn.GELU(approximate="tanh")
  from cache_dit_amd.nn import convert_linear_
  convert_linear_(lin, qt)
  cd.fuse_gelu_tanh_(lin, act)
  for M in (1, 40, 300):
    x = rand(M, 160, seed=M)
    check_product(act(lin(x)), x, lin.weight, lin.weight_scale, lin.bias, qt, gelu=True)


def test_module_on_codes(cd):
  """Siblings that read one activation: quantized once, the results are those of the plain calls."""
  from cache_dit_amd.nn import convert_linear_
  torch.manual_seed(2)
  lins = [nn.Linear(320, n, dtype=BF16).cuda() for n in (320, 64, 1000)]
  for lin in lins:
    convert_linear_(lin, "mxfp4")
  for M in (1, 77, 600):
    x = rand(2, M, 320, seed=M)
    codes = cd.mxfp4_quant(x)
    for lin in lins:
      # (few rows run another kernel: another order of additions)
      got, want = lin(codes), lin(x)
      assert got.shape == want.shape
      assert (got.float() - want.float()).abs().max() <= 2.0**-7 * want.float().abs().max()
  with pytest.raises(ValueError, match="shape mismatch"):
    lins[0](cd.mxfp4_quant(x[..., :64]))


@pytest.mark.parametrize("qt", TYPES)
def test_input_checks_of_the_modules(cd, qt):
  from cache_dit_amd.nn import convert_linear_
  lin = nn.Linear(64, 40, dtype=BF16).cuda()
  convert_linear_(lin, qt)
  with pytest.raises(ValueError, match="bfloat16"):
    lin(torch.zeros(4, 64, device="cuda"))
  with pytest.raises(RuntimeError, match="no CPU path"):
    lin(torch.zeros(4, 64, dtype=BF16))
  assert lin(torch.zeros(0, 64, dtype=BF16, device="cuda")).shape == (0, 40)
  y = lin(torch.zeros(3, 5, 64, dtype=BF16, device="cuda"))
  assert torch.equal(y, lin.bias.expand(3, 5, 40))


@pytest.mark.parametrize("qt", TYPES)
def test_a_whole_transformer(cd, qt):
  """A small FLUX-shaped model, GELU in the Linears: with the stage patch (which leaves these Linears as they are), replayed
  from a graph, and, weight-only, against plain Linears on the dequantized weights (bf16 holds them exactly)."""
  from cache_dit_amd import nn as cnn
  from cache_dit_amd.testing import dit_shapes as ds
  torch.manual_seed(5)
  model = ds.FluxLikeTransformer(dim=256, heads=4, mlp=1024, n_double=2, n_single=2, text_dim=192, pooled_dim=96).to(BF16).cuda()
  plain = copy.deepcopy(model)
  cd.quantize(model, cd.QuantizeConfig(quant_type=qt))
  converted = {n: m for n, m in model.named_modules() if isinstance(m, (cd.Mxfp4Linear, cd.Mxfp4WeightOnlyLinear))}
  assert len(converted) >= 2 * 10 + 2 * 5 and all(m.quant_type == qt for m in converted.values())
  for n, m in plain.named_modules():
    if n in converted:
      m.weight.data.copy_(cnn.dequantize_weight(converted[n]))
  assert ds.fuse_gelu_epilogues(model) > 0
  inputs = ds.flux_like_inputs("cuda", n_img=100, n_txt=20, text_dim=192, pooled_dim=96, seed=6)
  with torch.no_grad():
    out = model(**inputs)
    out = out[0] if isinstance(out, tuple) else out
    assert out.isfinite().all()
    if qt == "mxfp4_weight_only":
      want = plain(**inputs)
      want = want[0] if isinstance(want, tuple) else want
      # some 40 roundings to bf16 of half a step on either side, independent: 2^-9 sqrt(80), 2 % of the magnitude, 2e-4 in the cosine
      cos = torch.nn.functional.cosine_similarity(out.double().flatten(), want.double().flatten(), dim=0)
      assert cos >= 0.999, float(cos)
    cd.apply_stage_patch(model)
    patched = model(**inputs)
    assert torch.equal(patched[0] if isinstance(patched, tuple) else patched, out)
    cd.remove_stage_patch(model)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      model(**inputs)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      static = model(**inputs)
    static = static[0] if isinstance(static, tuple) else static
    for seed in range(3):
      new = ds.flux_like_inputs("cuda", n_img=100, n_txt=20, text_dim=192, pooled_dim=96, seed=seed)
      want = model(**new)
      torch.cuda.synchronize()
      for k in inputs:
        inputs[k].copy_(new[k])
      g.replay()
      torch.cuda.synchronize()
      assert torch.equal(static, want[0] if isinstance(want, tuple) else want), seed


# ----------------------------------------------------------------- one after the other


class Stage:
  """What stands between attention and the end of a block's feed-forward: h and y's codes, up, GELU, down, h again."""

  def __init__(self, cd, K, F, fp32_stream):
    self.cd = cd
    self.up, self.down = cd.mxfp4_quant(rand(F, K, seed=11, std=0.05)), cd.mxfp4_quant(rand(K, F, seed=12, std=0.03))
    self.bias = rand(F, seed=13, std=0.1)
    self.vec = [rand(2, 1, K, seed=14 + i, std=0.3) for i in range(3)]
    self.stream = torch.float32 if fp32_stream else BF16

  def __call__(self, x, branch):
    gate, shift, scale = self.vec
    h, codes, scales = self.cd.gate_residual_norm(x, branch, gate, shift, scale, norm="rms", quant_type="mxfp4")
    up = self.cd.mxfp4_mm(codes, scales, *self.up, bias=self.bias, epilogue=1)
    down = self.cd.mxfp4_mm(*self.cd.mxfp4_quant(up), *self.down)
    out, y = self.cd.gate_residual_norm(h, down, gate, norm="layer")
    return h, codes, scales, up, down, out, y


@pytest.mark.parametrize("tokens,K,F,fp32_stream", [(1, 256, 512, False), (9, 288, 1000 // 32 * 32, True), (200, 640, 2560, False)])
def test_a_stage_against_64_bits(cd, tokens, K, F, fp32_stream):
  """Each step against its own definition in 64 bits, on what the step before gave it."""
  s = Stage(cd, K, F, fp32_stream)
  x, branch = rand(2, tokens, K, seed=20).to(s.stream), rand(2, tokens, K, seed=21)
  h, codes, scales, up, down, out, y = s(x, branch)
  gate, shift, scale = (t.cpu() for t in s.vec)
  want_h, want_y = mo.gate_residual_norm(x.cpu(), branch.cpu(), gate, shift, scale, norm_kind="rms")
  assert h.dtype == s.stream
  terms = x.cpu().double().abs() + (gate.double() * branch.cpu().double()).abs()
  eps = torch.finfo(s.stream).eps / 2
  assert ((h.cpu().double() - want_h).abs() <= eps * want_h.abs() + 64 * 2.0**-24 * terms).all()
  # the codes are those of y rounded to bf16; y itself may be an fp32 rounding apart, so: of the unfused call
  h1, y1 = cd.gate_residual_norm(x, branch, *s.vec, norm="rms")
  q1 = cd.mxfp4_quant(y1)
  assert torch.equal(h, h1) and torch.equal(codes, q1[0]) and torch.equal(scales, q1[1])
  # a step of bf16 for an fp32 result next to a tie, and the statistics' roundings
  assert ((y1.cpu().double() - want_y).abs() <= 2.0**-8 * want_y.abs() + 1e-4).all()

  def product(got, codes, scales, w, bias, gelu):
    a = mo.dequantize(codes.reshape(-1, codes.shape[-1]).cpu(), scales.reshape(-1, scales.shape[-1]).cpu())
    want, sums = mo.product(a, mo.dequantize(*(t.cpu() for t in w)), None if bias is None else bias.cpu(), gelu)
    limit = product_limit(want, 1.13 * sums, a.shape[1], True) + 2e-6 * want.abs()
    assert ((got.reshape(want.shape).cpu().double() - want).abs() <= limit).all()

  product(up, codes, scales, s.up, s.bias, True)
  q = mo.quantize(up.reshape(-1, F).cpu())
  product(down, *q, s.down, None, False)
  want_out, want_last = mo.gate_residual_norm(h.cpu(), down.cpu(), gate)
  terms = h.cpu().double().abs() + (gate.double() * down.cpu().double()).abs()
  assert ((out.cpu().double() - want_out).abs() <= eps * want_out.abs() + 64 * 2.0**-24 * terms).all()
  assert ((y.cpu().double() - want_last).abs() <= 2.0**-8 * want_last.abs() + 1e-4).all()


@pytest.mark.parametrize("tokens", [1, 8, 150])
def test_a_captured_stage_replays(cd, tokens):
  """Two graphs of the same weights, replayed in turn with new inputs, eager work in between."""
  s = Stage(cd, 512, 1536, True)
  lin = nn.Linear(512, 520, dtype=BF16).cuda()
  from cache_dit_amd.nn import convert_linear_
  convert_linear_(lin, "mxfp4")
  w4 = s.up

  def run(x, branch):
    out = s(x, branch)
    return (*out, lin(out[-1]), cd.ops.w4a16_mm(out[-1], *w4, s.bias))

  graphs = []
  with torch.no_grad():
    for i in range(2):
      x, b = rand(2, tokens, 512, seed=30 + i).float(), rand(2, tokens, 512, seed=40 + i)
      run(x, b)
      side = torch.cuda.Stream()
      side.wait_stream(torch.cuda.current_stream())
      with torch.cuda.stream(side):
        run(x, b)
      torch.cuda.current_stream().wait_stream(side)
      g = torch.cuda.CUDAGraph()
      with torch.cuda.graph(g):
        out = run(x, b)
      graphs.append((g, x, b, out))
    for turn in range(4):
      for g, x, b, out in graphs:
        nx, nb = rand(2, tokens, 512, seed=50 + turn).float(), rand(2, tokens, 512, seed=60 + turn)
        want = run(nx, nb)
        torch.cuda.synchronize()
        x.copy_(nx)
        b.copy_(nb)
        g.replay()
        torch.cuda.synchronize()
        for i, (o, w) in enumerate(zip(out, want)):
          assert torch.equal(o, w), (turn, i)


@pytest.mark.parametrize("tokens", [2, 300])
def test_two_streams_at_once(cd, tokens):
  s = Stage(cd, 512, 1536, False)
  inputs = [(rand(2, tokens, 512, seed=70 + i), rand(2, tokens, 512, seed=80 + i)) for i in range(2)]
  want = [s(*i) for i in inputs]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream() for _ in range(2)]
  got = [[], []]
  for _ in range(5):
    for k, st in enumerate(streams):
      with torch.cuda.stream(st):
        got[k].append(s(*inputs[k]))
  torch.cuda.synchronize()
  for k in range(2):
    for out in got[k]:
      assert all(torch.equal(a, b) for a, b in zip(out, want[k]))


@pytest.mark.parametrize("qt", TYPES)
@pytest.mark.parametrize("M", [4, 70])
def test_compiled_module(cd, qt, M):
  from cache_dit_amd.nn import convert_linear_
  torch.manual_seed(3)
  net = nn.Sequential(nn.Linear(96, 64, dtype=BF16), nn.Linear(64, 40, dtype=BF16)).cuda()
  for lin in net:
    convert_linear_(lin, qt)
  x = rand(M, 96, seed=4)
  with torch.no_grad():
    eager = net(x)
    torch._dynamo.reset()
    compiled = torch.compile(net, fullgraph=True)
    assert torch.equal(compiled(x), eager)
    x3 = rand(2, M, 96, seed=5)
    assert torch.equal(compiled(x3), net(x3))

    # (an activation of which only FP8 codes exist must not stop the tracing of other calls)
    only_codes = cd.ln_modulate_quant(rand(M, 128, seed=8), rand(128, seed=9), rand(128, seed=10), materialize=False)

    def norm(x, b, g):
      return cd.gate_residual_norm(x, b, g, norm="rms", quant_type="mxfp4")

    b, g = rand(M, 96, seed=6), rand(96, seed=7)
    for got, want in zip(torch.compile(norm, fullgraph=True)(x, b, g), norm(x, b, g)):
      assert torch.equal(got, want)
  torch._dynamo.reset()
  for call in (lambda: norm(only_codes, only_codes, None), lambda: cd.mxfp4_quant(only_codes)):
    with pytest.raises(RuntimeError, match="codes only"):
      call()


def test_forms_that_layouts_may_take(cd):
  """One element a row at any stride; scales that do not lie like their codes."""
  x = rand(40, 1, seed=8)
  odd = torch.zeros(40, 3, dtype=BF16, device="cuda")
  odd[:, :1] = x
  apart = odd.as_strided((40, 1), (3, 7))
  for got, want in zip(cd.gate_residual_norm(apart, apart, apart[3], eps=1e-2), cd.gate_residual_norm(x, x, x[3], eps=1e-2)):
    assert torch.equal(got, want)
  codes, scales = cd.mxfp4_quant(rand(2, 3, 64, seed=9))
  with pytest.raises(ValueError, match="leading dimensions"):
    cd.mxfp4_dequant(codes, scales.reshape(3, 2, 4))
  with pytest.raises(ValueError, match="leading dimensions"):
    cd.mxfp4_mm(codes, scales.reshape(6, 4), codes[0], scales[0])


# ------------------------------------------------------------------------------- variants

#: below, at and above a tile, K of one block, of part of a step, of an odd number of steps, of many
EDGES = [(1, 1, 32), (31, 65, 96), (33, 64, 256), (64, 127, 288), (130, 260, 1056), (257, 255, 512), (300, 513, 1312),
         (520, 770, 4128)]


@pytest.fixture
def variant(cd):
  from cache_dit_amd import _native
  yield _native.set_gemm_variant
  _native.set_gemm_variant(-1)


@pytest.mark.parametrize("v", range(9))
@pytest.mark.parametrize("M,N,K", EDGES)
def test_every_variant(cd, variant, v, M, N, K):
  """0: without tiles, 1 .. 8: the tiles, whatever the automatic choice is for the size."""
  x, w, bias = rand(M, K, seed=M), rand(N, K, seed=N, std=0.05), rand(N, seed=K, std=0.1)
  codes, scales = cd.mxfp4_quant(w)
  variant(v)
  got = cd.ops.mxfp4_linear(x, codes, scales, bias)
  check_product(got, x, codes, scales, bias, "mxfp4")
  check_product(cd.ops.w4a16_mm(x, codes, scales, bias, 1), x, codes, scales, bias, "mxfp4_weight_only", gelu=True)
  a = cd.mxfp4_quant(x)
  for dtype in (torch.float32, torch.float16):
    y = cd.mxfp4_mm(*a, codes, scales, dtype, bias)
    assert (y.float() - got.float()).abs().max() <= 2.0**-7 * max(1.0, float(got.float().abs().max()))


@pytest.mark.parametrize("M", [1, 5, 16])
@pytest.mark.parametrize("N,K", [(40, 32), (1000, 16384), (16, 65568), (20000, 544)])
def test_few_rows(cd, variant, M, N, K):
  """K in one piece, in pieces, longer than all of LDS; one and two groups of columns a workgroup; codes and bf16 in."""
  x, w, bias = rand(M, K, seed=M), rand(N, K, seed=N, std=0.05), rand(N, seed=K, std=0.1)
  codes, scales = cd.mxfp4_quant(w)
  for v in (-1, 100):
    variant(v)
    check_product(cd.ops.mxfp4_linear(x, codes, scales, bias), x, codes, scales, bias, "mxfp4")
    check_product(cd.mxfp4_mm(*cd.mxfp4_quant(x), codes, scales, BF16, bias), x, codes, scales, bias, "mxfp4")
    check_product(cd.ops.w4a16_mm(x, codes, scales, bias), x, codes, scales, bias, "mxfp4_weight_only")


@pytest.mark.parametrize("M,N,K", [(17, 100, 5120), (33, 16, 9248), (48, 40, 20000 // 32 * 32), (300, 130, 544), (500, 33, 2048)])
def test_few_columns(cd, variant, M, N, K):
  """More than 16 rows of the kernel for few, where it is chosen and where it is not."""
  x, w, bias = rand(M, K, seed=M), rand(N, K, seed=N, std=0.05), rand(N, seed=K, std=0.1)
  codes, scales = cd.mxfp4_quant(w)
  for v in (-1, 100):
    variant(v)
    check_product(cd.ops.mxfp4_linear(x, codes, scales, bias), x, codes, scales, bias, "mxfp4")
    check_product(cd.ops.w4a16_mm(x, codes, scales, bias, 1), x, codes, scales, bias, "mxfp4_weight_only", gelu=True)
    got = cd.mxfp4_mm(*cd.mxfp4_quant(x), codes, scales, torch.float32, bias)
    check_product(got, x, codes, scales, bias, "mxfp4")


# -------------------------------------------------------------------- beyond 32 bits


def big(M, K, seed=0):
  """bf16 [M, K] whose rows differ, made without much time: every row is a multiple of a power of two of another."""
  x = torch.empty(M, K, dtype=BF16, device="cuda")
  x[:4096].normal_(generator=torch.Generator(device="cuda").manual_seed(seed))
  for at in range(4096, M, 4096):
    n = min(4096, M - at)
    x[at:at + n] = x[:n] * 2.0**((at // 4096) % 7 - 3)
  return x


def test_quantizer_beyond_32_bits(cd):
  """4.6e9 elements: 9.2 GB in, 2.3 GB of codes."""
  x = big(70001, 65536)
  codes, scales = cd.mxfp4_quant(x)
  for rows in (slice(0, 3), slice(32766, 32770), slice(65534, 65539), slice(69998, 70001)):
    q, s = cd.mxfp4_quant(x[rows].clone())
    assert torch.equal(codes[rows], q) and torch.equal(scales[rows], s)
  del x
  v = cd.mxfp4_dequant(codes, scales)
  for rows in (slice(0, 3), slice(32766, 32770), slice(65534, 65539), slice(69998, 70001)):
    assert torch.equal(v[rows], cd.mxfp4_dequant(codes[rows].clone(), scales[rows].clone()))


@pytest.mark.parametrize("K", [16384, 16416])
def test_norm_beyond_32_bits(cd, K):
  """2.3e9 elements, with the row in registers and read again."""
  M = 140001
  x, branch = big(M, K, 1), big(M, K, 2)
  h, y = cd.gate_residual_norm(x, branch)
  for rows in (slice(0, 2), slice(65535, 65538), slice(131000, 131080), slice(M - 2, M)):
    h1, y1 = cd.gate_residual_norm(x[rows].clone(), branch[rows].clone())
    assert torch.equal(h[rows], h1) and torch.equal(y[rows], y1)


@pytest.mark.parametrize("qt", TYPES)
def test_products_beyond_32_bits(cd, qt):
  f = cd.ops.mxfp4_linear if qt == "mxfp4" else cd.ops.w4a16_mm
  # an output of 2.3e9 elements; an activation row of it at a stride of 2^16
  x = big(70001, 64)
  w = cd.mxfp4_quant(rand(32800, 64, seed=1, std=0.1))
  out = f(x, *w)
  for rows in (slice(0, 2), slice(65535, 65538), slice(69990, 70001)):
    check_product(out[rows], x[rows], *w, None, qt)
  del out, x
  # a weight of 4.9 GB, for one row and for many
  N, K = 299999, 32768
  codes = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device="cuda",
                        generator=torch.Generator(device="cuda").manual_seed(2))
  scales = torch.full((N, K // 32), 120, dtype=torch.uint8, device="cuda")
  for M in (1, 40):
    x = rand(M, K, seed=M)
    out = f(x, codes, scales)
    for cols in (slice(0, 16), slice(262140, 262150), slice(N - 9, N)):
      check_product(out[:, cols], x, codes[cols].clone(), scales[cols].clone(), None, qt)


@pytest.mark.parametrize("qt", TYPES)
def test_strides_beyond_32_bits(cd, qt):
  """Rows of the weight a quarter of a GiB apart: 16 of them do not fit 32-bit offsets; and an output row that far apart."""
  f = cd.ops.mxfp4_linear if qt == "mxfp4" else cd.ops.w4a16_mm
  N, K = 20, 256
  wide = torch.zeros(N, 2**28, dtype=torch.uint8, device="cuda")
  codes, scales = cd.mxfp4_quant(rand(N, K, seed=3))
  wide[:, :K // 2] = codes
  for M in (1, 16, 100):
    x = rand(M, K, seed=M)
    check_product(f(x, wide[:, :K // 2], scales), x, codes, scales, None, qt)


# ------------------------------------------------------------------------- C interface


def framed(rows, row_bytes, ld_bytes):
  """Memory of 0x5a with room for `rows` rows, 64 bytes in front, one row and 64 bytes behind; the rows' view."""
  m = torch.full((64 + (rows + 1) * ld_bytes + 64, ), 0x5a, dtype=torch.uint8, device="cuda")
  return m, m[64:64 + rows * ld_bytes].view(rows, ld_bytes)[:, :row_bytes]


def rest_is_untouched(m, view):
  view.fill_(0x5a)
  assert (m == 0x5a).all()


@pytest.mark.parametrize("v", [-1, 0, 1, 2, 3, 4, 5, 6, 7, 8, 100])
@pytest.mark.parametrize("M,N,K", [(1, 77, 96), (13, 33, 544), (70, 131, 160), (300, 260, 512)])
def test_nothing_but_the_outputs_is_written(cd, variant, v, M, N, K):
  """Outputs, codes, scales and workspaces with rows further apart than they are long, in memory that is looked over."""
  from cache_dit_amd import _native
  lib, stream = _native.load(), torch.cuda.current_stream().cuda_stream
  S = mo.scale_bytes(K)
  x, w, bias = rand(M, K, seed=1), rand(N, K, seed=2, std=0.05), rand(N, seed=3, std=0.1)
  codes, scales = cd.mxfp4_quant(w)
  a, a_s = cd.mxfp4_quant(x)
  variant(v)
  want = [cd.ops.mxfp4_linear(x, codes, scales, bias), cd.ops.w4a16_mm(x, codes, scales, bias),
          cd.mxfp4_mm(a, a_s, codes, scales, BF16, bias)]

  def call(f, *args):
    assert f(*args) == 0, lib.cdit_last_error()
    torch.cuda.synchronize()

  ldo = N + 5
  for which in range(3):
    m, out = framed(M, 2 * N, 2 * ldo)
    mq, q = framed(M, K // 2, K // 2)
    ms, s = framed(M, S, S)
    p = [codes.data_ptr(), scales.data_ptr(), bias.data_ptr(), out.data_ptr()]
    if which == 0:
      call(lib.cdit_mxfp4_linear, x.data_ptr(), *p, q.data_ptr(), s.data_ptr(), M, N, K, K, K // 2, S, ldo, 0, stream)
    elif which == 1:
      call(lib.cdit_w4a16_gemm, x.data_ptr(), *p, M, N, K, K, K // 2, S, ldo, 0, stream)
    else:
      call(lib.cdit_mxfp4_gemm, a.data_ptr(), a_s.data_ptr(), *p, M, N, K, K // 2, S, K // 2, S, ldo, 0, 1, stream)
    assert torch.equal(out.contiguous().view(BF16), want[which]), which
    for memory, view in ((m, out), (mq, q), (ms, s)):
      rest_is_untouched(memory, view)
  if v != -1:
    return
  mq, q = framed(M, K // 2, K // 2 + 20)
  ms, s = framed(M, S, S + 8)
  call(lib.cdit_mxfp4_quant, x.data_ptr(), 1, M, K, K, q.data_ptr(), K // 2 + 20, s.data_ptr(), S + 8, stream)
  assert torch.equal(q, a) and torch.equal(s, a_s)
  md, d = framed(M, 2 * K, 2 * K + 48)
  call(lib.cdit_mxfp4_dequant, q.data_ptr(), K // 2 + 20, s.data_ptr(), S + 8, M, K, d.data_ptr(), 1, K + 24, stream)
  assert torch.equal(d.contiguous().view(BF16), cd.mxfp4_dequant(a, a_s))
  for memory, view in ((mq, q), (ms, s), (md, d)):
    rest_is_untouched(memory, view)


@pytest.mark.parametrize("K,gap", [(96, 8), (96, 3), (1000, 8), (5120, 24), (12288, 8), (16416, 8)])
@pytest.mark.parametrize("codes", [False, True])
def test_nothing_but_the_norm_is_written(cd, K, gap, codes):
  import ctypes

  from cache_dit_amd import _native
  from test_mxfp4_cpu import NormArgs
  if codes and K % 32:
    pytest.skip("codes need whole blocks")
  lib, stream, M = _native.load(), torch.cuda.current_stream().cuda_stream, 7
  x, b, g = rand(M, K, seed=1), rand(M, K, seed=2), rand(K, seed=3)
  ld, S = K + gap, mo.scale_bytes(K)
  (mh, h), (my, y) = framed(M, 2 * K, 2 * ld), framed(M, 2 * K, 2 * ld)
  (mq, q), (ms, s) = framed(M, K // 2, K // 2 + 4), framed(M, S, S + 4)
  args = NormArgs(M=M, K=K, x=x.data_ptr(), ld_x=K, branch=b.data_ptr(), ld_branch=K, x_dtype=1, dtype=1, gate=g.data_ptr(),
                  ld_gate=0, rows_per_gate=M, norm=2, residual_scale=1.0, eps=1e-6, h=h.data_ptr(), ld_h=ld, y=y.data_ptr(),
                  ld_y=ld)
  if codes:
    args.codes, args.ld_codes, args.code_scales, args.ld_code_scales = q.data_ptr(), K // 2 + 4, s.data_ptr(), S + 4
  assert lib.cdit_gate_residual_norm(ctypes.byref(args), stream) == 0, lib.cdit_last_error()
  torch.cuda.synchronize()
  want = cd.gate_residual_norm(x, b, g, norm="rms")
  assert torch.equal(h.contiguous().view(BF16), want[0])
  got = y.contiguous().view(BF16)
  # (rows off 16 bytes take the kernel that reads them again: another order of additions, a step of bf16 here and there)
  assert (got.float() - want[1].float()).abs().max() <= 2.0**-7 * want[1].float().abs().max()
  if codes:
    assert all(torch.equal(t, u) for t, u in zip((q, s), cd.mxfp4_quant(got)))
  for memory, view in ((mh, h), (my, y), (mq, q), (ms, s)):
    rest_is_untouched(memory, view)
