"""MXFP4 and the block norm without a GPU: the oracle against values worked out by hand, the refusals of the C
interface, the fake implementations, the layer selection."""
import ctypes

import pytest
import torch
from torch import nn

from cache_dit_amd import QuantizeConfig, _native, mxfp4
from cache_dit_amd import nn as cnn
from cache_dit_amd.quantization.policy import quantize_ao
from oracle import mxfp4_oracle as mo


def block(*values, K=32):
  x = torch.zeros(1, K)
  x[0, :len(values)] = torch.tensor(values)
  return x


@pytest.mark.parametrize("values,scale,codes", [
    ((6.0, ), 127, (7, )),  # the largest value of the grid under a scale of 1
    ((6.99, ), 127, (7, )),  # cut to it
    ((7.0, -7.0), 128, (6, 14)),  # 1.75 * 4: the scale is doubled, 3.5 is between 3 and 4: to the even code, 4
    ((4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), 127, (6, 0, 2, 2, 4, 4, 6, 6)),  # ties go to the even code
    ((4.0, -0.0, -0.2, 0.26), 127, (6, 8, 8, 1)),  # the sign is kept where the magnitude is lost
    ((2.0**-20, ), 127 - 22, (6, )),
    ((0.0, ), 1, (0, )),
    ((2.0**-130, ), 1, (0, )),  # below half a step of the smallest scale
    ((3.4028235e38, ), 252, (7, )),  # 2^128, in fp32: cut to 6 * 2^125
])
def test_oracle_by_hand(values, scale, codes):
  q, s = mo.quantize(block(*values))
  assert s[0].tolist() == [scale, 127, 127, 127]
  got = torch.stack((q[0] & 15, q[0] >> 4), -1).reshape(-1)
  assert got.tolist() == list(codes) + [0] * (32 - len(codes))


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_oracle_of_a_block_that_is_not_finite(bad):
  q, s = mo.quantize(block(1.0, bad, K=64))
  assert s[0].tolist() == [255, 1, 127, 127] and (q == 0).all()
  v = mo.dequantize(q, s)
  assert v[0, :32].isnan().all() and (v[0, 32:] == 0).all()


def test_oracle_is_off_by_a_fifth_of_the_largest_at_most():
  """With t the block's largest magnitude in units of the scale, 3.5 <= t < 7, and v a magnitude up to t: for v <= 4 the grid's
  steps are 1 at most, off by 1/2 <= t / 7; between 4 and 6 off by v - 4 or 6 - v, the less, at most (v - 4) / v <= 1/5 of t up to 5
  and less above; beyond 6 off by v - 6 < v / 7."""
  x = torch.randn(64, 256, generator=torch.Generator().manual_seed(0)).double()
  v = mo.dequantize(*mo.quantize(x))
  top = x.reshape(64, 8, 32).abs().amax(-1, keepdim=True)
  assert ((v - x).reshape(64, 8, 32).abs() <= top / 5).all()


# --------------------------------------------------------------------------- C interface

P = ctypes.c_void_p(64)
BF16 = 1


@pytest.fixture(scope="module")
def lib():
  if not _native.is_built():
    pytest.skip("libcdit_hip.so not built")
  return _native.load()


def refused(lib, status, text):
  assert status == 1 and text in lib.cdit_last_error(), (status, lib.cdit_last_error())


def test_refusals_of_the_quantizer(lib):
  f = lib.cdit_mxfp4_quant

  def call(x=P, dt=BF16, M=4, K=64, ld=64, q=P, ldq=32, s=P, lds=4):
    return f(x, dt, M, K, ld, q, ldq, s, lds, None)

  refused(lib, call(K=40), b"multiple of 32")
  refused(lib, call(M=-1), b"bad shape")
  refused(lib, call(K=2**29 + 32, ld=2**30, ldq=2**29, lds=2**25), b"bad shape")
  refused(lib, call(dt=5), b"dtype")
  refused(lib, call(ld=32), b"smaller than the row")
  refused(lib, call(ldq=16), b"smaller than the row")
  refused(lib, call(lds=0), b"smaller than the row")
  refused(lib, call(ld=68), b"16 bytes")
  refused(lib, call(x=ctypes.c_void_p(72)), b"16 bytes")
  refused(lib, call(ldq=34), b"must start on")
  refused(lib, call(lds=6), b"must start on")
  refused(lib, call(x=None), b"null pointer")
  refused(lib, call(q=None), b"null pointer")
  assert call(M=0) == 0 and call(K=0) == 0  # nothing to do
  refused(lib, lib.cdit_mxfp4_dequant(P, 32, P, 4, 4, 64, P, 9, 64, None), b"dtype")
  refused(lib, lib.cdit_mxfp4_dequant(P, 32, P, 4, 4, 64, P, BF16, 60, None), b"smaller than the row")
  refused(lib, lib.cdit_mxfp4_dequant(P, 32, None, 4, 4, 64, P, BF16, 64, None), b"null pointer")


def test_refusals_of_the_products(lib):

  def gemm(a=P, M=4, N=8, K=64, lda=32, ldb=32, ldbs=4, ldo=8, out=P, bias=None, epi=0, dt=BF16):
    return lib.cdit_mxfp4_gemm(a, P, P, P, bias, out, M, N, K, lda, 4, ldb, ldbs, ldo, epi, dt, None)

  refused(lib, gemm(K=48), b"multiple of 32")
  refused(lib, gemm(M=-1), b"bad shape")
  refused(lib, gemm(N=2**31), b"bad shape")
  refused(lib, gemm(lda=40), b"must start on 16")
  refused(lib, gemm(ldb=16), b"smaller than the row")
  refused(lib, gemm(ldbs=2), b"smaller than the row")
  refused(lib, gemm(ldo=7), b"smaller than the row")
  refused(lib, gemm(epi=2), b"epilogue")
  refused(lib, gemm(dt=3), b"out_dtype_id")
  refused(lib, gemm(a=None), b"null pointer")
  refused(lib, gemm(out=None), b"null pointer")
  refused(lib, gemm(out=ctypes.c_void_p(65)), b"misaligned")
  refused(lib, gemm(bias=ctypes.c_void_p(66), dt=2), b"misaligned")
  assert gemm(M=0) == 0 and gemm(N=0) == 0

  def linear(x=P, ws=P, M=4, K=64, ld=64, epi=0):
    return lib.cdit_mxfp4_linear(x, P, P, None, P, ws, P, M, 8, K, ld, 32, 4, 8, epi, None)

  refused(lib, linear(K=48), b"multiple of 32")
  refused(lib, linear(ws=ctypes.c_void_p(68)), b"workspaces")
  refused(lib, linear(ld=60), b"smaller than the row")
  refused(lib, linear(x=ctypes.c_void_p(66)), b"16 bytes")
  refused(lib, linear(epi=4), b"epilogue")

  def weight_only(x=P, M=4, N=8, K=64, ld=64, ldo=8):
    return lib.cdit_w4a16_gemm(x, P, P, None, P, M, N, K, ld, 32, 4, ldo, 0, None)

  refused(lib, weight_only(K=16), b"multiple of 32")
  refused(lib, weight_only(x=None), b"null pointer")
  refused(lib, weight_only(ld=65), b"16 bytes")
  refused(lib, weight_only(ldo=4), b"smaller than the row")
  assert weight_only(M=0) == 0 and weight_only(N=0) == 0


class NormArgs(ctypes.Structure):
  _fields_ = [("M", ctypes.c_int64), ("K", ctypes.c_int64), ("x", ctypes.c_void_p), ("ld_x", ctypes.c_int64),
              ("branch", ctypes.c_void_p), ("ld_branch", ctypes.c_int64), ("x_dtype", ctypes.c_int), ("dtype", ctypes.c_int),
              ("gate", ctypes.c_void_p), ("ld_gate", ctypes.c_int64), ("rows_per_gate", ctypes.c_int64),
              ("shift", ctypes.c_void_p), ("ld_shift", ctypes.c_int64), ("rows_per_shift", ctypes.c_int64),
              ("scale", ctypes.c_void_p), ("ld_scale", ctypes.c_int64), ("rows_per_scale", ctypes.c_int64),
              ("norm_weight", ctypes.c_void_p), ("post_weight", ctypes.c_void_p), ("vec_f32", ctypes.c_int),
              ("norm", ctypes.c_int), ("post_norm", ctypes.c_int), ("residual_scale", ctypes.c_float), ("eps", ctypes.c_float),
              ("h", ctypes.c_void_p), ("ld_h", ctypes.c_int64), ("y", ctypes.c_void_p), ("ld_y", ctypes.c_int64),
              ("codes", ctypes.c_void_p), ("ld_codes", ctypes.c_int64), ("code_scales", ctypes.c_void_p),
              ("ld_code_scales", ctypes.c_int64)]


def test_refusals_of_the_block_norm(lib):

  def call(**kw):
    a = dict(M=4, K=64, x=64, ld_x=64, branch=64, ld_branch=64, x_dtype=BF16, dtype=BF16, norm=1, residual_scale=1.0, eps=1e-6,
             h=64, ld_h=64, y=64, ld_y=64)
    a.update(kw)
    return lib.cdit_gate_residual_norm(ctypes.byref(NormArgs(**a)), None)

  refused(lib, lib.cdit_gate_residual_norm(None, None), b"null pointer")
  refused(lib, call(M=-1), b"bad shape")
  refused(lib, call(K=2**31), b"bad shape")
  refused(lib, call(dtype=7), b"dtype")
  refused(lib, call(x_dtype=0), b"x_dtype")  # an fp16 stream beside a bf16 branch
  refused(lib, call(norm=0), b"norm")
  refused(lib, call(post_norm=3), b"post_norm")
  refused(lib, call(post_weight=64), b"without post_norm")
  refused(lib, call(eps=-1.0), b"eps")
  refused(lib, call(eps=float("nan")), b"eps")
  refused(lib, call(ld_x=63), b"leading dimension")
  refused(lib, call(ld_y=63), b"leading dimension")
  refused(lib, call(gate=64), b"rows_per")
  refused(lib, call(y=None), b"null pointer")
  refused(lib, call(h=None), b"null pointer")
  refused(lib, call(x=65), b"misaligned")
  refused(lib, call(scale=66, rows_per_scale=1, vec_f32=1), b"misaligned")
  refused(lib, call(codes=64, ld_codes=32, code_scales=None, ld_code_scales=4), b"null pointer")
  refused(lib, call(K=40, codes=64, ld_codes=32, code_scales=64, ld_code_scales=4), b"multiple of 32")
  assert call(M=0) == 0 and call(K=0) == 0


# ------------------------------------------------------------------------- fakes and Python


def test_fake_implementations():
  ops = torch.ops.cdit
  x = torch.empty(2, 5, 96, dtype=torch.bfloat16, device="meta")
  codes, scales = ops.mxfp4_quant(x)
  assert codes.shape == (2, 5, 48) and scales.shape == (2, 5, 4) and codes.dtype == scales.dtype == torch.uint8
  assert ops.mxfp4_dequant(codes, scales, 2).shape == x.shape and ops.mxfp4_dequant(codes, scales, 2).dtype == torch.float32
  w, ws = ops.mxfp4_quant(torch.empty(40, 96, dtype=torch.bfloat16, device="meta"))
  for out in (ops.mxfp4_linear(x, w, ws, None), ops.w4a16_mm(x, w, ws, None, 1)):
    assert out.shape == (2, 5, 40) and out.dtype == torch.bfloat16
  assert ops.mxfp4_mm(codes, scales, w, ws, None, 0).dtype == torch.float16
  args = (x.float(), x, None, None, None, None, None, 1, 0, 1.0, 1e-6)
  h, y = ops.gate_residual_norm(*args)
  assert h.shape == y.shape == x.shape and h.dtype == torch.float32 and y.dtype == torch.bfloat16
  h, codes, scales = ops.gate_residual_norm_mxfp4(*args)
  assert h.dtype == torch.float32 and codes.shape == (2, 5, 48) and scales.shape == (2, 5, 4)


def test_cpu_tensors_are_refused():
  x = torch.zeros(2, 64, dtype=torch.bfloat16)
  w, s = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8)
  for call in (lambda: mxfp4.mxfp4_quant(x), lambda: mxfp4.mxfp4_dequant(w, s), lambda: mxfp4.mxfp4_mm(w, s, w, s),
               lambda: mxfp4.mxfp4_linear(x, w, s), lambda: mxfp4.w4a16_mm(x, w, s), lambda: mxfp4.gate_residual_norm(x, x)):
    with pytest.raises(RuntimeError, match="no CPU path"):
      call()


def lin(i=64, o=64, dtype=torch.bfloat16, bias=True):
  return nn.Linear(i, o, bias=bias, dtype=dtype)


@pytest.mark.parametrize("qt", ["mxfp4", "mxfp4_weight_only"])
def test_layer_selection(qt):
  calls = []
  m = nn.Sequential(lin(), lin(96, 33), lin(48, 64), lin(dtype=torch.float32))
  quantize_ao(m, QuantizeConfig(quant_type=qt, exclude_layers=[]), _convert_fn=lambda l, t: calls.append((l, t)))
  assert [t for _, t in calls] == [qt] * 2 and calls[0][0] is m[0] and calls[1][0] is m[1]  # any N
  assert m._quantize_context.skipped_map[qt] == ["skip: 2 -> pattern<weight_shape(64, 48)[-1]%32!=0>",
                                                 "skip: 3 -> pattern<dtype(torch.float32)!=bfloat16>"]


def test_a_plan_of_several_types():
  class Block(nn.Module):

    def __init__(self):
      super().__init__()
      self.to_q, self.proj_mlp, self.proj_out = lin(), lin(), lin()

  class Net(nn.Module):
    _repeated_blocks = ["Block"]

    def __init__(self):
      super().__init__()
      self.blocks = nn.ModuleList([Block(), Block()])

  calls = []
  net = Net()
  quantize_ao(net, QuantizeConfig(precision_plan={"proj_mlp": "mxfp4", "proj_out": "mxfp4_weight_only"}),
              _convert_fn=lambda l, t: calls.append(t))
  assert sorted(calls) == ["float8_per_row"] * 2 + ["mxfp4"] * 2 + ["mxfp4_weight_only"] * 2


def test_conversions_that_are_refused():
  with pytest.raises(ValueError, match="multiple of 32"):
    cnn.convert_linear_(lin(48, 64), "mxfp4")
  if not torch.cuda.is_available():
    with pytest.raises(RuntimeError, match="no CPU path"):
      cnn.convert_linear_(lin(), "mxfp4_weight_only")
