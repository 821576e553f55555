"""Operators on microscaled 4-bit floating point (MXFP4), and the block norm that feeds them.

MXFP4 is the block format the matrix cores of gfx950 multiply as it is: E2M1 elements (0, .5, 1, 1.5, 2,
3, 4, 6 and a sign), one power-of-two scale per 32 of them along K. Here it serves what the reference's
4-bit types serve ("nvfp4", "nvfp4_weight_only",
src/cache_dit/quantization/torchao/quantize_ao.py:16-27).

A matrix [..., K] in MXFP4 is two uint8 tensors:

  codes   [..., K / 2]             element 2j in the low half of byte j, 2j + 1 in the high half
  scales  [..., 4 * ceil(K / 128)] byte b is the exponent e of the scale 2^(e - 127) of elements 32 b to
                                   32 b + 31, 255 for a block with a value that is not finite; bytes
                                   behind K / 32 (none for K a multiple of 128) are 127

K is a multiple of 32. Everything runs on the tensors' device and its current stream; outputs are fresh.
There is no CPU path and no gradient.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native
from .ops import (_as_rows, _reject_codes_only, _require_cuda, _shaped, _vector, decode_output_dtype, encode_output_dtype)

NORM_IDS = {None: 0, "layer": 1, "rms": 2}

torch.library.define("cdit::mxfp4_quant", "(Tensor x) -> (Tensor, Tensor)")
torch.library.define("cdit::mxfp4_dequant", "(Tensor codes, Tensor scales, int out_dtype_id) -> Tensor")
torch.library.define(
    "cdit::mxfp4_mm",
    "(Tensor a_codes, Tensor a_scales, Tensor b_codes, Tensor b_scales, Tensor? bias, int out_dtype_id, "
    "int epilogue=0) -> Tensor")
torch.library.define(
    "cdit::mxfp4_linear",
    "(Tensor x, Tensor weight, Tensor weight_scale, Tensor? bias, int epilogue=0) -> Tensor")
torch.library.define(
    "cdit::w4a16_mm",
    "(Tensor x, Tensor weight, Tensor weight_scale, Tensor? bias, int epilogue=0) -> Tensor")
_NORM_ARGS = ("(Tensor x, Tensor branch, Tensor? gate, Tensor? shift, Tensor? scale, Tensor? norm_weight, "
              "Tensor? post_weight, int norm, int post_norm, float residual_scale, float eps)")
torch.library.define("cdit::gate_residual_norm", _NORM_ARGS + " -> (Tensor, Tensor)")
torch.library.define("cdit::gate_residual_norm_mxfp4", _NORM_ARGS + " -> (Tensor, Tensor, Tensor)")


def scale_bytes(K: int) -> int:
  """Bytes of a row of scales."""
  return 4 * -(-K // 128)


def _results(launched):
  """The tensors of a launcher's (status, tensors...)."""
  if launched[0]:
    _native.check(launched[0])
  return launched[1:]


# ------------------------------------------------------------------------- quantizer and inverse


def _check_k(name: str, K: int) -> None:
  if K % 32 != 0:
    raise ValueError(f"{name}: the last dimension must be a multiple of 32, got {K}")


def _aligned_rows(x: torch.Tensor, bytes_: int) -> torch.Tensor:
  """x as rows that start on a multiple of `bytes_`; copied where they do not."""
  x2 = _as_rows(x)
  if (x2.data_ptr() % bytes_ or x2.stride(0) * x2.element_size() % bytes_ or x2.stride(0) < x2.shape[1]):
    x2 = x2.clone(memory_format=torch.contiguous_format)
  return x2


@torch.library.impl("cdit::mxfp4_quant", "CUDA")
def _mxfp4_quant(x):
  name = "cdit::mxfp4_quant"
  _reject_codes_only(name, x)
  launched = _native.host().mxfp4_quant(x)
  if launched is not None:
    return _results(launched)
  if x.dtype not in (torch.float16, torch.bfloat16, torch.float32):
    raise ValueError(f"{name}: x must be float16, bfloat16 or float32, got {x.dtype}")
  if x.dim() < 1:
    raise ValueError(f"{name}: x must have at least one dimension")
  K = x.shape[-1]
  _check_k(name, K)
  if x.numel() == 0:
    return (x.new_empty((*x.shape[:-1], K // 2), dtype=torch.uint8),
            x.new_empty((*x.shape[:-1], scale_bytes(K)), dtype=torch.uint8))
  codes, scales = _results(_native.host().mxfp4_quant(_aligned_rows(x, 16)))
  return codes.view(*x.shape[:-1], -1), scales.view(*x.shape[:-1], -1)


@torch.library.register_fake("cdit::mxfp4_quant")
def _fake_mxfp4_quant(x):
  K = x.shape[-1]
  return (x.new_empty((*x.shape[:-1], K // 2), dtype=torch.uint8),
          x.new_empty((*x.shape[:-1], scale_bytes(K)), dtype=torch.uint8))


def _check_mx(name: str, what: str, codes: torch.Tensor, scales: torch.Tensor) -> int:
  """K of a matrix in MXFP4, looked over."""
  if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
    raise ValueError(f"{name}: codes and scales of {what} must be uint8, got {codes.dtype} and {scales.dtype}")
  if codes.dim() < 1 or codes.shape[:-1] != scales.shape[:-1]:
    raise ValueError(f"{name}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} of {what} differ in "
                     "their leading dimensions")
  K = 2 * codes.shape[-1]
  _check_k(name, K)
  if scales.shape[-1] != scale_bytes(K):
    raise ValueError(f"{name}: {what} of K={K} needs {scale_bytes(K)} scale bytes a row, got {scales.shape[-1]}")
  if codes.device != scales.device:
    raise RuntimeError(f"{name}: codes and scales of {what} are on {codes.device} and {scales.device}")
  return K


@torch.library.impl("cdit::mxfp4_dequant", "CUDA")
def _mxfp4_dequant(codes, scales, out_dtype_id):
  name = "cdit::mxfp4_dequant"
  launched = _native.host().mxfp4_dequant(codes, scales, out_dtype_id)
  if launched is not None:
    return _results(launched)[0]
  out_dtype = decode_output_dtype(out_dtype_id)
  K = _check_mx(name, "the matrix", codes, scales)
  if codes.numel() == 0:
    return codes.new_empty((*codes.shape[:-1], K), dtype=out_dtype)
  out = _results(_native.host().mxfp4_dequant(_aligned_rows(codes, 4), _aligned_rows(scales, 4), out_dtype_id))[0]
  return out.view(*codes.shape[:-1], K)


@torch.library.register_fake("cdit::mxfp4_dequant")
def _fake_mxfp4_dequant(codes, scales, out_dtype_id):
  return codes.new_empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=decode_output_dtype(out_dtype_id))


# ------------------------------------------------------------------------------------ products


def _check_weight(name: str, K: int, weight: torch.Tensor, weight_scale: torch.Tensor,
                  bias: Optional[torch.Tensor], x: torch.Tensor) -> int:
  """N of a weight [N, K] in MXFP4 that is to be multiplied by rows of K."""
  if weight.dim() != 2:
    raise ValueError(f"{name}: the weight's codes must be [N, K/2], got shape {tuple(weight.shape)}")
  wk = _check_mx(name, "the weight", weight, weight_scale)
  if wk != K:
    raise ValueError(f"{name}: shape mismatch: rows of {K} and a weight of K={wk}")
  N = weight.shape[0]
  if bias is not None and bias.numel() != N:
    raise ValueError(f"{name}: bias must have {N} elements, got {bias.numel()}")
  for t in (weight, bias):
    if t is not None and t.device != x.device:
      raise RuntimeError(f"{name}: tensors on {x.device} and {t.device}")
  return N


def _bias_vector(bias: Optional[torch.Tensor], dtype: torch.dtype) -> Optional[torch.Tensor]:
  if bias is None:
    return None
  bias = _vector(bias, dtype)
  return bias if bias.data_ptr() % 16 == 0 else bias.clone()


def _empty_product(rows: torch.Tensor, N: int, dtype: torch.dtype, bias, epilogue: int) -> torch.Tensor:
  """What a product without rows, columns or a sum is: the epilogue of the bias."""
  out = torch.zeros((*rows.shape[:-1], N), dtype=torch.float32, device=rows.device)
  if bias is not None:
    out = out + bias.reshape(-1).float()
  if epilogue:
    out = torch.nn.functional.gelu(out, approximate="tanh")
  return out.to(dtype)


@torch.library.impl("cdit::mxfp4_mm", "CUDA")
def _mxfp4_mm(a_codes, a_scales, b_codes, b_scales, bias, out_dtype_id, epilogue=0):
  name = "cdit::mxfp4_mm"
  host = _native.host()
  launched = host.mxfp4_mm(a_codes, a_scales, b_codes, b_scales, bias, out_dtype_id, epilogue)
  if launched is not None:
    return _results(launched)[0]
  out_dtype = decode_output_dtype(out_dtype_id)
  K = _check_mx(name, "the activation", a_codes, a_scales)
  N = _check_weight(name, K, b_codes, b_scales, bias, a_codes)
  if K == 0 or N == 0 or a_codes.numel() == 0:
    return _empty_product(a_codes, N, out_dtype, bias, epilogue)
  out = _results(host.mxfp4_mm(_aligned_rows(a_codes, 16), _aligned_rows(a_scales, 4), _aligned_rows(b_codes, 16),
                               _aligned_rows(b_scales, 4), _bias_vector(bias, out_dtype), out_dtype_id, epilogue))[0]
  return _shaped(out, *a_codes.shape[:-1], N)


@torch.library.register_fake("cdit::mxfp4_mm")
def _fake_mxfp4_mm(a_codes, a_scales, b_codes, b_scales, bias, out_dtype_id, epilogue=0):
  return a_codes.new_empty((*a_codes.shape[:-1], b_codes.shape[0]), dtype=decode_output_dtype(out_dtype_id))


def _linear(name, launch, x, weight, weight_scale, bias, epilogue):
  _reject_codes_only(name, x)
  launched = launch(x, weight, weight_scale, bias, epilogue)
  if launched is not None:
    return _results(launched)[0]
  if x.dtype != torch.bfloat16:
    raise ValueError(f"{name}: x must be bfloat16, got {x.dtype}")
  if x.dim() < 1:
    raise ValueError(f"{name}: x must have at least one dimension")
  _check_k(name, x.shape[-1])
  N = _check_weight(name, x.shape[-1], weight, weight_scale, bias, x)
  if N == 0 or x.numel() == 0:
    return _empty_product(x, N, torch.bfloat16, bias, epilogue)
  out = _results(launch(_aligned_rows(x, 16), _aligned_rows(weight, 16), _aligned_rows(weight_scale, 4),
                        _bias_vector(bias, torch.bfloat16), epilogue))[0]
  return _shaped(out, *x.shape[:-1], N)


@torch.library.impl("cdit::mxfp4_linear", "CUDA")
def _mxfp4_linear(x, weight, weight_scale, bias, epilogue=0):
  return _linear("cdit::mxfp4_linear", _native.host().mxfp4_linear, x, weight, weight_scale, bias, epilogue)


@torch.library.impl("cdit::w4a16_mm", "CUDA")
def _w4a16_mm(x, weight, weight_scale, bias, epilogue=0):
  return _linear("cdit::w4a16_mm", _native.host().w4a16, x, weight, weight_scale, bias, epilogue)


@torch.library.register_fake("cdit::mxfp4_linear")
def _fake_mxfp4_linear(x, weight, weight_scale, bias, epilogue=0):
  return x.new_empty((*x.shape[:-1], weight.shape[0]), dtype=torch.bfloat16)


@torch.library.register_fake("cdit::w4a16_mm")
def _fake_w4a16_mm(x, weight, weight_scale, bias, epilogue=0):
  return x.new_empty((*x.shape[:-1], weight.shape[0]), dtype=torch.bfloat16)


# -------------------------------------------------------------------------------- the block norm


def _norm_vector(name, what, t, x, dtype, per_row):
  """A vector [K], or (per_row) vectors for x's first dimension [count, K], or for each of its rows
  [1, count, K]; contiguous, in dtype."""
  if t is None:
    return None
  K = x.shape[-1]
  if t.dim() < 1 or t.shape[-1] != K or t.numel() == 0:
    raise ValueError(f"{name}: {what} {tuple(t.shape)} does not hold vectors of K={K} elements")
  if t.device != x.device:
    raise RuntimeError(f"{name}: {what} is on {t.device}, x on {x.device}")
  count, M = t.numel() // K, x.numel() // K
  batch = x.dim() >= 2 and count == x.shape[0] and t.shape[0] == count
  rows = count == M and t.shape[:-1] == x.shape[:-1]
  if count != 1 and not (per_row and (batch or rows)):
    raise ValueError(f"{name}: {what} {tuple(t.shape)} for x {tuple(x.shape)}: expected one vector" +
                     (", one per index of x's first dimension, or one per row" if per_row else ""))
  if t.dtype != dtype:
    t = t.to(dtype)
  if count == 1:
    return t.reshape(K).contiguous()
  t = t.reshape(count, K).contiguous()
  return t if batch else t[None]


def _gate_residual_norm_general(name, x, branch, gate, shift, scale, norm_weight, post_weight, norm, post_norm,
                                residual_scale, eps, codes):
  _reject_codes_only(name, x, branch)
  launch = _native.host().gate_residual_norm
  launched = launch(x, branch, gate, shift, scale, norm_weight, post_weight, norm, post_norm, residual_scale, eps, codes)
  if launched is not None:
    return _results(launched)
  dtype = branch.dtype
  if dtype not in (torch.float16, torch.bfloat16, torch.float32) or x.dtype not in (dtype, torch.float32):
    raise ValueError(f"{name}: branch must be float16, bfloat16 or float32 and x of its type or float32, got "
                     f"{branch.dtype} and {x.dtype}")
  if x.shape != branch.shape or x.dim() < 1:
    raise ValueError(f"{name}: x {tuple(x.shape)} and branch {tuple(branch.shape)} must have one shape")
  if x.device != branch.device:
    raise RuntimeError(f"{name}: x is on {x.device}, branch on {branch.device}")
  K = x.shape[-1]
  if codes:
    _check_k(name, K)
  if x.numel() == 0:
    h = torch.empty_like(x, memory_format=torch.contiguous_format)
    if codes:
      return (h, *_fake_mxfp4_quant(branch))
    return h, torch.empty_like(branch, memory_format=torch.contiguous_format)
  vectors = (("gate", gate, True), ("shift", shift, True), ("scale", scale, True), ("norm_weight", norm_weight, False),
             ("post_weight", post_weight, False))
  # vectors of several types: all in fp32, which holds each of them
  same = all(t is None or t.dtype == dtype for _, t, _ in vectors)
  prepared = [_norm_vector(name, what, t, x, dtype if same else torch.float32, per_row) for what, t, per_row in vectors]
  # as [first dimension, rows of it, K]: what the launcher takes with every form of vectors
  first = x.shape[0] if x.dim() >= 2 else 1
  prepared = [t.reshape(first, -1, K) if t is not None and t.dim() == 3 else t for t in prepared]
  outs = _results(launch(x.contiguous().view(first, -1, K), branch.contiguous().view(first, -1, K), *prepared, norm,
                         post_norm, residual_scale, eps, codes))
  return tuple(o.view(*x.shape[:-1], o.shape[-1]) for o in outs)


@torch.library.impl("cdit::gate_residual_norm", "CUDA")
def _gate_residual_norm(*args):
  return _gate_residual_norm_general("cdit::gate_residual_norm", *args, False)


@torch.library.impl("cdit::gate_residual_norm_mxfp4", "CUDA")
def _gate_residual_norm_mxfp4(*args):
  return _gate_residual_norm_general("cdit::gate_residual_norm_mxfp4", *args, True)


@torch.library.register_fake("cdit::gate_residual_norm")
def _fake_gate_residual_norm(x, branch, *args):
  return x.new_empty(x.shape), branch.new_empty(branch.shape)


@torch.library.register_fake("cdit::gate_residual_norm_mxfp4")
def _fake_gate_residual_norm_mxfp4(x, branch, *args):
  return (x.new_empty(x.shape), *_fake_mxfp4_quant(branch))


# The overloads, looked up once: a call through the packet resolves them again each time.
_quant_op = torch.ops.cdit.mxfp4_quant.default
_dequant_op = torch.ops.cdit.mxfp4_dequant.default
_mm_op = torch.ops.cdit.mxfp4_mm.default
mxfp4_linear_op = torch.ops.cdit.mxfp4_linear.default
w4a16_mm_op = torch.ops.cdit.w4a16_mm.default
_norm_op = torch.ops.cdit.gate_residual_norm.default
_norm_mxfp4_op = torch.ops.cdit.gate_residual_norm_mxfp4.default

# --------------------------------------------------------------------------- python-level API


def mxfp4_quant(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
  """x [..., K] fp16, bf16 or fp32 -> (codes, scales). The scale of a block is 2 to the exponent of its
  largest magnitude less 2, twice that where the magnitude is 1.75 times a power of two or more;
  values are rounded to the nearest code, ties to the even one."""
  _require_cuda("mxfp4_quant", x)
  return _quant_op(x)


def mxfp4_dequant(codes: torch.Tensor, scales: torch.Tensor,
                  output_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
  """The values [..., K] that codes and scales stand for (exact in bf16 and fp32)."""
  _require_cuda("mxfp4_dequant", codes, scales)
  return _dequant_op(codes, scales, encode_output_dtype(output_dtype))


def mxfp4_mm(a_codes: torch.Tensor, a_scales: torch.Tensor, b_codes: torch.Tensor, b_scales: torch.Tensor,
             output_dtype: torch.dtype = torch.bfloat16, bias: Optional[torch.Tensor] = None,
             epilogue: int = 0) -> torch.Tensor:
  """a [..., K] times the transpose of b [N, K], both in MXFP4, plus bias [N], optionally through
  GELU-tanh (epilogue = _native.EPI_GELU_TANH), in fp16, bf16 or fp32. Sums are held in fp32: for each 64
  products the matrix instruction loses at most 3.7e-7 of the magnitudes' sum."""
  _require_cuda("mxfp4_mm", a_codes, a_scales, b_codes, b_scales, bias)
  return _mm_op(a_codes, a_scales, b_codes, b_scales, bias, encode_output_dtype(output_dtype), epilogue)


def mxfp4_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                 bias: Optional[torch.Tensor] = None, epilogue: int = 0) -> torch.Tensor:
  """A Linear forward with both sides in MXFP4: x bf16 [..., K] is quantized by the call, weight and
  weight_scale are the codes [N, K/2] and scales of mxfp4_quant. Returns bf16 [..., N]."""
  _require_cuda("mxfp4_linear", x, weight, weight_scale, bias)
  return mxfp4_linear_op(x, weight, weight_scale, bias, epilogue)


def w4a16_mm(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
             bias: Optional[torch.Tensor] = None, epilogue: int = 0) -> torch.Tensor:
  """A Linear forward with the weight alone in MXFP4 and x bf16 [..., K] as it is."""
  _require_cuda("w4a16_mm", x, weight, weight_scale, bias)
  return w4a16_mm_op(x, weight, weight_scale, bias, epilogue)


def gate_residual_norm(x: torch.Tensor, branch: torch.Tensor, gate: Optional[torch.Tensor] = None,
                       shift: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, *,
                       norm: str = "layer", norm_weight: Optional[torch.Tensor] = None,
                       post_norm: Optional[str] = None, post_weight: Optional[torch.Tensor] = None,
                       residual_scale: float = 1.0, eps: float = 1e-6, quant_type: Optional[str] = None):
  """What stands between two branches of a block, in one pass:

    h = residual_scale * x + gate * branch          (branch through its own norm first with post_norm)
    y = norm(h) * norm_weight * (1 + scale) + shift

  x, the residual stream, has the branch's type or is float32, and so is h; y has the branch's type.
  Everything is computed in fp32 and rounded where h and y are stored (y from the unrounded h).
  norm and post_norm: "layer" or "rms". gate, shift, scale: K elements, or as many for each index of x's
  first dimension (AdaLN: [B, 1, K]), or for each row of x; what is None is left out.
  Returns (h, y), or with quant_type="mxfp4" (h, codes, scales): y rounded to its type and then to
  MXFP4, as mxfp4_quant does it, for mxfp4_mm. For inference: a tensor that requires a gradient is
  refused while gradients are recorded.

  The reference runs these as separate tensor operations in the blocks it patches
  (src/cache_dit/caching/patch_functors/functor_flux.py:48-80)."""
  name = "gate_residual_norm"
  grad = torch.is_grad_enabled()
  for t in (x, branch, gate, shift, scale, norm_weight, post_weight):
    if t is not None:
      if not t.is_cuda:
        _require_cuda(name, t)
      if grad and t.requires_grad:
        raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad()")
  if norm not in ("layer", "rms") or post_norm not in NORM_IDS:
    raise ValueError(f"{name}: norm must be 'layer' or 'rms' and post_norm one of them or None, got {norm!r} and "
                     f"{post_norm!r}")
  if post_weight is not None and post_norm is None:
    raise ValueError(f"{name}: post_weight without post_norm")
  if quant_type not in (None, "mxfp4"):
    raise ValueError(f"{name}: quant_type must be None or 'mxfp4', got {quant_type!r}")
  if not eps >= 0:
    raise ValueError(f"{name}: eps must not be negative, got {eps}")
  op = _norm_op if quant_type is None else _norm_mxfp4_op
  return op(x, branch, gate, shift, scale, norm_weight, post_weight, NORM_IDS[norm], NORM_IDS[post_norm],
            float(residual_scale), float(eps))
