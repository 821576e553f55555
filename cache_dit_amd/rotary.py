"""Rotary positions: what stands between the q and k projections of a block and its attention.

A head's first `rot` values are pairs that are turned by an angle of the token's position. Two orders of pairs are in use:
"half" (value i and value i + rot / 2) and "interleaved" (values 2i and 2i + 1). Images and videos have a position per axis,
and each axis turns pairs of its own. The angles come from positions and inverse frequencies, made in fp64 by the kernel (no
table that grows with the context), or from tables of cosines and sines that a program has already.

The models this package serves turn q and k so, behind an RMSNorm of each head
(src/cache_dit/caching/patch_functors/functor_flux.py:48-80); the reference leaves both to separate tensor operations.

Everything runs on the tensors' device and its current stream; outputs are fresh. There is no CPU path and no gradient.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import _native
from .mxfp4 import _results
from .ops import _reject_codes_only, _require_cuda

LAYOUT_IDS = {"half": 0, "interleaved": 1}

torch.library.define(
    "cdit::rotary_embed",
    "(Tensor q, Tensor? k, Tensor? positions, Tensor? inv_freq, Tensor? cos, Tensor? sin, Tensor? q_weight, "
    "Tensor? k_weight, int layout, int[] section_ends, float scale, float eps) -> Tensor[]")


def _check_per_token(name, what, t, q, last):
  """[S] or [B, S] tokens of q [B, S, H, D] or [S, H, D], and `last` values for each (None: one)."""
  lead = t.shape if last is None else t.shape[:-1]
  if (last is not None and t.shape[-1:] != (last, )) or lead not in (q.shape[:-2], q.shape[-3:-2]):
    tail = "" if last is None else f" with {last} values each"
    raise ValueError(f"{name}: {what} {tuple(t.shape)} for q {tuple(q.shape)}: expected one for each token "
                     f"{tuple(q.shape[:-2])} or {tuple(q.shape[-3:-2])}{tail}")
  if t.device != q.device:
    raise RuntimeError(f"{name}: {what} is on {t.device}, q on {q.device}")


def _rotary_general(q, k, positions, inv_freq, cos, sin, q_weight, k_weight, layout, section_ends, scale, eps):
  name = "cdit::rotary_embed"
  _reject_codes_only(name, q, *([] if k is None else [k]))
  ends = list(section_ends)
  launch = _native.host().rotary
  launched = launch(q, k, positions, inv_freq, cos, sin, q_weight, k_weight, layout, ends, scale, eps)
  if launched is not None:
    return list(_results(launched))
  if q.dtype not in (torch.float16, torch.bfloat16, torch.float32):
    raise ValueError(f"{name}: q must be float16, bfloat16 or float32, got {q.dtype}")
  if q.dim() not in (3, 4):
    raise ValueError(f"{name}: q must be [tokens, heads, D] or [batch, tokens, heads, D], got {tuple(q.shape)}")
  D = q.shape[-1]
  if k is not None:
    if k.dtype != q.dtype or k.dim() != q.dim() or k.shape[-1] != D or k.shape[:-2] != q.shape[:-2]:
      raise ValueError(f"{name}: k {k.dtype} {tuple(k.shape)} must be as q {q.dtype} {tuple(q.shape)}, but for its heads")
    if k.device != q.device:
      raise RuntimeError(f"{name}: k is on {k.device}, q on {q.device}")
  if max(q.shape[-2], k.shape[-2] if k is not None else 0) > 32767:
    raise ValueError(f"{name}: at most 32767 heads, got {tuple(q.shape)}")
  if inv_freq is not None:
    if inv_freq.dim() != 1 or not inv_freq.is_floating_point() or inv_freq.device != q.device:
      raise ValueError(f"{name}: inv_freq must be a vector of floating point numbers on {q.device}, got {inv_freq.dtype} "
                       f"{tuple(inv_freq.shape)} on {inv_freq.device}")
    if positions.dtype in (torch.float16, torch.bfloat16):
      positions = positions.float()
    elif positions.dtype not in (torch.int32, torch.int64, torch.float32):
      if positions.is_floating_point() or positions.is_complex() or positions.dtype == torch.bool:
        raise ValueError(f"{name}: positions must be whole numbers or float32, got {positions.dtype}")
      positions = positions.long()
    if len(ends) > 4:
      raise ValueError(f"{name}: at most 4 axes, got {len(ends)}")
    _check_per_token(name, "positions", positions, q, len(ends) if ends else None)
    pairs, inv_freq = inv_freq.numel(), inv_freq.double().contiguous()
  else:
    if cos.shape != sin.shape or cos.dim() < 2:
      raise ValueError(f"{name}: cos {tuple(cos.shape)} and sin {tuple(sin.shape)} must have one shape [..., tokens, pairs]")
    pairs = cos.shape[-1]
    _check_per_token(name, "cos", cos, q, pairs)
    _check_per_token(name, "sin", sin, q, pairs)
    cos, sin = cos.float().contiguous(), sin.float().contiguous()
  if not 1 <= pairs <= D // 2 or D > 512:
    raise ValueError(f"{name}: {pairs} pairs in heads of {D} values: expected 1 to {D // 2}, and heads of at most 512")
  weights = []
  for what, w in (("q_weight", q_weight), ("k_weight", k_weight)):
    if w is not None:
      if w.numel() != D or not w.is_floating_point():
        raise ValueError(f"{name}: {what} {w.dtype} {tuple(w.shape)} does not hold {D} values")
      if w.device != q.device:
        raise RuntimeError(f"{name}: {what} is on {w.device}, q on {q.device}")
      w = w.reshape(D).float().contiguous()
    weights.append(w)
  if q.numel() == 0 and (k is None or k.numel() == 0):
    return [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k) if t is not None]
  if q.numel() == 0:  # no heads of q: what is left are k's
    return [torch.empty(q.shape, dtype=q.dtype, device=q.device),
            *_rotary_general(k, None, positions, inv_freq, cos, sin, weights[1], None, layout, ends, scale, eps)]
  q = q if q.stride(-1) == 1 else q.contiguous()
  k = k if k is None or k.stride(-1) == 1 else k.contiguous()
  launched = launch(q, k, positions, inv_freq, cos, sin, *weights, layout, ends, scale, eps)
  if launched is None:
    raise RuntimeError(f"{name}: arguments that were laid out for the kernels were not taken")
  return list(_results(launched))


torch.library.impl("cdit::rotary_embed", "CUDA")(_rotary_general)


@torch.library.register_fake("cdit::rotary_embed")
def _fake_rotary_embed(q, k, *args):
  return [q.new_empty(q.shape)] + ([] if k is None else [k.new_empty(k.shape)])


_rotary_op = torch.ops.cdit.rotary_embed.default


def rotary_embed(q: torch.Tensor, k: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                 inv_freq: Optional[torch.Tensor] = None, *, tables: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                 layout: str = "half", sections: Optional[Sequence[int]] = None, scale: float = 1.0,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6):
  """q and k with their positions, in one pass:

    v = x, or x / sqrt(mean(x^2) + eps) * weight over each head's values where a weight is given
    (a, b) -> scale * (a cos t - b sin t, a sin t + b cos t), t = positions * inv_freq

  q [batch, tokens, heads, D] or [tokens, heads, D], k the same with heads of its own (or None), fp16, bf16 or fp32, any
  strides (parts of a fused projection are taken as they are). D is at most 512. inv_freq holds one frequency for each of the
  1 to D / 2 pairs, float64 (see rotary_frequencies); the values behind the pairs go through (with the norm, without `scale`).
  positions [tokens] or [batch, tokens], int32, int64 or float32; with sections=(n0, n1, ...), pairs of each axis (up to 4,
  together all pairs), [..., axes]. tables=(cos, sin), [tokens, pairs] or [batch, tokens, pairs], stands in place of positions
  and inv_freq. layout: "half" pairs value i with value i + pairs, "interleaved" value 2i with 2i + 1.
  q_weight and k_weight [D] ask for the RMSNorm, each for itself.
  Everything is computed in fp32 (the angles in fp64) and rounded once. Returns (q, k), contiguous, or q where k is None. For
  inference: a tensor that requires a gradient is refused while gradients are recorded."""
  name = "rotary_embed"
  grad = torch.is_grad_enabled()
  cos, sin = (None, None) if tables is None else tables
  tensors = (q, k, positions, inv_freq, cos, sin, q_weight, k_weight)
  for t in tensors:
    if t is not None:
      if not t.is_cuda:
        _require_cuda(name, t)
      if grad and t.requires_grad:
        raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad()")
  if layout not in LAYOUT_IDS:
    raise ValueError(f"{name}: layout must be 'half' or 'interleaved', got {layout!r}")
  if (positions is None) != (inv_freq is None) or (inv_freq is None) == (tables is None):
    raise ValueError(f"{name}: either positions and inv_freq, or tables")
  if not eps >= 0:
    raise ValueError(f"{name}: eps must not be negative, got {eps}")
  if k is None and k_weight is not None:
    raise ValueError(f"{name}: k_weight without k")
  ends: List[int] = []
  if sections is not None:
    if inv_freq is None or any(int(n) < 0 for n in sections) or sum(sections) != inv_freq.numel():
      raise ValueError(f"{name}: sections {tuple(sections)} must be the numbers of pairs of each axis, "
                       f"{0 if inv_freq is None else inv_freq.numel()} together, with positions and inv_freq")
    at = 0
    for n in sections:
      at += int(n)
      ends.append(at)
  run = _rotary_general if not torch.compiler.is_compiling() and _native.host().eager(*tensors) else _rotary_op
  out = run(*tensors, LAYOUT_IDS[layout], ends, float(scale), float(eps))
  return out[0] if k is None else (out[0], out[1])


def rotary_frequencies(rot: int, theta: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: int = 4096, low: float = 1.0, high: float = 32.0,
                       device="cuda") -> Tuple[torch.Tensor, float]:
  """(inv_freq float64 [rot / 2], scale) for rotary_embed: theta^(-2i / rot), stretched for contexts `factor` times as long as
  the `original_length` tokens that the model was trained on:

    None          as trained; scale 1
    "linear"      all frequencies divided by factor
    "ntk"         theta times factor^(rot / (rot - 2)): the slowest frequency is divided by factor, the fastest stays
    "wavelength"  frequencies that turn less than `low` times in original_length are divided by factor, those that turn
                  more than `high` times stay, and between them the share kept is linear in the number of turns
    "yarn"        the share kept is linear in the frequency's index, between the (fractional) indices, rounded outwards, that
                  turn `high` and `low` times; scale is 0.1 ln(factor) + 1
  """
  name = "rotary_frequencies"
  if rot < 2 or rot % 2 or not theta > 1 or not factor >= 1:
    raise ValueError(f"{name}: an even rot, theta > 1 and factor >= 1, got {rot}, {theta}, {factor}")
  if scaling not in (None, "linear", "ntk", "wavelength", "yarn"):
    raise ValueError(f"{name}: scaling must be None, 'linear', 'ntk', 'wavelength' or 'yarn', got {scaling!r}")
  if not 0 < low < high or not original_length > 0:
    raise ValueError(f"{name}: 0 < low < high and a positive original_length, got {low}, {high}, {original_length}")
  if scaling == "ntk":
    if rot == 2:
      raise ValueError(f"{name}: 'ntk' needs more than one frequency")
    theta = theta * factor**(rot / (rot - 2))
  index = torch.arange(rot // 2, dtype=torch.float64)
  freq = torch.exp(index * (-2.0 * math.log(theta) / rot))
  scale = 1.0
  if scaling == "linear":
    freq = freq / factor
  elif scaling == "wavelength":
    turns = freq * (original_length / (2 * math.pi))
    kept = ((turns - low) / (high - low)).clamp(0, 1)
    freq = freq * (kept + (1 - kept) / factor)
  elif scaling == "yarn":
    def index_of(turns):  # theta^(-2i / rot) original_length = 2 pi turns
      return rot * math.log(original_length / (2 * math.pi * turns)) / (2 * math.log(theta))
    # (the ramp may end behind the last pair: its upper end is kept within the dimensions, not the pairs)
    first, last = max(math.floor(index_of(high)), 0), min(math.ceil(index_of(low)), rot - 1)
    kept = 1 - ((index - first) / max(last - first, 0.001)).clamp(0, 1)
    freq = freq * (kept + (1 - kept) / factor)
    scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
  return freq.to(device), scale
