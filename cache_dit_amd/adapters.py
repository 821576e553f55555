"""Low-rank adapters of many requests beside a shared projection.

A quantized weight is shared by all requests, and no adapter can be merged into it: its codes would have to be made again
for each. So the adapters stand beside it: out = base + scale[i] (x down[i]^T) up[i]^T for the adapter i of each row, whatever
the rows of a call name, in two launches for the whole batch.

`lora_add` is the operator on packed adapters, `LoraAdapters` packs them and holds them beside a Linear (`attach_lora_`),
`set_lora_ids` says which rows of the next calls use which. The reference merges adapters into the weights before it
quantizes them; requests with adapters of their own then need a copy of the model each.

Everything runs on the tensors' device and its current stream; outputs are fresh. There is no CPU path and no gradient.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch
from torch import nn

from . import _native
from .mxfp4 import _results
from .ops import FP8, _reject_codes_only, _require_cuda

MAX_RANK = 256

torch.library.define(
    "cdit::lora_add",
    "(Tensor base, Tensor x, Tensor down, Tensor up, Tensor ids, Tensor? scale, Tensor? rank, Tensor? x_scale, "
    "int epilogue=0) -> Tensor")


def _lora_add(base, x, down, up, ids, scale, rank, x_scale, epilogue=0):
  name = "cdit::lora_add"
  _reject_codes_only(name, x)
  launch = _native.host().lora_add
  launched = launch(base, x, down, up, ids, scale, rank, x_scale, epilogue)
  if launched is not None:
    return _results(launched)[0]
  if base.dtype != torch.bfloat16 or x.dtype not in (torch.bfloat16, FP8):
    raise ValueError(f"{name}: base must be bfloat16 and x bfloat16 or float8_e4m3fn, got {base.dtype} and {x.dtype}")
  if (x.dtype == FP8) != (x_scale is not None):
    raise ValueError(f"{name}: x_scale goes with float8_e4m3fn codes, and they with it")
  if x.dim() < 1 or x.dim() != base.dim() or x.shape[:-1] != base.shape[:-1]:
    raise ValueError(f"{name}: base {tuple(base.shape)} and x {tuple(x.shape)} differ in their leading dimensions")
  K, N = x.shape[-1], base.shape[-1]
  if down.dtype != torch.bfloat16 or up.dtype != torch.bfloat16 or down.dim() != 3 or up.dim() != 3:
    raise ValueError(f"{name}: down and up must be bfloat16 [adapters, R, K] and [adapters, N, R], got {down.dtype} "
                     f"{tuple(down.shape)} and {up.dtype} {tuple(up.shape)}")
  count, R = down.shape[:2]
  if down.shape[2] != K or up.shape != (count, N, R):
    raise ValueError(f"{name}: down {tuple(down.shape)} and up {tuple(up.shape)} for x of {K} and base of {N} values: expected "
                     f"[adapters, R, {K}] and [adapters, {N}, R]")
  if R % 16 or not 16 <= R <= MAX_RANK:
    raise ValueError(f"{name}: R must be a multiple of 16 up to {MAX_RANK} (ranks below it in `rank`), got {R}")
  if epilogue not in (_native.EPI_NONE, _native.EPI_GELU_TANH):
    raise ValueError(f"{name}: unknown epilogue {epilogue}")
  if ids.is_floating_point() or ids.is_complex() or ids.dtype == torch.bool:
    raise ValueError(f"{name}: ids must be whole numbers, got {ids.dtype}")
  if ids.dim() >= x.dim() or ids.shape != x.shape[:ids.dim()]:
    raise ValueError(f"{name}: ids {tuple(ids.shape)} for x {tuple(x.shape)}: expected one for all rows (no dimensions), or "
                     "one for each index of x's first dimensions")
  for what, t in (("scale", scale), ("rank", rank)):
    if t is not None and t.numel() != count:
      raise ValueError(f"{name}: {what} must hold {count} values, one an adapter, got {tuple(t.shape)}")
  rows = x.shape[:-1].numel()
  if max(K, N) >= 1 << 22 or rows >= 1 << 29:
    raise ValueError(f"{name}: x {tuple(x.shape)}, base {tuple(base.shape)}: must have fewer than 2^22 values a row and 2^29 rows")
  if x_scale is not None and x_scale.numel() != rows:
    raise ValueError(f"{name}: x_scale must hold {rows} values, one a row, got {tuple(x_scale.shape)}")
  for t in (x, down, up, ids, scale, rank, x_scale):
    if t is not None and t.device != base.device:
      raise RuntimeError(f"{name}: tensors on {base.device} and {t.device}")
  if rows == 0 or N == 0:
    return torch.empty(base.shape, dtype=base.dtype, device=base.device)
  if K == 0 or count == 0:  # nothing to add
    y = base.float()
    return (torch.nn.functional.gelu(y, approximate="tanh") if epilogue else y).to(base.dtype).contiguous()
  ids = ids.contiguous() if ids.dtype in (torch.int32, torch.int64) else ids.long()
  scale = None if scale is None else scale.reshape(count).float().contiguous()
  rank = None if rank is None else rank.reshape(count).int().contiguous()
  x_scale = None if x_scale is None else x_scale.reshape(rows).float().contiguous()
  up = up.contiguous()
  up = up if up.data_ptr() % 16 == 0 else up.clone()
  lead = base.shape[:-1]
  if x.dim() == 2:
    base = base if base.stride(1) == 1 and N <= base.stride(0) < 1 << 24 else base.contiguous().view(rows, N)
    x = x if x.stride(1) == 1 and K <= x.stride(0) < 1 << 24 else x.contiguous().view(rows, K)
  else:  # as many rows for each of the ids
    ids = ids.reshape(-1)
    base = base.contiguous().view(ids.numel(), -1, N)
    x = x.contiguous().view(ids.numel(), -1, K)
  launched = launch(base, x, down.contiguous(), up, ids, scale, rank, x_scale, epilogue)
  if launched is None:
    raise RuntimeError(f"{name}: arguments that were laid out for the kernels were not taken")
  return _results(launched)[0].view(*lead, N)


torch.library.impl("cdit::lora_add", "CUDA")(_lora_add)


@torch.library.register_fake("cdit::lora_add")
def _fake_lora_add(base, x, down, up, ids, scale, rank, x_scale, epilogue=0):
  return base.new_empty(base.shape)


_lora_op = torch.ops.cdit.lora_add.default


def lora_add(base: torch.Tensor, x: torch.Tensor, down: torch.Tensor, up: torch.Tensor, ids: torch.Tensor, *,
             scale: Optional[torch.Tensor] = None, rank: Optional[torch.Tensor] = None,
             x_scale: Optional[torch.Tensor] = None, epilogue: int = 0) -> torch.Tensor:
  """base + scale[i] (x down[i]^T) up[i]^T for the adapter i of each row, base alone for rows whose i is not in 0 ..
  adapters - 1 (-1, say), optionally through GELU-tanh (epilogue = _native.EPI_GELU_TANH).

  base bf16 [..., N] is the projection of x [..., K]: bf16, or the FP8 codes that the projection reads, with their scales
  x_scale [..., 1]. down bf16 [adapters, R, K] and up [adapters, N, R], R a multiple of 16 up to 256; rank [adapters] holds
  the ranks that are used of them (what lies behind is never looked at), scale [adapters] the adapters' strengths. ids, whole
  numbers: one for each index of x's first dimensions ([batch] for x [batch, tokens, K], or one a row), or one for all.
  Rows of one adapter next to one another are the fast case, any order is right. Sums are held in fp32, x down^T is carried on with
  16 bits, the result is rounded once; a row's result has the same bits whatever the rows beside it name. up holds finite numbers.
  For inference: a tensor that requires a gradient is refused while gradients are recorded."""
  name = "lora_add"
  grad = torch.is_grad_enabled()
  tensors = (base, x, down, up, ids, scale, rank, x_scale)
  for t in tensors:
    if t is not None:
      if not t.is_cuda:
        _require_cuda(name, t)
      if grad and t.requires_grad:
        raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad()")
  run = _lora_add if not torch.compiler.is_compiling() and _native.host().eager(*tensors) else _lora_op
  return run(*tensors, epilogue)


class LoraAdapters(nn.Module):
  """Adapters of one Linear, packed for lora_add. `pairs` holds (down [r, K], up [N, r]) of each, of any ranks up to 256;
  `scales` their strengths (alpha / r, say; 1 by default).

  `ids` (see lora_add) says which rows of the Linear's next inputs use which; None, the start, none do. The tensor is held, not
  copied: its values may be changed in place, between replays of a captured graph too."""

  def __init__(self, pairs: Sequence[Tuple[torch.Tensor, torch.Tensor]], scales: Optional[Sequence[float]] = None):
    super().__init__()
    pairs = list(pairs)
    if not pairs:
      raise ValueError("LoraAdapters: no adapters")
    scales = [1.0] * len(pairs) if scales is None else [float(s) for s in scales]
    if len(scales) != len(pairs):
      raise ValueError(f"LoraAdapters: {len(pairs)} adapters and {len(scales)} scales")
    first, last = pairs[0]
    if first.dim() != 2 or last.dim() != 2:
      raise ValueError("LoraAdapters: expected pairs of matrices (down [r, K], up [N, r])")
    K, N = first.shape[1], last.shape[0]
    for down, up in pairs:
      if down.dim() != 2 or up.dim() != 2 or down.shape[1] != K or up.shape[0] != N or down.shape[0] != up.shape[1]:
        raise ValueError(f"LoraAdapters: pairs must be (down [r, {K}], up [{N}, r]), got {tuple(down.shape)} and {tuple(up.shape)}")
      if not 1 <= down.shape[0] <= MAX_RANK:
        raise ValueError(f"LoraAdapters: ranks from 1 to {MAX_RANK}, got {down.shape[0]}")
    ranks = [down.shape[0] for down, _ in pairs]
    R, device = 16 * -(-max(ranks) // 16), first.device
    self.in_features, self.out_features = K, N
    self.register_buffer("down", torch.zeros((len(pairs), R, K), dtype=torch.bfloat16, device=device))
    self.register_buffer("up", torch.zeros((len(pairs), N, R), dtype=torch.bfloat16, device=device))
    self.register_buffer("scale", torch.tensor(scales, dtype=torch.float32, device=device))
    self.register_buffer("rank", torch.tensor(ranks, dtype=torch.int32, device=device))
    for i, (down, up) in enumerate(pairs):
      self.down[i, :ranks[i]] = down.detach()
      self.up[i, :, :ranks[i]] = up.detach()
    self._ids: Optional[torch.Tensor] = None

  @property
  def ids(self) -> Optional[torch.Tensor]:
    return self._ids

  @ids.setter
  def ids(self, ids: Optional[torch.Tensor]) -> None:
    _forget_outputs()
    self._ids = ids

  def extra_repr(self) -> str:
    return f"adapters={self.down.shape[0]}, in_features={self.in_features}, out_features={self.out_features}, R={self.down.shape[1]}"

  def forward(self, base: torch.Tensor, x, epilogue: int = 0) -> torch.Tensor:
    """lora_add for the Linear's output `base` and its input x, a tensor or FP8 (codes, scales)."""
    x, x_scale = x if isinstance(x, tuple) else (x, None)
    if x.dtype == torch.uint8:
      raise ValueError("LoraAdapters: the input has to be bfloat16 or FP8 codes; MXFP4 codes are not taken")
    return lora_add(base, x, self.down, self.up, self.ids, scale=self.scale, rank=self.rank, x_scale=x_scale, epilogue=epilogue)


def attach_lora_(linear: nn.Linear, adapters: LoraAdapters) -> nn.Linear:
  """Puts `adapters` beside a quantized Linear (in place of those it had) and returns it. A fused GELU is applied behind them."""
  from .nn import _Fp8LinearBase
  if not isinstance(linear, _Fp8LinearBase):
    raise TypeError("attach_lora_ expects a quantized Linear (an adapter can be merged into any other)")
  if (adapters.in_features, adapters.out_features) != (linear.in_features, linear.out_features):
    raise ValueError(f"attach_lora_: adapters of {adapters.in_features} x {adapters.out_features} beside a Linear of "
                     f"{linear.in_features} x {linear.out_features}")
  _forget_outputs()
  linear.add_module("lora", adapters.to(linear.weight.device))
  return linear


def _forget_outputs() -> None:
  """Outputs computed ahead for sibling Linears have their activation already, which is left to adapters that come with them."""
  from . import nn as quantized
  quantized.release_pending_outputs()
  quantized.release_precomputed(quantized._precomputed_holders)


def detach_lora_(module: nn.Module) -> int:
  """Takes the adapters of all quantized Linears under `module` away; returns of how many."""
  from .nn import _Fp8LinearBase
  _forget_outputs()
  n = 0
  for m in module.modules():
    if isinstance(m, _Fp8LinearBase) and m._modules.pop("lora", None) is not None:
      n += 1
  return n


def set_lora_ids(module: nn.Module, ids: Union[torch.Tensor, int, None]) -> int:
  """Which adapters the next calls of the Linears under `module` use: `ids` as in lora_add, a number for all rows, or None
  for none. A tensor is held as it is, by all of them: its values may be changed in place. Returns the number of Linears with
  adapters."""
  n = 0
  for m in module.modules():
    if isinstance(m, LoraAdapters):
      m.ids = torch.tensor(ids, dtype=torch.int32, device=m.down.device) if isinstance(ids, int) else ids
      n += 1
  return n
