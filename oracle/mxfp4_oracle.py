"""CPU restatement, in 64 bits, of the MXFP4 operators and of the block norm: what the tests compare the
kernels with. Written from the definitions in include/cdit_hip.h."""
import torch

GRID = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def scale_bytes(K):
  return (K + 127) // 128 * 4


def quantize(x):
  """x [M, K] -> codes uint8 [M, K/2], scales uint8 [M, scale_bytes(K)]."""
  M, K = x.shape
  b = x.double().reshape(M, K // 32, 32)
  top = b.abs().amax(-1)
  finite = torch.isfinite(top)
  mantissa, exponent = torch.frexp(torch.where(finite, top, 1.0))
  # (top = mantissa 2^exponent: a significand of 1.75 is a mantissa of .875)
  e = (exponent - 1 + 127 + (mantissa >= 0.875).long() - 2).clamp(1, 252)
  e = torch.where(top > 0, e, 1)
  e = torch.where(finite, e, 255)
  v = torch.where(finite[..., None], b * torch.exp2(127.0 - e.double())[..., None], torch.zeros_like(b))
  a = v.abs()
  above = torch.searchsorted(GRID, a.contiguous()).clamp(1, 7)
  low, high = a - GRID[above - 1], GRID[above] - a
  code = torch.where((low > high) | ((low == high) & (above % 2 == 0)), above, above - 1)
  sign = torch.signbit(b) & finite[..., None]
  code = (code + 8 * sign.long()).reshape(M, K).to(torch.uint8)
  scales = torch.full((M, scale_bytes(K)), 127, dtype=torch.uint8)
  scales[:, :K // 32] = e.to(torch.uint8)
  return code[:, 0::2] | (code[:, 1::2] << 4), scales


def dequantize(codes, scales):
  """The values, fp64 [M, K]."""
  M, K = codes.shape[0], 2 * codes.shape[1]
  c = torch.stack((codes & 15, codes >> 4), -1).reshape(M, K // 32, 32).long()
  v = GRID[c & 7] * torch.where(c > 7, -1.0, 1.0).double()
  e = scales[:, :K // 32].double()
  return torch.where((e == 255)[..., None], torch.nan, v * torch.exp2(e - 127)[..., None]).reshape(M, K)


def gelu_tanh(v):
  return torch.nn.functional.gelu(v, approximate="tanh")


def product(a, w, bias=None, gelu=False):
  """(result, the sum of the products' magnitudes) for fp64 a [M, K] and w [N, K]."""
  out = a @ w.t()
  if bias is not None:
    out = out + bias.double()
  return (gelu_tanh(out) if gelu else out), a.abs() @ w.abs().t()


def norm(v, kind, eps):
  if kind == "layer":
    v = v - v.mean(-1, keepdim=True)
  return v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)


def gate_residual_norm(x, branch, gate=None, shift=None, scale=None, norm_kind="layer", norm_weight=None, post_norm=None,
                       post_weight=None, residual_scale=1.0, eps=1e-6):
  """(h, y) in fp64; the vectors broadcast against x."""
  t = branch.double()
  if post_norm is not None:
    t = norm(t, post_norm, eps)
    if post_weight is not None:
      t = t * post_weight.double()
  h = residual_scale * x.double() + (t if gate is None else gate.double() * t)
  y = norm(h, norm_kind, eps)
  if norm_weight is not None:
    y = y * norm_weight.double()
  if scale is not None:
    y = y * (1 + scale.double())
  if shift is not None:
    y = y + shift.double()
  return h, y
