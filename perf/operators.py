"""What the speed of the MXFP4 operators and of the block norm is measured on.

Operators (all of `cache_dit_amd.ops`), and what they compute:

  mxfp4_quant, mxfp4_dequant
      Microscaled 4-bit floating point: along K, blocks of 32 values share a power-of-two scale
      2^(e - 127), e one byte, and each value is one of 0, .5, 1, 1.5, 2, 3, 4, 6 and a sign. Two
      values a byte (the lower half byte is the earlier one). e is the exponent of the block's
      largest magnitude less 2, one more where that magnitude is 1.75 times a power of two or
      above (it would be cut to 6/7 otherwise), in 1 .. 252; values are rounded to the nearest,
      ties to the even code. A row of scales has 4 ceil(K / 128) bytes, those behind K / 32 are 127.
  mxfp4_linear
      x W^T + bias (optionally GELU-tanh of it), x quantised per call, W kept in MXFP4.
  w4a16_mm
      The same with x as it is: only the weight is in MXFP4.
  gate_residual_norm
      What stands between two branches of a block: h = r x + gate * post(branch), y = norm(h) *
      weight * (1 + scale) + shift, with LayerNorm or RMSNorm; post: an RMSNorm of the branch or
      nothing. Returns h and y, or h and the MXFP4 codes of y.
  mxfp4_mm
      The product on codes: what follows gate_residual_norm's.

Kinds of cases: `quant` (there and back), `linear`, `weight_only`, `norm`, and `stage`: the norm,
its codes, and the feed-forward's first Linear on them, as a block runs them.
"""
import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
  return [
      # The embedded tokens of one prompt, in fp16: a launch, little more.
      {"name": "quant_prompt_77", "kind": "quant", "m": 77, "k": 4096, "dtype": "fp16"},
      # What the second feed-forward Linear of a video model reads: the largest activation there is.
      {"name": "quant_video_32760", "kind": "quant", "m": 32760, "k": 13824, "dtype": "bf16"},
      # Modulation from the timestep's embedding: one row, six vectors out; a stream of weights.
      {"name": "linear_modulation_1", "kind": "linear", "m": 1, "k": 5120, "n": 30720, "gelu": False},
      # The text embedder's Linear on a full prompt.
      {"name": "linear_text_512", "kind": "linear", "m": 512, "k": 4096, "n": 5120, "gelu": True},
      # Sizes that are multiples of nothing: an odd number of tokens and of outputs, K of 69 blocks.
      {"name": "linear_ragged_1357", "kind": "linear", "m": 1357, "k": 2208, "n": 4463, "gelu": False},
      # Feed-forward of the video model, the largest product.
      {"name": "linear_video_32760", "kind": "linear", "m": 32760, "k": 5120, "n": 13824, "gelu": True},
      # One token through a feed-forward Linear: what serving a language model does all the time.
      {"name": "weight_only_token_1", "kind": "weight_only", "m": 1, "k": 5120, "n": 13824, "gelu": False},
      # A prompt through the same width.
      {"name": "weight_only_prompt_77", "kind": "weight_only", "m": 77, "k": 4096, "n": 5120, "gelu": False},
      # An image's tokens, weights in 4 bits to fit and activations left alone.
      {"name": "weight_only_image_4608", "kind": "weight_only", "m": 4608, "k": 5120, "n": 5120, "gelu": False},
      # One token between attention and feed-forward with norms on both sides (RMS, weights).
      {"name": "norm_token_1", "kind": "norm", "batch": 1, "tokens": 1, "k": 5120, "dtype": "bf16", "stream": "bf16",
       "norm": "rms", "post": True, "mod": "weight"},
      # The video model's block: residual stream in fp32, one gate, scale and shift a batch entry.
      {"name": "norm_video_32760", "kind": "norm", "batch": 1, "tokens": 32760, "k": 5120, "dtype": "bf16",
       "stream": "fp32", "norm": "layer", "post": False, "mod": "batch"},
      # Norm, codes and the first feed-forward Linear of an image model's block, two images.
      {"name": "stage_image_2x4096", "kind": "stage", "batch": 2, "tokens": 4096, "k": 2560, "n": 10240, "dtype": "bf16",
       "stream": "bf16", "norm": "rms", "post": True, "mod": "batch"},
  ]


def _spread(rng, low, high, step=1):
  """A multiple of `step` between `low` and `high`, spread over the logarithm."""
  x = low * (high / low)**rng.random()
  return min(max(step * round(x / step), step * -(-low // step)), step * (high // step))


_MOST_BYTES, _MOST_VALUES, _MOST_PRODUCTS = 2 * 32760 * 13824, 32760 * 5120, 32760 * 5120 * 13824


def draw(rng):
  kind = rng.choice(("quant", "linear", "linear", "weight_only", "weight_only", "norm", "norm", "stage"))
  if kind == "quant":
    k, dtype = _spread(rng, 32, 15360, 32), rng.choice(("bf16", "bf16", "fp16", "fp32"))
    return {"kind": kind, "m": _spread(rng, 1, min(65536, _MOST_BYTES // (k * _BYTES[dtype]))), "k": k, "dtype": dtype}
  if kind in ("linear", "weight_only"):
    few = rng.random() < 0.4  # tokens of a step, conditioning rows
    k, n = _spread(rng, 128, 15360, 32), _spread(rng, 16, 30720, rng.choice((1, 8, 16, 64)))
    m = rng.randint(1, 16) if few else _spread(rng, 17, 16384)
    return {"kind": kind, "m": min(m, max(1, _MOST_PRODUCTS // (k * n))), "k": k, "n": n, "gelu": rng.random() < 0.3}
  dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
  c = {"kind": kind, "batch": rng.choice((1, 1, 2, 3)), "tokens": _spread(rng, 1, 10920),
       "k": _spread(rng, 64, 15360, rng.choice((1, 8, 64))), "dtype": dtype, "stream": rng.choice((dtype, "fp32")),
       "norm": rng.choice(("layer", "rms")), "post": rng.random() < 0.5,
       "mod": rng.choice(("batch", "batch", "weight", "token"))}
  if kind == "stage":
    c.update(k=_spread(rng, 128, 8192, 32), n=_spread(rng, 64, 16384, 16), dtype="bf16", stream=rng.choice(("bf16", "fp32")),
             tokens=_spread(rng, 1, 5460))
  c["tokens"] = min(c["tokens"], _MOST_VALUES // (c["batch"] * c["k"]))
  return c


# ------------------------------------------------------------------------------ preparation


def _normal(shape, g, std=1.0):
  return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).mul_(std)


def _activation(shape, g, dtype):
  """N(0, 1) in which 0.1 % of the channels are outliers (x 20)."""
  k = shape[-1]
  x = _normal(shape, g)
  x[..., torch.randint(0, k, (max(1, k // 1000), ), generator=g, device=DEV)] *= 20.0
  return x.to(dtype)


def _weight(n, k, g):
  """A Linear's weight in MXFP4, and its bias: N(0, 0.02) and N(0, 0.01), the channels of different size."""
  w = _normal((n, k), g, 0.02) * torch.exp(_normal((n, 1), g, 0.5))
  codes, scales = _codes(w)
  return {"w": codes, "w_scale": scales, "bias": _normal((n, ), g, 0.01).to(torch.bfloat16)}


def prepare(case, seed):
  g = torch.Generator(device=DEV).manual_seed(seed)
  s = {"case": case}
  if case["kind"] == "quant":
    s["x"] = _activation((case["m"], case["k"]), g, _DT[case["dtype"]])
    return s
  if case["kind"] in ("linear", "weight_only"):
    s["x"] = _activation((case["m"], case["k"]), g, torch.bfloat16)
    s.update(_weight(case["n"], case["k"], g))
    return s
  t, k, b, m = _DT[case["dtype"]], case["k"], case["batch"], case["tokens"]
  s["x"] = _activation((b, m, k), g, _DT[case["stream"]])
  s["branch"] = _normal((b, m, k), g, 0.7).to(t)
  s["gate"] = s["scale"] = s["shift"] = s["norm_weight"] = None
  s["post_weight"] = (1 + _normal((k, ), g, 0.1)).to(t) if case["post"] else None
  if case["mod"] == "weight":
    s["norm_weight"] = (1 + _normal((k, ), g, 0.1)).to(t)
  else:
    shape = (b, m if case["mod"] == "token" else 1, k)
    s["gate"], s["scale"], s["shift"] = (_normal(shape, g, d).to(t) for d in (0.5, 0.2, 0.2))
  if case["kind"] == "stage":
    s.update(_weight(case["n"], k, g))
  return s


# --------------------------------------------------------------------- one pass, in plain operations


def _block_exponents(blocks):
  """The scale bytes of fp32 blocks [..., 32], as int32 [..., 1]; 255 where a value is not finite."""
  top = blocks.abs().amax(-1, keepdim=True)
  e = (((top.view(torch.int32) + 0x200000) >> 23) - 2).clamp(1, 252)
  return torch.where(torch.isfinite(top), e, 255)


def _on_grid(v):
  """The nearest value of the 4-bit format, in fp32; ties go to the even code."""
  a = v.abs()
  step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
  return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), v)


def _power(e):
  """2^(e - 127) in fp32 for int32 e in 1 .. 254; NaN for 255."""
  return torch.where(e == 255, float("nan"), (e << 23).view(torch.float32))


def _quantised(x):
  """x rounded to MXFP4 along its last dimension, in fp32."""
  blocks = x.float().reshape(*x.shape[:-1], -1, 32)
  e = _block_exponents(blocks)
  return (_on_grid(blocks * _power(254 - e.clamp(max=253))) * _power(e)).reshape(x.shape)


def _codes(w):
  """Codes [N, K / 2] and scales [N, 4 ceil(K / 128)] of fp32 w [N, K]: what a program keeps of a weight."""
  n, k = w.shape
  blocks = w.reshape(n, k // 32, 32)
  e = _block_exponents(blocks)
  v = _on_grid(blocks * _power(254 - e.clamp(max=253)))
  a = v.abs()
  code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
  code = (code | (torch.signbit(v).to(torch.uint8) << 3)).reshape(n, k)
  scales = torch.full((n, 4 * -(-k // 128)), 127, dtype=torch.uint8, device=w.device)
  scales[:, :k // 32] = e[..., 0].to(torch.uint8)
  return code[:, 0::2] | (code[:, 1::2] << 4), scales


def _values(codes, scales):
  """The fp32 values that codes and scales stand for."""
  table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
  v = table[torch.stack((codes & 15, codes >> 4), -1).int()].reshape(codes.shape[0], -1, 32)
  return (v * _power(scales[:, :v.shape[1], None].int())).reshape(codes.shape[0], -1)


def _gelu_tanh(v):
  return 0.5 * v * (1 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))


def _product(x, s):
  """x in fp32 times the kept weight."""
  out = x.reshape(-1, x.shape[-1]) @ _values(s["w"], s["w_scale"]).t() + s["bias"].float()
  out = _gelu_tanh(out) if s["case"].get("gelu", s["case"]["kind"] == "stage") else out
  return out.to(torch.bfloat16).reshape(*x.shape[:-1], -1)


def _norm(v, kind, eps=1e-6):
  if kind == "layer":
    v = v - v.mean(-1, keepdim=True)
  return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)


def _gate_residual_norm(s):
  """(h, y) in fp32."""
  f = {name: None if s[name] is None else s[name].float()
       for name in ("x", "branch", "gate", "scale", "shift", "norm_weight", "post_weight")}
  t = f["branch"] if f["post_weight"] is None else _norm(f["branch"], "rms") * f["post_weight"]
  h = f["x"] + (t if f["gate"] is None else f["gate"] * t)
  y = _norm(h, s["case"]["norm"])
  if f["norm_weight"] is not None:
    y = y * f["norm_weight"]
  if f["scale"] is not None:
    y = y * (1 + f["scale"]) + f["shift"]
  return h, y


def run(s):
  kind = s["case"]["kind"]
  with torch.no_grad():
    if own:
      return _run_own(kind, s)
    if kind == "quant":
      return _quantised(s["x"]).to(s["x"].dtype)
    if kind == "linear":
      return _product(_quantised(s["x"]), s)
    if kind == "weight_only":
      return _product(s["x"].float(), s)
    h, y = _gate_residual_norm(s)
    h, y = h.to(s["x"].dtype), y.to(s["branch"].dtype)
    return (h, y) if kind == "norm" else (h, _product(_quantised(y), s))


def _run_own(kind, s):
  from cache_dit_amd import ops

  gelu = int(s["case"].get("gelu", kind == "stage"))  # the epilogue flag of the framework's GEMMs
  if kind == "quant":
    codes, scales = ops.mxfp4_quant(s["x"])
    return ops.mxfp4_dequant(codes, scales, s["x"].dtype)
  if kind == "linear":
    return ops.mxfp4_linear(s["x"], s["w"], s["w_scale"], s["bias"], epilogue=gelu)
  if kind == "weight_only":
    return ops.w4a16_mm(s["x"], s["w"], s["w_scale"], s["bias"], epilogue=gelu)
  block = dict(gate=s["gate"], shift=s["shift"], scale=s["scale"], norm=s["case"]["norm"], norm_weight=s["norm_weight"],
               post_norm="rms" if s["case"]["post"] else None, post_weight=s["post_weight"])
  if kind == "norm":
    return ops.gate_residual_norm(s["x"], s["branch"], **block)
  h, codes, scales = ops.gate_residual_norm(s["x"], s["branch"], **block, quant_type="mxfp4")
  return h, ops.mxfp4_mm(codes, scales, s["w"], s["w_scale"], torch.bfloat16, bias=s["bias"], epilogue=gelu)


# --------------------------------------------------------------------------- the definition, in 64 bits


def _exact_quantised(x):
  x = x.double()
  b = x.reshape(*x.shape[:-1], -1, 32)
  mantissa, exponent = torch.frexp(b.abs().amax(-1, keepdim=True))  # mantissa in [.5, 1)
  exponent = torch.where(mantissa >= 0.875, exponent + 1, exponent) - 1 - 2
  scale = torch.exp2(exponent.clamp(-126, 125).double())
  grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
  a = b.abs() / scale
  above = torch.searchsorted(grid, a).clamp(1, 7)  # grid[above - 1] < a <= grid[above]
  low, high = grid[above - 1], grid[above]
  up = (a - low > high - a) | ((a - low == high - a) & (above % 2 == 0))
  return (torch.where(up, high, low) * torch.sign(b) * scale).reshape(x.shape)


def _exact_weight(s):
  c, n = s["w"].long(), s["w"].shape[0]
  c = torch.stack((c % 16, c // 16), -1).reshape(n, -1, 32)
  two, one = (c % 8) // 2, c % 2  # exponent and mantissa bits
  v = torch.where(two == 0, 0.5 * one, (1 + 0.5 * one) * torch.exp2(two.double() - 1)) * (1 - 2.0 * (c // 8))
  e = s["w_scale"][:, :v.shape[1], None].double()
  return (v * torch.exp2(e - 127)).reshape(n, -1)


def _exact_product(x, s, gelu):
  out = torch.addmm(s["bias"].double(), x.reshape(-1, x.shape[-1]), _exact_weight(s).t())
  if gelu:
    out = torch.nn.functional.gelu(out, approximate="tanh")
  return out.reshape(*x.shape[:-1], -1)


def exact(case, seed):
  s = prepare(case, seed)
  kind = case["kind"]
  if kind == "quant":
    return _exact_quantised(s["x"])
  if kind in ("linear", "weight_only"):
    return _exact_product(_exact_quantised(s["x"]) if kind == "linear" else s["x"].double(), s, case["gelu"])
  x, t = s["x"].double(), s["branch"].double()
  if case["post"]:
    t = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * s["post_weight"].double()
  h = x + (t * s["gate"].double() if s["gate"] is not None else t)
  if case["norm"] == "layer":
    var, mean = torch.var_mean(h, -1, correction=0, keepdim=True)
    y = (h - mean) / torch.sqrt(var + 1e-6)
  else:
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6)
  if case["mod"] == "weight":
    y = y * s["norm_weight"].double()
  else:
    y = y + y * s["scale"].double() + s["shift"].double()
  if kind == "norm":
    return h, y
  return h, _exact_product(_exact_quantised(y.to(torch.bfloat16)), s, True)


# ------------------------------------------------------------------- what a pass cannot do without


def _weight_bytes(k, n):  # codes, scales, bias
  return n * (k // 2 + 4 * -(-k // 128) + 2)


def work(case):
  kind, k = case["kind"], case["k"]
  if kind == "quant":  # in, codes and scales written and read again, values out
    m = case["m"]
    return {"bytes": m * (2 * k * _BYTES[case["dtype"]] + 2 * (k // 2 + 4 * -(-k // 128))), "flops": 0.0}
  if kind in ("linear", "weight_only"):
    m, n = case["m"], case["n"]
    return {"bytes": 2 * m * k + _weight_bytes(k, n) + 2 * m * n, "flops": 2.0 * m * k * n}
  m, e = case["batch"] * case["tokens"], _BYTES[case["dtype"]]
  vectors = {"weight": 1, "batch": 3 * case["batch"], "token": 3 * m}[case["mod"]] + case["post"]
  through = m * k * (2 * _BYTES[case["stream"]] + e) + vectors * k * e
  if kind == "norm":
    return {"bytes": through + m * k * e, "flops": 0.0}
  return {"bytes": through + _weight_bytes(k, case["n"]) + 2 * m * case["n"], "flops": 2.0 * m * k * case["n"]}
