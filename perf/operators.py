"""The layers beside attention in a DiT block: layer norm (plain, affine or modulated), dense layers whose operands are
e4m3 with one power-of-two scale per block of 128, and the two fused; in inference and in training.

A case is one call on one batch that is already on the GPU.  `path` names the call:

  norm          y = h * (offset + w) + b,  h the normalised row; w and b per channel, or per batch element (`modulated`)
  norm_train    the same with its backward pass: y and the gradients of x, w and b
  linear        y = x8 w8^T + b from a quantised weight that the program keeps; x is quantised within the call
  norm_linear   the norm, its output quantised without being stored, and the product with a quantised weight
  linear_train  from a weight in bf16, with its backward pass, all three products in e4m3: y and the gradients of x, w and b

Products of e4m3 operands come out in bf16, whatever the type of the rows that were quantised.

Quantisation.  Over a block, m = max |x| and e is the smallest integer, -127 at least, with m <= 448 * 2^e; the block
holds x * 2^-e rounded to e4m3 and the byte e + 127.  Blocks are 1 x 128 along the axis that the product sums over, and
128 x 128 for weights.  A product by a power of two is exact, so that the stored values do not depend on how they were
computed.
"""
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-6


def listed():
  return [
      # the repository's smoke run (4 heads of 128, a 3 x 6 x 7 latent): what a modulated norm costs in latency
      dict(name="norm_tiny", path="norm", batch=1, tokens=126, channels=512, x="bf16", w="f32", modulated=True),
      # a short clip's f32 stream with a channel count that no vector divides, affine
      dict(name="norm_odd", path="norm", batch=2, tokens=1337, channels=1001, x="f32", w="f32", modulated=False),
      # Wan-14B on an 81-frame 720p clip: the norm in front of its self-attention, the largest
      dict(name="norm_wan14b", path="norm", batch=1, tokens=75600, channels=5120, x="bf16", w="f32", modulated=True),
      # training an image encoder of 16 heads of 80, a batch of frames of 257 tokens, affine
      dict(name="norm_encoder_train", path="norm_train", batch=16, tokens=257, channels=1280, x="bf16", w="bf16", modulated=False),
      # training one rank of Wan-14B, a quarter of the tokens: the modulated norm and the gradients of its modulation
      dict(name="norm_wan14b_train", path="norm_train", batch=1, tokens=18900, channels=5120, x="bf16", w="f32", modulated=True),
      # one token against the projection to six modulation vectors of Wan-14B: bound by the weight's bytes
      dict(name="linear_token", path="linear", batch=1, tokens=1, inner=5120, outer=30720, x="bf16", w="bf16"),
      # an image's 257 tokens projected from the encoder's width to the model's
      dict(name="linear_image", path="linear", batch=1, tokens=257, inner=1280, outer=5120, x="bf16", w="bf16"),
      # Wan-14B's output projection over the headline sequence
      dict(name="linear_wan14b", path="linear", batch=1, tokens=75600, inner=5120, outer=5120, x="bf16", w="bf16"),
      # LTX-2's audio stream (32 heads of 64), two short ragged clips: f32 rows, norm and q|k|v projection
      dict(name="norm_linear_audio", path="norm_linear", batch=2, tokens=1337, channels=2048, outer=6144, x="f32", w="f32", modulated=False),
      # Wan-1.3B at 480p: modulated norm and q|k|v projection
      dict(name="norm_linear_wan1.3b", path="norm_linear", batch=1, tokens=32760, channels=1536, outer=4608, x="bf16", w="f32", modulated=True),
      # a small head in training with sizes that nothing divides
      dict(name="linear_odd_train", path="linear_train", batch=3, tokens=111, inner=1000, outer=333, x="bf16", w="bf16"),
      # training one rank of Wan-14B: its q|k|v projection over a quarter of the tokens, the largest product
      dict(name="linear_wan14b_train", path="linear_train", batch=1, tokens=18900, inner=5120, outer=15360, x="bf16", w="bf16"),
  ]


def _log(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
  """A channel count: mostly a multiple of 64 or 8, now and then any."""
  n = _log(rng, lo, hi)
  step = rng.choice([1, 8, 64, 64])
  n = max(lo, n // step * step)
  return n + 8 if n == 3072 else n


def draw(rng):
  """One more case: any of the paths, sizes spread over the logarithm of their range, cut where it would cost more than the
  largest listed one."""
  most = work(listed()[-1])["flops"]
  while True:
    path = rng.choice(["norm", "norm_train", "linear", "norm_linear", "linear_train"])
    c = dict(path=path, batch=rng.choice([1, 1, 2, 3, 4]), tokens=_log(rng, 1, 75600), x=rng.choice(["bf16", "bf16", "f32"]))
    if path.startswith("norm"):
      c.update(channels=_width(rng, 64, 8192), w=rng.choice(["bf16", "f32"]), modulated=rng.random() < 0.5)
    else:
      c.update(inner=_width(rng, 64, 8192), w="bf16")
    if "linear" in path:
      c["outer"] = _width(rng, 16, 30720)
    if path == "linear_train":
      c["x"] = "bf16"
    w = work(c)
    if c["batch"] * c["tokens"] <= 75600 and w["flops"] <= most and w["bytes"] <= 2.5e9:
      return c


_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------ quantisation, plain
def _scale_byte(m):
  """The byte of a block's scale from its largest magnitude."""
  frac, exp = torch.frexp(m)  # m = frac * 2^exp, frac in [1/2, 1); 448 = 7/8 * 2^9
  e = torch.where(m > 0, exp - 9 + (frac > 0.875).to(exp.dtype), torch.full_like(exp, -127))
  return torch.where(torch.isfinite(m), e.clamp(min=-127) + 127, torch.full_like(e, 255))


def _pad(x, rows, cols):
  return torch.nn.functional.pad(x, (0, -x.shape[1] % cols, 0, -x.shape[0] % rows))


def _quant(x, block_rows):
  """x [R, C] -> (e4m3 values [R', C'], scale bytes [R' / block_rows, C' / 128]), padded with zeros to whole blocks."""
  x = _pad(x, block_rows, 128)
  b = x.view(x.shape[0] // block_rows, block_rows, x.shape[1] // 128, 128)
  byte = _scale_byte(b.abs().amax(dim=(1, 3)))
  unit = torch.exp2((127 - byte).to(x.dtype))[:, None, :, None]
  return (b * unit).to(torch.float8_e4m3fn).view_as(x), byte.to(torch.uint8)


def _dequant(v, byte, block_rows, rows, cols, dtype):
  """The numbers that the blocks stand for, [rows, cols]."""
  s = torch.exp2(byte.to(dtype) - 127)
  s = torch.where(byte == 255, torch.full_like(s, math.nan), s)
  v = v.to(dtype)
  return (v.view(v.shape[0] // block_rows, block_rows, -1, 128) * s[:, None, :, None]).view_as(v)[:rows, :cols]


def _held(x, block_rows):
  """x as the numbers that its quantised form stands for."""
  v, byte = _quant(x, block_rows)
  return _dequant(v, byte, block_rows, x.shape[0], x.shape[1], x.dtype)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
  c = dict(case)
  gen = torch.Generator(device=DEV).manual_seed(seed)

  def normal(*shape, dtype=torch.float32, std=1.0):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).mul_(std).to(dtype)

  B, T, path = c["batch"], c["tokens"], c["path"]
  C = c.get("channels", c.get("inner"))
  xt, wt = _TYPES[c["x"]], _TYPES[c["w"]]
  s = dict(case=c)
  # a residual stream: channels of different size, a few of them large and far from zero
  gain = torch.exp(normal(C, std=0.5))
  loud = torch.rand(C, generator=gen, device=DEV) < 0.01
  x = normal(B, T, C)
  if path.startswith("norm"):
    x = x * torch.where(loud, 8 * gain, gain) + torch.where(loud, 5.0, 0.1) * gain
    shape = (B, C) if c["modulated"] else (C,)
    s.update(weight=normal(*shape, std=0.2).add_(0.0 if c["modulated"] else 1.0).to(wt), bias=normal(*shape, std=0.2).to(wt))
  s["x"] = x.to(xt)
  if path in ("linear", "norm_linear"):
    N = c["outer"]
    v, byte = _quant(normal(N, C, std=C**-0.5), 128)
    # as the program keeps it: rows of whole blocks, the blocks' bytes padded to whole words
    values = v[:N].view(torch.uint8).contiguous()
    scales = torch.nn.functional.pad(byte, (0, -byte.shape[1] % 4)).contiguous()
    s.update(values=values, scales=scales, out_bias=normal(N, std=0.2, dtype=torch.bfloat16))
  elif path == "linear_train":
    N = c["outer"]
    s.update(weight=normal(N, C, std=C**-0.5).to(wt), bias=normal(N, std=0.2).to(wt))
  if path.endswith("train"):
    s["dy"] = normal(B, T, c.get("outer", C), std=1e-3).to(xt)
    for n in ("x", "weight", "bias"):  # what a training program asks gradients of
      s[n].requires_grad_(True)
  return s


def _offset(c):
  return 1.0 if c["modulated"] else 0.0


# ------------------------------------------------------------------------------------------------ one pass
def _run_own(s):
  from maxdiffusion_amd import layer_op as L
  from maxdiffusion_amd import ops

  c, path = s["case"], s["case"]["path"]
  if "values" in s:
    w8 = ops.BlockQuant(s["values"], s["scales"], c["outer"], c.get("channels", c.get("inner")), 128)
  if path == "linear":
    with torch.no_grad():
      return L.hip_linear_fp8(s["x"], w8, s["out_bias"])
  if path == "norm_linear":
    with torch.no_grad():
      return L.hip_layer_norm_linear_fp8(s["x"], s["weight"], s["bias"], w8, s["out_bias"], eps=EPS, weight_offset=_offset(c))
  if path == "norm":
    with torch.no_grad():
      return L.hip_layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, weight_offset=_offset(c))
  if path == "norm_train":
    y = L.hip_layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, weight_offset=_offset(c))
  else:
    y = L.hip_linear_fp8(s["x"], s["weight"], s["bias"])
  return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])


def _rows(t):
  """A per-channel or per-batch-element vector against [B, T, C]."""
  return t[:, None] if t.dim() == 2 else t


def _plain_norm(x, weight, bias, offset):
  mean = x.mean(dim=-1, keepdim=True)
  d = x - mean
  r = torch.rsqrt((d * d).mean(dim=-1, keepdim=True) + EPS)
  h = d * r
  return h * (_rows(weight) + offset) + _rows(bias), h, r


@torch.no_grad()
def _run_plain(s):
  c, path = s["case"], s["case"]["path"]
  x = s["x"].float()
  xt = s["x"].dtype
  if path == "linear" or path == "norm_linear":
    if path == "norm_linear":
      x = _plain_norm(x, s["weight"].float(), s["bias"].float(), _offset(c))[0]
    K, N = x.shape[-1], c["outer"]
    v, byte = s["values"].view(torch.float8_e4m3fn), s["scales"]
    w = _dequant(_pad8(v), byte[:, :v.shape[1] // 128], 128, N, K, torch.float32)
    y = _held(x.reshape(-1, K), 1) @ w.t() + s["out_bias"].float()
    return y.to(torch.bfloat16).view(c["batch"], c["tokens"], N)
  weight, bias = s["weight"].float(), s["bias"].float()
  if path == "norm":
    return _plain_norm(x, weight, bias, _offset(c))[0].to(xt)
  dy = s["dy"].float()
  if path == "norm_train":
    y, h, r = _plain_norm(x, weight, bias, _offset(c))
    a = dy * (_rows(weight) + _offset(c))
    dx = r * (a - a.mean(dim=-1, keepdim=True) - h * (a * h).mean(dim=-1, keepdim=True))
    over = 1 if c["modulated"] else (0, 1)
    return y.to(xt), dx.to(xt), (dy * h).sum(dim=over).to(s["weight"].dtype), dy.sum(dim=over).to(s["bias"].dtype)
  K, N = c["inner"], c["outer"]
  x, dy = x.view(-1, K), dy.view(-1, N)
  w = _held(weight, 128)
  y = _held(x, 1) @ w.t() + bias
  dx = _held(dy, 1) @ w
  dw = _held(dy.t(), 1) @ _held(x.t(), 1).t()
  shape = (c["batch"], c["tokens"])
  return y.to(xt).view(*shape, N), dx.to(xt).view(*shape, K), dw.to(s["weight"].dtype), dy.sum(dim=0).to(s["bias"].dtype)


def _pad8(v):
  """e4m3 rows padded with zero rows to whole blocks of 128."""
  return _pad(v.view(torch.uint8), 128, 128).view(torch.float8_e4m3fn)


def run(state):
  return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_blocks(x, block_rows):
  """x [R, C] in 64 bits as its blocks hold it: each block divided by its power of two, rounded to three bits behind the
  leading one (multiples of 2^-9 below 2^-6), half to even, and multiplied back."""
  R, C = x.shape
  t = torch.nn.functional.pad(x, (0, -C % 128, 0, -R % block_rows))
  t = t.reshape(-1, block_rows, t.shape[1] // 128, 128)
  m = t.abs().amax(dim=(1, 3), keepdim=True)
  e = torch.ceil(torch.log2(m / 448)).clamp(min=-127)
  e = torch.where(448 * torch.exp2(e - 1) >= m, e - 1, e)  # a logarithm that came out a little too high or low
  e = torch.where(448 * torch.exp2(e) < m, e + 1, e).clamp(min=-127)
  t = t / torch.exp2(e)
  grid = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0**-6))) - 3)
  t = torch.round(t / grid) * grid * torch.exp2(e)
  return t.reshape(-1, t.shape[2] * 128)[:R, :C]


def exact(case, seed):
  s = prepare(case, seed)
  c, path = s["case"], s["case"]["path"]
  f = lambda n: s[n].detach().double()
  x = f("x")
  B, T, C = x.shape
  if path.startswith("norm"):
    w, b = f("weight") + _offset(c), f("bias")
    if c["modulated"]:
      w, b = w.unsqueeze(1), b.unsqueeze(1)
    var, mu = torch.var_mean(x, dim=2, correction=0, keepdim=True)
    sd = torch.sqrt(var + EPS)
    h = (x - mu) / sd
    if path == "norm":
      return h * w + b
    if path == "norm_train":
      g = f("dy")
      a = g * w
      dx = (a - a.sum(2, keepdim=True) / C - h * ((a * h).sum(2, keepdim=True) / C)) / sd
      dw, db = (g * h).sum(1), g.sum(1)
      return h * w + b, dx, (dw if c["modulated"] else dw.sum(0)), (db if c["modulated"] else db.sum(0))
    x = h * w + b
  N = c["outer"]
  x = x.reshape(B * T, C)
  if path != "linear_train":
    value = s["values"].view(torch.float8_e4m3fn)[:, :C].double()
    power = torch.exp2(s["scales"].double() - 127)
    w = value * power.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :C]
    return (torch.matmul(_exact_blocks(x, 1), w.T) + f("out_bias")).reshape(B, T, N)
  g = f("dy").reshape(B * T, N)
  w = _exact_blocks(f("weight"), 128)
  y = torch.matmul(_exact_blocks(x, 1), w.T) + f("bias")
  dx = torch.matmul(_exact_blocks(g, 1), w)
  dw = torch.matmul(_exact_blocks(g.T.contiguous(), 1), _exact_blocks(x.T.contiguous(), 1).T)
  return y.reshape(B, T, N), dx.reshape(B, T, C), dw, g.sum(0)


# ------------------------------------------------------------------------------------------------ what it cannot do without
def work(case):
  c, path = case, case["path"]
  M = c["batch"] * c["tokens"]
  C = c.get("channels", c.get("inner"))
  size = {"bf16": 2.0, "f32": 4.0}
  xb, wb = size[c["x"]], size[c["w"]]
  vectors = 2.0 * C * wb * (c["batch"] if c.get("modulated") else 1)
  if path == "norm":
    return {"bytes": 2 * M * C * xb + vectors, "flops": 8.0 * M * C}
  if path == "norm_train":
    return {"bytes": 4 * M * C * xb + 2 * vectors, "flops": 24.0 * M * C}
  N = c["outer"]
  if path == "linear_train":
    return {"bytes": 2 * M * (C + N) * xb + 2 * N * C * wb + 2 * N * wb, "flops": 6.0 * M * N * C}
  nbytes = M * C * xb + N * C + -(-N // 128) * -(-C // 128) + 2.0 * N + 2.0 * M * N
  return {"bytes": nbytes + (vectors if path == "norm_linear" else 0), "flops": 2.0 * M * N * C + (8.0 * M * C if path == "norm_linear" else 0)}
