"""A prompt encoder's layers in front of a DiT block: attention over packed sequences with grouped heads, and the RMS norm with the
residual's addition; in inference and in training.

A case is one call on one batch that is already on the GPU.  `path` names the call:

  attn          attention over packed sequences: sequence i of the batch is the rows offsets[i] .. offsets[i + 1] of q, k and v; causal
                or not; the heads of q in groups that share a head of k and v
  attn_token    one token of each sequence against its part of a cache with room for `room` tokens, of which some are filled
  attn_train    `attn` with its backward pass: the output and the gradients of q, k and v
  rms           s = x + residual and y = s * (mean s^2 + eps)^-1/2 * (offset + w) [+ b]; w and b per channel, or per batch
                element (`modulated`); y and s
  rms_train     the same with its backward pass from the gradients of y and s: y, s and the gradients of x, residual, w (and b)
  rms_linear    the norm, its output quantised to e4m3 without being stored, and the product with a quantised weight that the program
                keeps; the product and s

Causal: of a sequence with m queries and n keys, query i sees the keys up to i + n - m.

Quantisation.  Over a block, m = max |x| and e is the smallest integer, -127 at least, with m <= 448 * 2^e; the block
holds x * 2^-e rounded to e4m3 and the byte e + 127.  Blocks are 1 x 128 along the axis that the product sums over, and
128 x 128 for weights.
"""
import math
import random

import torch

own = False
DEV = "cuda"
EPS = 1e-6


def listed():
  return [
      # answering: one token for each of 16 sequences, against caches of up to 4,096 tokens, some just begun
      dict(name="token_batch", path="attn_token", sequences=16, room=4096, shortest=1, mix=1, heads=32, kv_heads=8, head_dim=128),
      # one token against a long document: the cache's bytes
      dict(name="token_long", path="attn_token", sequences=1, room=131072, shortest=131000, mix=2, heads=32, kv_heads=8, head_dim=128),
      # a single short prompt of the smallest encoder: what a call costs in latency
      dict(name="prompt_tiny", path="attn", causal=True, sequences=1, longest=77, shortest=77, mix=3, heads=12, kv_heads=12, head_dim=64),
      # a batch of prompts of 1 to 512 tokens, packed without padding
      dict(name="prompts_packed", path="attn", causal=True, sequences=16, longest=512, shortest=1, mix=4, heads=32, kv_heads=8, head_dim=128),
      # one document of 16,384 tokens, the largest
      dict(name="prompt_long", path="attn", causal=True, sequences=1, longest=16384, shortest=16384, mix=5, heads=32, kv_heads=8, head_dim=128),
      # image tokens of several sizes through an encoder that sees them all, heads of 80
      dict(name="images_packed", path="attn", causal=False, sequences=9, longest=1337, shortest=257, mix=6, heads=16, kv_heads=16, head_dim=80),
      # training on packed texts, 8 of 100 to 4,096 tokens
      dict(name="texts_train", path="attn_train", causal=True, sequences=8, longest=4096, shortest=100, mix=7, heads=32, kv_heads=8, head_dim=128),
      # training a small encoder: groups of three heads of 64, short ragged prompts
      dict(name="prompts_odd_train", path="attn_train", causal=True, sequences=23, longest=231, shortest=1, mix=8, heads=12, kv_heads=4, head_dim=64),
      # one token's hidden state: latency
      dict(name="rms_token", path="rms", batch=1, tokens=1, channels=5120, x="bf16", residual="bf16", w="bf16", modulated=False),
      # a video's stream at the headline size, modulated as adaLN does
      dict(name="rms_wan14b", path="rms", batch=1, tokens=75600, channels=5120, x="bf16", residual="bf16", w="f32", modulated=True),
      # training, with the stream in f32, and a channel count that no vector divides
      dict(name="rms_odd_train", path="rms_train", batch=2, tokens=1337, channels=1001, x="bf16", residual="f32", w="f32", modulated=False),
      # the norm in front of the k | v projection of 8 + 8 heads over 4,096 tokens, in e4m3
      dict(name="rms_linear_kv", path="rms_linear", batch=1, tokens=4096, channels=4096, outer=2048, x="bf16", residual="bf16", w="bf16", modulated=False),
  ]


def _log(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  """One more case: any of the paths, sizes spread over the logarithm of their range, cut where it would cost more than the
  largest listed ones."""
  while True:
    path = rng.choice(["attn", "attn", "attn_token", "attn_train", "rms", "rms_train", "rms_linear"])
    c = dict(path=path)
    if path.startswith("attn"):
      kv = rng.choice([1, 2, 4, 5, 8, 8, 16])
      c.update(sequences=_log(rng, 1, 100), mix=rng.randrange(1000), heads=kv * rng.choice([1, 1, 2, 3, 4, 5, 8]), kv_heads=kv,
               head_dim=rng.choice([64, 128, 128, 128, 40, 72, 80, 96]))
      if path == "attn_token":
        c["room"] = _log(rng, 16, 131072)
        c["shortest"] = _log(rng, 1, c["room"])
      else:
        c.update(causal=rng.random() < 0.75, longest=_log(rng, 1, 16384))
        c["shortest"] = _log(rng, 1, c["longest"])
    else:
      step = rng.choice([1, 8, 64, 64])
      c.update(batch=rng.choice([1, 1, 2, 3, 4]), tokens=_log(rng, 1, 75600), channels=_log(rng, 64, 8192) // step * step, modulated=rng.random() < 0.4)
      c["x"], c["residual"] = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
      c["w"] = rng.choice(["bf16", "f32"])
      if path == "rms_linear":
        c["outer"] = _log(rng, 16, 8192)
    w = work(c)
    rows = c["sequences"] * c["room"] if path == "attn_token" else sum(_lengths(c)) if path.startswith("attn") else c["batch"] * c["tokens"]
    if rows <= 131072 and w["flops"] <= 2.2e12 and w["bytes"] <= 3.2e9:
      return c


_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _lengths(case):
  """The sequences' lengths: the longest, the shortest, and others between them, spread over the logarithm."""
  rng = random.Random(case["mix"])
  lo, hi = case["shortest"], case.get("longest", case.get("room"))
  n = [hi, lo] + [_log(rng, lo, hi) for _ in range(case["sequences"])]
  n = n[:case["sequences"]]
  rng.shuffle(n)
  return n


def _starts(lengths):
  at = [0]
  for n in lengths:
    at.append(at[-1] + n)
  return at


# ------------------------------------------------------------------------------------------------ quantisation, plain
def _scale_byte(m):
  """The byte of a block's scale from its largest magnitude."""
  frac, exp = torch.frexp(m)  # m = frac * 2^exp, frac in [1/2, 1); 448 = 7/8 * 2^9
  e = torch.where(m > 0, exp - 9 + (frac > 0.875).to(exp.dtype), torch.full_like(exp, -127))
  return e.clamp(min=-127) + 127


def _quant(x, block_rows):
  """x [R, C] -> (e4m3 values [R', C'], scale bytes [R' / block_rows, C' / 128]), padded with zeros to whole blocks."""
  x = torch.nn.functional.pad(x, (0, -x.shape[1] % 128, 0, -x.shape[0] % block_rows))
  b = x.view(x.shape[0] // block_rows, block_rows, x.shape[1] // 128, 128)
  byte = _scale_byte(b.abs().amax(dim=(1, 3)))
  unit = torch.exp2((127 - byte).to(x.dtype))[:, None, :, None]
  return (b * unit).to(torch.float8_e4m3fn).view_as(x), byte.to(torch.uint8)


def _dequant(v, byte, block_rows, rows, cols):
  """The numbers that the blocks stand for, [rows, cols]."""
  v = v.float()
  s = torch.exp2(byte.float() - 127)
  return (v.view(v.shape[0] // block_rows, block_rows, -1, 128) * s[:, None, :, None]).view_as(v)[:rows, :cols]


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
  c = dict(case)
  gen = torch.Generator(device=DEV).manual_seed(seed)

  def normal(*shape, dtype=torch.float32, std=1.0):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).mul_(std).to(dtype)

  s = dict(case=c)
  path = c["path"]
  if path.startswith("attn"):
    n = _lengths(c)
    H, G, D = c["heads"], c["kv_heads"], c["head_dim"]
    bf16 = torch.bfloat16
    if path == "attn_token":
      starts = [i * c["room"] for i in range(c["sequences"] + 1)]
      s["q"] = normal(c["sequences"], H, D, dtype=bf16)
      kv = normal(2, starts[-1], G, D, dtype=bf16)
      s["k"], s["v"] = kv[0], kv[1]
      s["q_offsets"] = torch.arange(c["sequences"] + 1, dtype=torch.int32, device=DEV)
      s["k_lengths"] = torch.tensor(n, dtype=torch.int32).to(DEV)
      s["longest_q"], s["longest_k"] = 1, max(n)
    else:
      starts = _starts(n)
      rows = normal(starts[-1], H + 2 * G, D)
      # what a trained encoder has: heads whose queries lean one way, and a first token that many look at
      lean = normal(G, D, std=0.4)
      rows[:, :H] += lean.repeat_interleave(H // G, 0)
      first = torch.tensor([a for a, b in zip(starts, starts[1:]) if b > a], device=DEV)
      rows[first, H:H + G] += 2 * lean
      rows = rows.to(bf16)
      # inference: views of one projection's output; training: tensors of their own, as the rotation leaves them
      q, k, v = rows[:, :H], rows[:, H:H + G], rows[:, H + G:]
      if path == "attn_train":
        q, k, v = (t.contiguous().requires_grad_(True) for t in (q, k, v))
        s["dout"] = normal(starts[-1], H, D, dtype=bf16, std=1e-3)
      s.update(q=q, k=k, v=v)
      s["q_offsets"] = torch.tensor(starts, dtype=torch.int32).to(DEV)
      s["longest_q"] = s["longest_k"] = max(n)
    s["k_offsets"] = torch.tensor(starts, dtype=torch.int32).to(DEV)
    return s

  B, T, C = c["batch"], c["tokens"], c["channels"]
  xt, rt, wt = _TYPES[c["x"]], _TYPES[c["residual"]], _TYPES[c["w"]]
  # a residual stream: channels of different size, a few of them large and far from zero; and what a layer adds to it
  gain = torch.exp(normal(C, std=0.5))
  loud = torch.rand(C, generator=gen, device=DEV) < 0.01
  s["residual"] = (normal(B, T, C) * torch.where(loud, 8 * gain, gain) + torch.where(loud, 5.0, 0.1) * gain).to(rt)
  s["x"] = (normal(B, T, C, std=0.3) * gain).to(xt)
  shape = (B, C) if c["modulated"] else (C,)
  s["weight"] = normal(*shape, std=0.2).add_(0.0 if c["modulated"] else 1.0).to(wt)
  s["bias"] = normal(*shape, std=0.2).to(wt) if c["modulated"] else None
  if path == "rms_linear":
    N = c["outer"]
    v, byte = _quant(normal(N, C, std=C**-0.5), 128)
    # as the program keeps it: rows of whole blocks, the blocks' bytes padded to whole words
    s["values"] = v[:N].view(torch.uint8).contiguous()
    s["scales"] = torch.nn.functional.pad(byte, (0, -byte.shape[1] % 4)).contiguous()
  if path == "rms_train":
    s["dy"], s["ds"] = normal(B, T, C, std=1e-3).to(xt), normal(B, T, C, std=1e-3).to(rt)
    for n in ("x", "residual", "weight", "bias"):
      if s[n] is not None:
        s[n].requires_grad_(True)
  return s


def _offset(c):
  return 1.0 if c["modulated"] else 0.0


# ------------------------------------------------------------------------------------------------ one pass
def _run_own(s):
  from maxdiffusion_amd import attention_op as A
  from maxdiffusion_amd import layer_op as L
  from maxdiffusion_amd import ops

  c, path = s["case"], s["case"]["path"]
  if path.startswith("attn"):
    hints = dict(max_q=s["longest_q"], max_k=s["longest_k"])
    if path == "attn_train":
      y = A.hip_flash_packed(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], causal=c["causal"], **hints)
      return (y.detach(),) + torch.autograd.grad(y, (s["q"], s["k"], s["v"]), s["dout"])
    with torch.no_grad():
      if path == "attn_token":
        return A.hip_flash_packed(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], k_lengths=s["k_lengths"], **hints)
      return A.hip_flash_packed(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], causal=c["causal"], **hints)
  norm = dict(residual=s["residual"], eps=EPS, weight_offset=_offset(c))
  if path == "rms_train":
    y, total = L.hip_rms_norm(s["x"], s["weight"], s["bias"], **norm)
    leaves = [s[n] for n in ("x", "residual", "weight", "bias") if s[n] is not None]
    return (y.detach(), total.detach()) + torch.autograd.grad((y, total), leaves, (s["dy"], s["ds"]))
  with torch.no_grad():
    if path == "rms":
      return L.hip_rms_norm(s["x"], s["weight"], s["bias"], **norm)
    w8 = ops.BlockQuant(s["values"], s["scales"], c["outer"], c["channels"], 128)
    return L.hip_rms_norm_linear_fp8(s["x"], s["weight"], s["bias"], w8, **norm)


def _hidden(m, n, at, causal):
  """Which of n keys the queries `at`, of m, do not see."""
  keys = torch.arange(n, device=DEV)
  return keys[None] > (at + (n - m))[:, None] if causal else torch.zeros(len(at), n, dtype=torch.bool, device=DEV)


def _softmax(q, k, hide, scale):
  """q [h, g, m, D] against k [h, n, D] -> probabilities [h, g, m, n] in 32 bits, rows without a key all zero."""
  x = (q.flatten(1, 2) @ k.transpose(1, 2)).view(*q.shape[:3], -1).mul_(scale).masked_fill_(hide, -math.inf)
  top = x.amax(dim=-1, keepdim=True).clamp_(min=-1e30)
  x = torch.exp_(x.sub_(top))
  return x.div_(x.sum(dim=-1, keepdim=True).clamp_(min=1e-30))


def _plain_attention(s):
  c, train = s["case"], s["case"]["path"] == "attn_train"
  n = _lengths(c)
  token = c["path"] == "attn_token"
  m = [1] * len(n) if token else n
  q_at, k_at = _starts(m), [i * c["room"] for i in range(len(n))] if token else _starts(n)
  G, group, scale = c["kv_heads"], c["heads"] // c["kv_heads"], c["head_dim"]**-0.5
  # [h, g, rows, D] and [h, rows, D]
  by_group = lambda t: t.detach().unflatten(1, (G, group)).permute(1, 2, 0, 3)
  by_head = lambda t: t.detach().transpose(0, 1)
  q, k, v = by_group(s["q"]), by_head(s["k"]), by_head(s["v"])
  new = lambda name: torch.zeros(s[name].shape, device=DEV)
  out = new("q")
  if train:
    dout, dq, dk, dv = by_group(s["dout"]), new("q"), new("k"), new("v")
  for i in range(len(n)):
    hide = _hidden(m[i], n[i], torch.arange(m[i], device=DEV), c.get("causal", True))
    rows, keys = slice(q_at[i], q_at[i] + m[i]), slice(k_at[i], k_at[i] + n[i])
    step = max(1, min(G, 2**29 // (group * m[i] * n[i])))  # heads whose probabilities are held at a time
    for h in range(0, G, step):
      some = slice(h, h + step)
      qh, kh, vh = q[some, :, rows].float(), k[some, keys].float(), v[some, keys].float()
      p = _softmax(qh, kh, hide, scale)
      o = (p.flatten(1, 2) @ vh).view(qh.shape)
      by_group(out)[some, :, rows] = o
      if train:
        g = dout[some, :, rows].float()
        delta = (g * o).sum(dim=-1, keepdim=True)
        by_head(dv)[some, keys] = p.flatten(1, 2).transpose(1, 2) @ g.flatten(1, 2)
        p = p.mul_((g.flatten(1, 2) @ vh.transpose(1, 2)).view(p.shape).sub_(delta)).mul_(scale)
        by_group(dq)[some, :, rows] = (p.flatten(1, 2) @ kh).view(qh.shape)
        by_head(dk)[some, keys] = p.flatten(1, 2).transpose(1, 2) @ qh.flatten(1, 2)
  if train:
    return tuple(t.to(s["q"].dtype) for t in (out, dq, dk, dv))
  return out.to(s["q"].dtype)


def _rows(t):
  """A per-channel or per-batch-element vector against [B, T, C]."""
  return t[:, None] if t.dim() == 2 else t


@torch.no_grad()
def _run_plain(s):
  c, path = s["case"], s["case"]["path"]
  if path.startswith("attn"):
    return _plain_attention(s)
  xt, rt, wt = s["x"].dtype, s["residual"].dtype, s["weight"].dtype
  total = s["x"].float() + s["residual"].float()
  factor = _rows(s["weight"].float() + _offset(c))
  r = torch.rsqrt((total * total).mean(dim=-1, keepdim=True) + EPS)
  h = total * r
  y = h * factor
  if s["bias"] is not None:
    y = y + _rows(s["bias"].float())
  if path == "rms":
    return y.to(xt), total.to(rt)
  if path == "rms_train":
    dy = s["dy"].float()
    a = dy * factor
    ds = r * (a - h * (a * h).mean(dim=-1, keepdim=True)) + s["ds"].float()
    over = 1 if c["modulated"] else (0, 1)
    res = (y.to(xt), total.to(rt), ds.to(xt), ds.to(rt), (dy * h).sum(dim=over).to(wt))
    return res if s["bias"] is None else res + (dy.sum(dim=over).to(wt),)
  K, N = c["channels"], c["outer"]
  v = torch.nn.functional.pad(s["values"], (0, 0, 0, -N % 128)).view(torch.float8_e4m3fn)
  w = _dequant(v, s["scales"][:, :v.shape[1] // 128], 128, N, K)
  y = y.reshape(-1, K)
  y = _dequant(*_quant(y, 1), 1, y.shape[0], K) @ w.t()
  return y.to(torch.bfloat16).view(c["batch"], c["tokens"], N), total.to(rt)


def run(state):
  return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_attention(c, s):
  """Head by head and a stretch of queries at a time, by weights exp(logit - logsumexp)."""
  f = lambda n: s[n].detach().double()
  q, k, v = f("q"), f("k"), f("v")
  H, G, D = c["heads"], c["kv_heads"], c["head_dim"]
  train = c["path"] == "attn_train"
  n = _lengths(c)
  out = torch.zeros_like(q)
  if train:
    g = f("dout")
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
  rows = 0
  for i, keys in enumerate(n):
    queries = 1 if c["path"] == "attn_token" else keys
    begin = i * c["room"] if c["path"] == "attn_token" else rows
    K, V = k[begin:begin + keys], v[begin:begin + keys]
    for first in range(0, queries, 4096):
      last = min(queries, first + 4096)
      seen = keys if not c.get("causal", True) else keys - queries + last  # no query of the stretch sees more
      at = torch.arange(first, last, device=DEV)
      mask = torch.arange(seen, device=DEV).unsqueeze(0) <= at.unsqueeze(1) + (keys - queries) if c.get("causal", True) else None
      part = slice(rows + first, rows + last)
      for h in range(H):
        j = h * G // H
        logits = torch.matmul(q[part, h], K[:seen, j].T) / math.sqrt(D)
        if mask is not None:
          logits = torch.where(mask, logits, torch.full_like(logits, -math.inf))
        w = torch.exp(logits - torch.logsumexp(logits, dim=1, keepdim=True))
        o = torch.matmul(w, V[:seen, j])
        out[part, h] = o
        if train:
          go = g[part, h]
          dv[begin:begin + seen, j] += torch.matmul(w.T, go)
          dl = w * (torch.matmul(go, V[:seen, j].T) - torch.sum(go * o, 1, keepdim=True)) / math.sqrt(D)
          dq[part, h] = torch.matmul(dl, K[:seen, j])
          dk[begin:begin + seen, j] += torch.matmul(dl.T, q[part, h])
    rows += queries
  return (out, dq, dk, dv) if train else out


def _exact_blocks(x):
  """x [R, C] in 64 bits as its blocks of 1 x 128 hold it: each block divided by its power of two, rounded to three bits behind the
  leading one (multiples of 2^-9 below 2^-6), half to even, and multiplied back."""
  R, C = x.shape
  t = torch.nn.functional.pad(x, (0, -C % 128)).reshape(R, -1, 128)
  m = t.abs().amax(dim=2, keepdim=True)
  e = torch.ceil(torch.log2(m / 448)).clamp(min=-127)
  e = torch.where(448 * torch.exp2(e - 1) >= m, e - 1, e)  # a logarithm that came out a little too high or low
  e = torch.where(448 * torch.exp2(e) < m, e + 1, e).clamp(min=-127)
  t = t / torch.exp2(e)
  grid = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0**-6))) - 3)
  return (torch.round(t / grid) * grid * torch.exp2(e)).reshape(R, -1)[:, :C]


def exact(case, seed):
  s = prepare(case, seed)
  c, path = s["case"], s["case"]["path"]
  with torch.no_grad():
    if path.startswith("attn"):
      return _exact_attention(c, s)
    f = lambda n: s[n].detach().double()
    t = f("x") + f("residual")
    w = f("weight") + _offset(c)
    b = torch.zeros_like(w) if s["bias"] is None else f("bias")
    if c["modulated"]:
      w, b = w.unsqueeze(1), b.unsqueeze(1)
    C = c["channels"]
    rms = torch.sqrt(torch.linalg.vector_norm(t, dim=2, keepdim=True)**2 / C + EPS)
    h = t / rms
    if path == "rms":
      return h * w + b, t
    if path == "rms_train":
      g = f("dy")
      a = g * w
      d = (a - h * ((a * h).sum(2, keepdim=True) / C)) / rms + f("ds")
      dw, db = (g * h).sum(1), g.sum(1)
      if not c["modulated"]:
        dw, db = dw.sum(0), db.sum(0)
      return (h * w + b, t, d, d, dw) + (() if s["bias"] is None else (db,))
    N = c["outer"]
    value = s["values"].view(torch.float8_e4m3fn)[:, :C].double()
    power = torch.exp2(s["scales"].double() - 127)
    value = value * power.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :C]
    return torch.matmul(_exact_blocks((h * w + b).reshape(-1, C)), value.T).reshape(c["batch"], c["tokens"], N), t


# ------------------------------------------------------------------------------------------------ what it cannot do without
def work(case):
  c, path = case, case["path"]
  if path.startswith("attn"):
    n = _lengths(c)
    H, G, D = c["heads"], c["kv_heads"], c["head_dim"]
    m = [1] * len(n) if path == "attn_token" else n
    pairs = float(sum(a * (a + 1) // 2 if c.get("causal") else a * b for a, b in zip(m, n)))
    queries, keys = 2.0 * sum(m) * H * D, 2.0 * sum(n) * G * D
    if path == "attn_train":  # q, k, v, dout; out, dq, dk, dv
      return {"bytes": 4 * queries + 4 * keys, "flops": 14.0 * D * H * pairs}
    return {"bytes": 2 * queries + 2 * keys, "flops": 4.0 * D * H * pairs}
  M, C = c["batch"] * c["tokens"], c["channels"]
  size = {"bf16": 2.0, "f32": 4.0}
  xb, rb, wb = size[c["x"]], size[c["residual"]], size[c["w"]]
  vectors = C * wb * (2 * c["batch"] if c["modulated"] else 1)
  if path == "rms":
    return {"bytes": 2 * M * C * (xb + rb) + vectors, "flops": 6.0 * M * C}
  if path == "rms_train":  # x, residual, their gradients, y, s and theirs
    return {"bytes": 4 * M * C * (xb + rb) + 2 * vectors, "flops": 18.0 * M * C}
  N = c["outer"]
  return {"bytes": M * C * (xb + 2 * rb) + vectors + N * C + -(-N // 128) * -(-C // 128) + 2.0 * M * N, "flops": 2.0 * M * N * C + 6.0 * M * C}
