"""One Wan-shaped transformer block with its dense layers in blocks of e4m3: modulated norm and q|k|v projection in one pass, q | k norm and
rotation, attention, output projection, modulated norm and feed-forward, each with its residual.

  python examples/wan_block_fp8.py [--heads 12] [--frames 3 --rows 30 --cols 52] [--train] [--steps 10]

Random weights and inputs.  Inference keeps the dense layers' weights quantised between the steps; with --train the block is
differentiated, its three products per dense layer in e4m3 and the gradients of every weight in bf16.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from maxdiffusion_amd import attention_op, layer_op, ops  # noqa: E402

HEAD_DIM, FFN = 128, 4


def rotary_table(frames, rows, cols, device):
  """complex64 [1, 1, S, 64], one rotation per token and channel pair, the axes' shares as Wan has them (44, 42, 42 channels)."""
  at = torch.meshgrid(*(torch.arange(n, device=device, dtype=torch.float64) for n in (frames, rows, cols)), indexing="ij")
  angles = [p.reshape(-1, 1) * 10000.0 ** (-torch.arange(0, d, 2, device=device, dtype=torch.float64) / d) for p, d in zip(at, (44, 42, 42))]
  a = torch.cat(angles, dim=1)
  return torch.polar(torch.ones_like(a), a).to(torch.complex64)[None, None]


def make_block(heads, device, seed=0):
  gen = torch.Generator(device=device).manual_seed(seed)
  n = heads * HEAD_DIM

  def normal(*shape, std):
    return (torch.randn(shape, generator=gen, device=device) * std).to(torch.bfloat16)

  dense = {"qkv": (3 * n, n), "out": (n, n), "up": (FFN * n, n), "down": (n, FFN * n)}
  block = {name: normal(*shape, std=shape[1] ** -0.5) for name, shape in dense.items()}
  block.update({name + "_bias": normal(shape[0], std=0.02) for name, shape in dense.items()})
  block.update({name: 1 + normal(n, std=0.1) for name in ("norm_q", "norm_k")})
  return block


def quantize(block):
  """The block as inference keeps it: the dense layers' weights in blocks of e4m3."""
  return {name: layer_op.quantize_weight(w) if w.dim() == 2 else w for name, w in block.items()}


def run_block(block, x, modulation, freqs, heads):
  """x [B, S, H*D] bf16; modulation [6, B, H*D] f32: shift, scale and gate of the attention half, then of the feed-forward half."""
  shift1, scale1, gate1, shift2, scale2, gate2 = modulation
  train = not isinstance(block["qkv"], ops.BlockQuant)

  def norm_dense(h, scale, shift, name, bias=True):
    b = block[name + "_bias"] if bias else None
    if train:
      return layer_op.hip_linear_fp8(layer_op.hip_layer_norm(h, scale, shift, weight_offset=1.0), block[name], b)
    return layer_op.hip_layer_norm_linear_fp8(h, scale, shift, block[name], b, weight_offset=1.0)

  qkv = norm_dense(x, scale1, shift1, "qkv", bias=False)  # (the prologue adds the bias)
  q, k, v = attention_op.hip_norm_rope_qkv(qkv, block["norm_q"], block["norm_k"], freqs, heads, bias=block["qkv_bias"], q_mul=ops.folded_q_mul(HEAD_DIM))
  op = attention_op.AttentionOp(attention_kernel="hip_flash", scale=ops.FOLDED_SCALE, heads=heads, dim_head=HEAD_DIM, dtype=torch.bfloat16)
  att = op.apply_attention(*(t.reshape(t.shape[0], t.shape[1], -1) for t in (q, k, v)))
  x = x + (gate1[:, None] * layer_op.hip_linear_fp8(att, block["out"], block["out_bias"])).to(x.dtype)
  h = torch.nn.functional.gelu(norm_dense(x, scale2, shift2, "up"), approximate="tanh")
  return x + (gate2[:, None] * layer_op.hip_linear_fp8(h, block["down"], block["down_bias"])).to(x.dtype)


def main():
  ap = argparse.ArgumentParser()
  ap.add_argument("--heads", type=int, default=12)
  ap.add_argument("--frames", type=int, default=3)
  ap.add_argument("--rows", type=int, default=30)
  ap.add_argument("--cols", type=int, default=52)
  ap.add_argument("--steps", type=int, default=10)
  ap.add_argument("--train", action="store_true")
  a = ap.parse_args()
  device = torch.device("cuda:0")
  n, tokens = a.heads * HEAD_DIM, a.frames * a.rows * a.cols
  block = make_block(a.heads, device)
  gen = torch.Generator(device=device).manual_seed(1)
  x = torch.randn((1, tokens, n), generator=gen, device=device).to(torch.bfloat16)
  modulation = 0.1 * torch.randn((6, 1, n), generator=gen, device=device)
  freqs = rotary_table(a.frames, a.rows, a.cols, device)
  if a.train:
    leaves = [t.requires_grad_(True) for t in block.values()]

    def step():
      y = run_block(block, x, modulation, freqs, a.heads)
      return torch.autograd.grad(y.float().square().mean(), leaves)
  else:
    kept = quantize(block)

    def step():
      with torch.no_grad():
        return run_block(kept, x, modulation, freqs, a.heads)
  step()
  torch.cuda.synchronize()
  start = time.perf_counter()
  for _ in range(a.steps):
    step()
  torch.cuda.synchronize()
  ms = (time.perf_counter() - start) / a.steps * 1e3
  print(f"{'training' if a.train else 'inference'}: {tokens} tokens x {n} channels, {ms:.3f} ms a step")


if __name__ == "__main__":
  main()
