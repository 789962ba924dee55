"""The layers beside attention in a DiT block, as a model calls them: layer norm and dense layers in blocks of e4m3.

Differentiable where an input requires a gradient while autograd is recording; once, and not in forward mode: second derivatives and
tensors with a tangent raise NotImplementedError (paths relative to ``src/maxdiffusion/``):

  hip_layer_norm                FP32LayerNorm with adaLN's scale and shift, or affine   models/wan/transformers/transformer_wan.py:487
  hip_linear_fp8                a dense layer on e4m3 operands (the reference's qwix quantisation of dense layers, per tensor or
                                channel there, pipelines/wan/wan_pipeline.py:581-626)
  hip_layer_norm_linear_fp8     the norm and the dense layer behind it, the normalised rows never stored
"""
from __future__ import annotations

import torch

from . import _lib, ops
from .ops import BlockQuant

__all__ = ["hip_layer_norm", "hip_linear_fp8", "hip_layer_norm_linear_fp8", "quantize_weight", "BlockQuant"]


def _wants_grad(*ts) -> bool:
  return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _forms(*ts):
  """What a saved-tensor hook has to hand back as it was (strides are read again)."""
  return [None if t is None else (t.dtype, t.shape, t.device) for t in ts]


def _rows(x):
  """x [..., C] as the norm walks it: its last axis contiguous and the axes between the first and the last dense."""
  if x.dim() < 2:
    return x  # (refused by the call)
  return x if (x.stride(-1) == 1 or x.shape[-1] == 1) and ops.row_stride(x) is not None else x.contiguous()


class _HipLayerNorm(torch.autograd.Function):
  """Saved for the backward: the inputs only; the rows' statistics are computed again."""

  @staticmethod
  def forward(ctx, x, weight, bias, eps, weight_offset):
    ctx.save_for_backward(x, weight, bias)
    ctx.cfg, ctx.forms = (eps, weight_offset), _forms(x, weight, bias)
    return ops.layer_norm(x, weight, bias, eps, weight_offset)

  @staticmethod
  @_lib.first_order
  def backward(ctx, g):
    x, weight, bias = ctx.saved_tensors
    if _forms(x, weight, bias) != ctx.forms:
      raise ValueError("a tensor saved for the backward pass came back from its hook with another dtype, shape or device")
    dx, dw, db = ops.layer_norm_backward(x, weight, bias, _rows(g.to(x.dtype)), *ctx.cfg, needs_vectors=any(ctx.needs_input_grad[1:3]))
    return dx, dw, db, None, None


def hip_layer_norm(x, weight=None, bias=None, eps: float = 1e-6, weight_offset: float = 0.0):
  """x [..., C], bf16 or f32 -> the same: h * (weight_offset + weight) + bias, h the row less its mean, over its deviation.

  weight and bias [C], or, where x has three axes or more, per element of its first one [B, C] or [B, 1, C]: adaLN is (scale, shift,
  weight_offset=1).  Views that are not contiguous (chunks of a [B, 6, C]) are copied."""
  if x.is_cuda:
    y = _lib.host().layer_norm(x, weight, bias, eps, weight_offset)
    if y is not None:
      return y
  # what the native path leaves: views to be copied, nothing to compute, and every error
  _lib.no_tangents(x, weight, bias)
  weight, bias = (t if t is None else t.contiguous() for t in (weight, bias))
  if _wants_grad(x, weight, bias):
    return _HipLayerNorm.apply(_rows(x), weight, bias, eps, weight_offset)
  return ops.layer_norm(_rows(x), weight, bias, eps, weight_offset)


def quantize_weight(weight) -> BlockQuant:
  """A dense layer's weight [N, K] (bf16 or f32) in blocks of 128 x 128, as `hip_linear_fp8` takes it."""
  return ops.quant_block_e4m3(weight.contiguous(), block_rows=128)


def _matrix(x):
  if x.dim() == 0:
    raise ValueError("x must have shape [..., K], got a tensor without axes")
  return x.reshape(x.shape[:-1].numel(), x.shape[-1])  # (-1 stands for nothing where the last axis is empty)


class _HipLinearFp8(torch.autograd.Function):
  """y = x8 w8^T + b, dx = dy8 w8, dw = dy8'^T x8', ' quantised along the tokens.  Saved for the backward: the weight and x in
  e4m3, transposed (half the bytes of x in bf16); the forms come from one read of each tensor."""

  @staticmethod
  def forward(ctx, x, weight, bias):
    need_dx, need_dw, _ = ctx.needs_input_grad
    rows = _matrix(x)
    xq, xt = ops.quant_block_e4m3(rows, transposed=True) if need_dw else (ops.quant_block_e4m3(rows), None)
    wq, wt = ops.quant_block_e4m3(weight, block_rows=128, transposed=True) if need_dx else (ops.quant_block_e4m3(weight, block_rows=128), None)
    keep = [q for q in (xt, wt) if q is not None]
    ctx.save_for_backward(*(t for q in keep for t in (q.values, q.scales)))
    ctx.cfg = (x.shape, weight.shape, xt is not None, wt is not None, None if bias is None else bias.dtype)
    return ops.matmul_fp8_block_as(xq, wq, bias, x.shape[:-1])

  @staticmethod
  @_lib.first_order
  def backward(ctx, dy):
    shape, (n, k), has_x, has_w, bias_dtype = ctx.cfg
    saved = list(ctx.saved_tensors)
    m = shape[:-1].numel()
    xt = BlockQuant(saved.pop(0), saved.pop(0), k, m, 1) if has_x else None
    wt = BlockQuant(saved.pop(0), saved.pop(0), k, n, 128) if has_w else None
    g = dy.to(torch.bfloat16).reshape(m, n)
    g = g if g.stride(1) == 1 else g.contiguous()
    need_db = bias_dtype is not None and ctx.needs_input_grad[2]
    dx = dw = db = None
    if has_x or has_w or need_db:
      parts = list(_tuple(ops.quant_block_e4m3(g, plain=has_w or not has_x, transposed=has_x, sums=need_db)))
      gq = parts.pop(0) if has_w or not has_x else None
      if has_w:
        dx = ops.matmul_fp8_block_as(gq, wt, None, shape[:-1])
      if has_x:
        dw = ops.matmul_fp8_block(parts.pop(0), xt)
      if need_db:
        db = ops.sum_rows(parts.pop(0), bias_dtype)
    return dx, dw, db


def _tuple(x):
  return x if isinstance(x, tuple) else (x,)


def hip_linear_fp8(x, weight, bias=None):
  """x [..., K] -> bf16 [..., N], x weight^T + bias with both operands in blocks of e4m3 (x quantised here, 1 x 128).

  weight: a BlockQuant (`quantize_weight`), which a program keeps between calls, or, for training, a bf16 [N, K] tensor, quantised in
  every call.  bias bf16 or f32 [N], or None.  Differentiable with a bf16 x and weight; all three products run on e4m3 operands."""
  if isinstance(weight, BlockQuant):
    if x.is_cuda:
      y = _lib.host().linear_quantized(x, weight.values, weight.scales, weight.rows, weight.cols, weight.block_rows, bias, False, None, None, 0.0, 0.0)
      if y is not None:
        return y
    _lib.no_tangents(x, bias)
    if _wants_grad(x, bias):
      raise NotImplementedError("hip_linear_fp8 has no gradient through a quantised weight: give the weight itself, or call it under torch.no_grad()")
    rows = _matrix(x)
    rows = rows if rows.stride(1) == 1 else rows.contiguous()
    return ops.matmul_fp8_block_as(ops.quant_block_e4m3(rows), weight, bias, x.shape[:-1])
  if x.is_cuda and _wants_grad(x, weight, bias):
    y = _lib.host().linear_autograd(x, weight, bias)
    if y is not None:
      return y
  _lib.no_tangents(x, weight, bias)
  if weight.dim() != 2 or x.dim() == 0 or x.shape[-1] != weight.shape[1]:
    raise ValueError(f"weight must be a BlockQuant or a [N, K] tensor for an x [..., K], got {tuple(weight.shape)} for {tuple(x.shape)}")
  x, weight = (t if t.stride(-1) == 1 else t.contiguous() for t in (x, weight))
  if _wants_grad(x, weight, bias):
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
      raise ValueError(f"gradients of e4m3 products come in bf16: x and weight must be bf16, got {x.dtype} and {weight.dtype}")
    return _HipLinearFp8.apply(x, weight, bias)
  return hip_linear_fp8(x, quantize_weight(weight), bias)


def hip_layer_norm_linear_fp8(x, weight, bias, w8: BlockQuant, out_bias=None, eps: float = 1e-6, weight_offset: float = 0.0):
  """`hip_linear_fp8(hip_layer_norm(x, weight, bias, eps, weight_offset), w8, out_bias)` with the norm's f32 rows quantised where they are
  made: x is read once, and what the product reads is written once, a byte per channel.  Inference only."""
  if x.is_cuda:
    y = _lib.host().linear_quantized(x, w8.values, w8.scales, w8.rows, w8.cols, w8.block_rows, out_bias, True, weight, bias, eps, weight_offset)
    if y is not None:
      return y
  _lib.no_tangents(x, weight, bias, out_bias)
  if _wants_grad(x, weight, bias, out_bias):
    raise NotImplementedError("hip_layer_norm_linear_fp8 has no backward pass: use hip_layer_norm and hip_linear_fp8 for training")
  weight, bias = (t if t is None else t.contiguous() for t in (weight, bias))
  return ops.matmul_fp8_block_as(ops.layer_norm_quant(_rows(x), weight, bias, eps, weight_offset), w8, out_bias, x.shape[:-1])
