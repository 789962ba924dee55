"""Host-side operators of the DiT attention hot path (torch tensors in HBM -> libmdattn.so).

torch is used for device memory and the current HIP stream only; every computation below is
a hand-written HIP kernel reached through the C ABI.  Tensors are logical [B, S, H, D] views
(any strides, D contiguous), so a [B, H, S, D] buffer is passed as ``x.permute(0, 2, 1, 3)``
and the reference's rank-3 [B, S, H*D] as ``x.view(B, S, H, D)`` -- never copied.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import Strides

__all__ = [
    "norm_rope_fullrow", "norm_rope_qkv", "norm_rope_perhead", "norm_rope_rows",
    "norm_rope_fullrow_backward", "norm_rope_perhead_backward", "norm_rope_rows_backward", "flash_attention", "flash_attention_backward", "flash_attention_backward_static", "flash_attention_fp8", "quant_e4m3", "key_mask_bias",
    "flash_attention_packed", "flash_attention_packed_backward",
    "layer_norm", "layer_norm_quant", "layer_norm_backward", "rms_norm", "rms_norm_quant", "rms_norm_backward", "BlockQuant", "quant_block_e4m3", "sum_rows", "matmul_fp8_block",
    "merge_partial", "flash_attention_merge", "finalize", "new_merge_state", "LSE_INIT", "FOLDED_SCALE", "folded_q_mul", "set_fwd_schedule", "FWD_SCHEDULES", "FP8_SOFTMAX_MODES",
]

LSE_INIT = -1e30

FWD_SCHEDULES = {"auto": 0, "pipelined8": 1, "pipelined4": 2, "flat": 3}


def set_fwd_schedule(schedule) -> int:
  """Test and tuning hook: forces the schedule of the bf16 forward at head dim 128 for the whole process ("auto"
  restores the choice by shape).  Returns the previous setting."""
  rc = _lib.load().mdattn_set_fwd_schedule(FWD_SCHEDULES.get(schedule, schedule))
  if rc < 0:
    _lib.check(rc, "mdattn_set_fwd_schedule")
  return rc

# Folding the softmax scale into the prologue: norm_rope_*(..., q_mul=folded_q_mul(D)) emits q * D^-1/2 * log2(e)
# (still one rounding), and the attention entry points, given scale=FOLDED_SCALE = ln 2, see scale * log2(e) == 1:
# their logits come out of the MFMA in log2 units and need no multiply.  Results are those of scale = D^-1/2.
FOLDED_SCALE = math.log(2.0)


def folded_q_mul(head_dim: int, scale: float | None = None) -> float:
  return (head_dim**-0.5 if scale is None else scale) * math.log2(math.e)


def _ptr(t):
  return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _stream():
  # the raw handle of the current stream of the current device (building a torch.cuda.Stream object around it costs 10 us)
  return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(_current_device()))


def _current_device() -> int:
  return torch._C._cuda_getDevice()  # (once there is a tensor on a device; half the time of torch.cuda.current_device)


def _check_dev(*ts):
  """All in the memory of the current device, whose stream the kernels run on: another one's may not be theirs to read."""
  device = None
  for t in ts:
    if t is None:
      continue
    if not t.is_cuda:
      raise ValueError("mdattn operators need tensors in device memory (cuda/HIP); there is no CPU path")
    if device is None:
      device = _current_device()
    if t.get_device() != device:
      raise ValueError(f"mdattn operators need their tensors on the current device, cuda:{device}: one is on cuda:{t.get_device()}")


def _strides(t: torch.Tensor) -> Strides:
  if t.dim() != 4 or t.stride(3) != 1:
    raise ValueError(f"expected a [B,S,H,D] view with contiguous D, got shape {tuple(t.shape)} strides {t.stride()}")
  return Strides(t.stride(0), t.stride(1), t.stride(2))


def _alloc_like_layout(b, s, h, d, layout: str, dtype, device):
  """Returns a logical [B,S,H,D] view over a fresh buffer laid out as `layout`."""
  if layout == "bshd":
    return torch.empty((b, s, h, d), dtype=dtype, device=device)
  if layout == "bhsd":
    return torch.empty((b, h, s, d), dtype=dtype, device=device).permute(0, 2, 1, 3)
  raise ValueError(f"unknown layout {layout!r} (want 'bshd' or 'bhsd')")


def _table(t, s, d, name):
  if t is None:
    return None
  if t.dtype != torch.float32 or tuple(t.shape) != (s, d // 2) or not t.is_contiguous():
    raise ValueError(f"{name} must be a contiguous float32 [S, D/2] = [{s}, {d // 2}] tensor, got {tuple(t.shape)} {t.dtype}")
  return t


class RopeTable:
  """A rotary table as a model made it, for the hooks of `attention_op`: the kernels read it in place.  `kind` is
  mdattn_host.h's MDATTN_TABLE_*: 0 cos, sin f32 [S, D/2]; 1 cos complex64 [S, D/2]; 2 cos, sin f32 [S, D] (repeated
  pairwise); 3 cos f32 [S, D/2, 2, 2].  Passed in place of `cos`, with `sin` None."""
  __slots__ = ("cos", "sin", "kind")

  def __init__(self, cos, sin, kind):
    self.cos, self.sin, self.kind = cos, sin, kind


def _table_args(cos, sin, s, d):
  """(cos pointer, sin pointer, kind) of the table arguments of a prologue call."""
  if isinstance(cos, RopeTable):
    if cos.kind:
      _check_dev(cos.cos, cos.sin)
      return _ptr(cos.cos), _ptr(cos.sin), cos.kind
    cos, sin = cos.cos, cos.sin
  _check_dev(cos, sin)
  return _ptr(_table(cos, s, d, "cos")), _ptr(_table(sin, s, d, "sin")), 0


def _check_weights(n, **weights):
  for name, w in weights.items():
    if w is not None and (w.dtype != torch.bfloat16 or w.numel() != n or not w.is_contiguous()):
      raise ValueError(f"{name} must be a contiguous bf16 tensor of {n} elements, got {tuple(w.shape)} {w.dtype} strides {w.stride()}")


def norm_rope_fullrow(q, k, wq, wk, cos, sin, heads: int, eps: float = 1e-6, out_layout: str = "bshd", q_mul: float = 1.0):
  """q, k: bf16 [B, S, H*D] (k may be None) -> (q_out, k_out) logical [B,S,H,D] views in `out_layout`.

  RMSNorm over H*D, then rotation of interleaved pairs by the [S, D/2] table (cos/sin None: norm only).
  `q_mul` is multiplied into q_out before its single rounding (see FOLDED_Q_MUL / FOLDED_SCALE).
  """
  _check_dev(q, k, wq, wk)
  if q.dim() != 3 or q.dtype != torch.bfloat16 or q.stride(2) != 1:
    raise ValueError("q must be bf16 [B, S, H*D] with a contiguous last axis")
  b, s, n = q.shape
  if n % heads:
    raise ValueError(f"inner dim {n} is not divisible by heads={heads}")
  d = n // heads
  if k is not None and (k.shape != q.shape or k.dtype != q.dtype or k.stride() != q.stride()):
    raise ValueError("k must match q in shape, dtype and strides")
  _check_weights(n, wq=wq, wk=wk if k is not None else None)
  pcos, psin, kind = _table_args(cos, sin, s, d)
  q_out = _alloc_like_layout(b, s, heads, d, out_layout, torch.bfloat16, q.device)
  k_out = _alloc_like_layout(b, s, heads, d, out_layout, torch.bfloat16, q.device) if k is not None else None
  st = _strides(q_out)
  rc = _lib.load().mdattn_host_norm_rope_fullrow(
      _stream(), _ptr(q), _ptr(k), _ptr(q_out), _ptr(k_out), _ptr(wq), _ptr(wk), pcos, psin, kind,
      b, s, heads, d, eps, q_mul, q.stride(0), q.stride(1), ctypes.byref(st))
  _lib.check(rc, "mdattn_norm_rope_fullrow")
  return q_out, k_out


def norm_rope_qkv(qkv, wq, wk, cos, sin, heads: int, bias=None, eps: float = 1e-6, out_layout: str = "bshd", q_mul: float = 1.0,
                  inplace: bool = False):
  """The prologue over the output of one fused q|k|v projection: qkv bf16 [B, S, 3*H*D] (column blocks q | k | v).

  bias bf16 [3*H*D] or None: the projections' biases, added in f32 before the statistics.  Returns (q, k, v) logical
  [B,S,H,D] views.  Without bias v is a view of the fused buffer itself (never copied).  inplace=True writes q, k
  (and the biased v) back into the fused buffer, which then holds the three attention operands."""
  _check_dev(qkv, wq, wk, bias)
  if qkv.dim() != 3 or qkv.dtype != torch.bfloat16 or qkv.stride(2) != 1 or qkv.shape[2] % (3 * heads):
    raise ValueError("qkv must be bf16 [B, S, 3*H*D] with a contiguous last axis")
  b, s, n3 = qkv.shape
  n = n3 // 3
  d = n // heads
  _check_weights(n, wq=wq, wk=wk)
  pcos, psin, kind = _table_args(cos, sin, s, d)
  if bias is not None and (bias.dtype != torch.bfloat16 or bias.numel() != n3 or not bias.is_contiguous()):
    raise ValueError("bias must be a contiguous bf16 [3*H*D] tensor")
  blocks = [qkv[:, :, i * n:(i + 1) * n].unflatten(2, (heads, d)) for i in range(3)]  # views of the fused buffer
  if inplace:
    q_out, k_out = blocks[0], blocks[1]
    v_out = blocks[2] if bias is not None else None
  else:
    q_out = _alloc_like_layout(b, s, heads, d, out_layout, torch.bfloat16, qkv.device)
    k_out = _alloc_like_layout(b, s, heads, d, out_layout, torch.bfloat16, qkv.device)
    v_out = _alloc_like_layout(b, s, heads, d, out_layout, torch.bfloat16, qkv.device) if bias is not None else None
  st = _strides(q_out)
  rc = _lib.load().mdattn_host_norm_rope_qkv(
      _stream(), _ptr(qkv), _ptr(bias), _ptr(q_out), _ptr(k_out), _ptr(v_out), _ptr(wq), _ptr(wk), pcos, psin, kind,
      b, s, heads, d, eps, q_mul, qkv.stride(0), qkv.stride(1), ctypes.byref(st))
  _lib.check(rc, "mdattn_norm_rope_qkv")
  return q_out, k_out, (v_out if v_out is not None else blocks[2])


def norm_rope_rows(x, w, cos=None, sin=None, heads: int = 1, mode: str = "none", eps: float = 1e-6, out_layout: str = "bshd"):
  """One tensor x [B,S,H*D] (bf16 or f32) -> bf16 logical [B,S,H,D]: full-row RMSNorm with the f32 weight w [H*D],
  then `mode` "none", "interleaved" (cos/sin f32 [B,S,H*D]) or "split" (cos/sin f32 [B,H,S,D/2])."""
  _check_dev(x, w, cos, sin)
  if x.dim() != 3 or x.dtype not in (torch.bfloat16, torch.float32) or x.stride(2) != 1:
    raise ValueError("x must be bf16 or f32 [B, S, H*D] with a contiguous last axis")
  b, s, n = x.shape
  if n % heads:
    raise ValueError(f"inner dim {n} is not divisible by heads={heads}")
  d = n // heads
  modes = {"none": 0, "interleaved": 1, "split": 2}
  if mode not in modes:
    raise ValueError(f"mode={mode!r} not supported. Choose between 'none', 'interleaved' and 'split'.")
  if w.dtype != torch.float32 or w.numel() != n or not w.is_contiguous():
    raise ValueError("w must be a contiguous f32 [H*D] tensor")
  if mode != "none":
    want = (b, s, n) if mode == "interleaved" else (b, heads, s, d // 2)
    for name, t in (("cos", cos), ("sin", sin)):
      if t is None or tuple(t.shape) != want or t.dtype != torch.float32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous f32 tensor of shape {want} for mode={mode!r}")
  out = _alloc_like_layout(b, s, heads, d, out_layout, torch.bfloat16, x.device)
  st = _strides(out)
  rc = _lib.load().mdattn_norm_rope_rows(
      _stream(), _ptr(x), int(x.dtype == torch.float32), _ptr(out), _ptr(w), _ptr(cos if mode != "none" else None),
      _ptr(sin if mode != "none" else None), modes[mode], b, s, heads, d, eps, x.stride(0), x.stride(1), ctypes.byref(st))
  _lib.check(rc, "mdattn_norm_rope_rows")
  return out


def norm_rope_perhead(q, k, wq, wk, cos, sin, eps: float = 1e-6, wq_txt=None, wk_txt=None, n_txt: int = 0,
                      out_layout: str = "bshd", q_mul: float = 1.0):
  """q, k: bf16 logical [B, S, H, D] views (k may be None); RMSNorm over D per head, then RoPE.
  `q_mul` is multiplied into q_out before its single rounding."""
  _check_dev(q, k, wq, wk, wq_txt, wk_txt)
  if q.dtype != torch.bfloat16:
    raise ValueError("q must be bf16")
  b, s, h, d = q.shape
  if k is not None and (k.shape != q.shape or k.stride() != q.stride() or k.dtype != q.dtype):
    raise ValueError("k must match q in shape, dtype and strides")
  _check_weights(d, wq=wq, wk=wk if k is not None else None, wq_txt=wq_txt, wk_txt=wk_txt if k is not None else None)
  pcos, psin, kind = _table_args(cos, sin, s, d)
  q_out = _alloc_like_layout(b, s, h, d, out_layout, torch.bfloat16, q.device)
  k_out = _alloc_like_layout(b, s, h, d, out_layout, torch.bfloat16, q.device) if k is not None else None
  si, so = _strides(q), _strides(q_out)
  rc = _lib.load().mdattn_host_norm_rope_perhead(
      _stream(), _ptr(q), _ptr(k), _ptr(q_out), _ptr(k_out), _ptr(wq), _ptr(wk), _ptr(wq_txt), _ptr(wk_txt), n_txt,
      pcos, psin, kind, b, s, h, d, eps, q_mul, ctypes.byref(si), ctypes.byref(so))
  _lib.check(rc, "mdattn_norm_rope_perhead")
  return q_out, k_out


def _bwd_workspace(rows: int, columns: int, device):
  n = _lib.load().mdattn_norm_rope_bwd_workspace_floats(rows, columns)
  return torch.empty(n, dtype=torch.float32, device=device), n


def _grad_view(g, like_shape, name):
  if g.dim() != 4 or tuple(g.shape) != tuple(like_shape) or g.dtype != torch.bfloat16:
    raise ValueError(f"{name} must be a bf16 logical [B,S,H,D] = {tuple(like_shape)} view, got {tuple(g.shape)} {g.dtype}")
  if g.stride(3) != 1:
    g = g.contiguous()
  return g


def norm_rope_fullrow_backward(q, k, wq, wk, cos, sin, heads: int, gq, gk, eps: float = 1e-6, q_mul: float = 1.0, bias=None,
                               dq=None, dk=None):
  """Backward of `norm_rope_fullrow` (and, with `bias` bf16 [2*H*D], of the q | k blocks of `norm_rope_qkv`).

  q, k: the saved bf16 [B,S,H*D] inputs (k may be None, then gk is None); gq, gk: bf16 logical [B,S,H,D] gradients of
  the prologue's outputs.  Returns (dq, dk, dwq, dwk) -- dq, dk bf16 shaped and strided like q, k (or written into
  the given dq / dk, which may be the column blocks of a fused gradient buffer), dwq, dwk f32 [H*D] -- plus dbias
  f32 [2*H*D] when bias is given."""
  _check_dev(q, k, wq, wk, gq, gk, bias, dq, dk)
  if q.dim() != 3 or q.dtype != torch.bfloat16 or q.stride(2) != 1:
    raise ValueError("q must be bf16 [B, S, H*D] with a contiguous last axis")
  b, s, n = q.shape
  if n % heads:
    raise ValueError(f"inner dim {n} is not divisible by heads={heads}")
  d = n // heads
  has_k = k is not None
  if has_k and (k.shape != q.shape or k.dtype != q.dtype or k.stride() != q.stride()):
    raise ValueError("k must match q in shape, dtype and strides")
  if has_k != (gk is not None):
    raise ValueError("gk must be given exactly when k is")
  _check_weights(n, wq=wq, wk=wk if has_k else None)
  pcos, psin, kind = _table_args(cos, sin, s, d)
  gq = _grad_view(gq, (b, s, heads, d), "gq")
  if has_k:
    gk = _grad_view(gk, (b, s, heads, d), "gk")
    if gk.stride() != gq.stride():
      gk = torch.empty_strided(gq.shape, gq.stride(), dtype=gk.dtype, device=gk.device).copy_(gk)
  if bias is not None and (not has_k or bias.dtype != torch.bfloat16 or bias.numel() != 2 * n or not bias.is_contiguous()):
    raise ValueError("bias must be a contiguous bf16 [2*H*D] tensor (q | k blocks) and needs k")
  if dq is None:
    dq = torch.empty_strided(q.shape, q.stride(), dtype=torch.bfloat16, device=q.device)
  if has_k and dk is None:
    dk = torch.empty_strided(q.shape, q.stride(), dtype=torch.bfloat16, device=q.device)
  for name, t in (("dq", dq), ("dk", dk)):
    if t is not None and (t.shape != q.shape or t.dtype != torch.bfloat16 or t.stride(2) != 1 or (has_k and t.stride() != dq.stride())):
      raise ValueError(f"{name} must be bf16 [B, S, H*D] with a contiguous last axis (dq and dk sharing their strides)")
  dwq = torch.empty(n, dtype=torch.float32, device=q.device)
  dwk = torch.empty(n, dtype=torch.float32, device=q.device) if has_k else None
  dbias = torch.empty(2 * n, dtype=torch.float32, device=q.device) if bias is not None else None
  ws, nws = _bwd_workspace(b * s, (2 if has_k else 1) * (2 if bias is not None else 1) * n, q.device)
  st = _strides(gq)
  rc = _lib.load().mdattn_host_norm_rope_fullrow_bwd(
      _stream(), _ptr(q), _ptr(k), _ptr(bias), _ptr(gq), _ptr(gk), _ptr(dq), _ptr(dk), _ptr(wq), _ptr(wk), _ptr(dwq), _ptr(dwk),
      _ptr(dbias), 0, None, None, pcos, psin, kind, b, s, heads, d, eps, q_mul, q.stride(0), q.stride(1), dq.stride(0), dq.stride(1),
      ctypes.byref(st), _ptr(ws), nws)
  _lib.check(rc, "mdattn_norm_rope_fullrow_bwd")
  return (dq, dk, dwq, dwk) if bias is None else (dq, dk, dwq, dwk, dbias)


def norm_rope_perhead_backward(q, k, wq, wk, cos, sin, gq, gk, eps: float = 1e-6, wq_txt=None, wk_txt=None, n_txt: int = 0,
                               q_mul: float = 1.0):
  """Backward of `norm_rope_perhead`: q, k the saved bf16 logical [B,S,H,D] inputs (k may be None), gq, gk the
  gradients of its outputs.  Returns (dq, dk, dwq, dwk, dwq_txt, dwk_txt): dq, dk bf16 laid out like q; the weight
  gradients f32 [D] (the *_txt ones None when no text weights were given)."""
  _check_dev(q, k, wq, wk, wq_txt, wk_txt, gq, gk)
  if q.dtype != torch.bfloat16:
    raise ValueError("q must be bf16")
  b, s, h, d = q.shape
  has_k = k is not None
  if has_k and (k.shape != q.shape or k.stride() != q.stride() or k.dtype != q.dtype):
    raise ValueError("k must match q in shape, dtype and strides")
  if has_k != (gk is not None):
    raise ValueError("gk must be given exactly when k is")
  _check_weights(d, wq=wq, wk=wk if has_k else None, wq_txt=wq_txt, wk_txt=wk_txt if has_k else None)
  pcos, psin, kind = _table_args(cos, sin, s, d)
  gq = _grad_view(gq, q.shape, "gq")
  if has_k:
    gk = _grad_view(gk, q.shape, "gk")
    if gk.stride() != gq.stride():
      gk = torch.empty_strided(gq.shape, gq.stride(), dtype=gk.dtype, device=gk.device).copy_(gk)
  dq = torch.empty_strided(q.shape, q.stride(), dtype=torch.bfloat16, device=q.device)
  dk = torch.empty_strided(q.shape, q.stride(), dtype=torch.bfloat16, device=q.device) if has_k else None
  f32 = lambda: torch.empty(d, dtype=torch.float32, device=q.device)
  dwq, dwk = f32(), (f32() if has_k else None)
  dwq_t = f32() if wq_txt is not None else None
  dwk_t = f32() if (wk_txt is not None and has_k) else None
  ws, nws = _bwd_workspace(b * s * h, 4 * d, q.device)
  si, sd, sg = _strides(q), _strides(dq), _strides(gq)
  rc = _lib.load().mdattn_host_norm_rope_perhead_bwd(
      _stream(), _ptr(q), _ptr(k), _ptr(gq), _ptr(gk), _ptr(dq), _ptr(dk), _ptr(wq), _ptr(wk), _ptr(wq_txt),
      _ptr(wk_txt if has_k else None), n_txt, _ptr(dwq), _ptr(dwk), _ptr(dwq_t), _ptr(dwk_t), 0, pcos, psin, kind, b, s, h, d, eps, q_mul,
      ctypes.byref(si), ctypes.byref(sd), ctypes.byref(sg), _ptr(ws), nws)
  _lib.check(rc, "mdattn_norm_rope_perhead_bwd")
  return dq, dk, dwq, dwk, dwq_t, dwk_t


def norm_rope_rows_backward(x, w, g, cos=None, sin=None, heads: int = 1, mode: str = "none", eps: float = 1e-6):
  """Backward of `norm_rope_rows`: x the saved [B,S,H*D] input (bf16 or f32), g the bf16 logical [B,S,H,D] gradient of
  its output.  Returns (dx in x's dtype and strides, dw f32 [H*D])."""
  _check_dev(x, w, cos, sin, g)
  if x.dim() != 3 or x.dtype not in (torch.bfloat16, torch.float32) or x.stride(2) != 1:
    raise ValueError("x must be bf16 or f32 [B, S, H*D] with a contiguous last axis")
  b, s, n = x.shape
  if n % heads:
    raise ValueError(f"inner dim {n} is not divisible by heads={heads}")
  d = n // heads
  modes = {"none": 0, "interleaved": 1, "split": 2}
  if mode not in modes:
    raise ValueError(f"mode={mode!r} not supported. Choose between 'none', 'interleaved' and 'split'.")
  if w.dtype != torch.float32 or w.numel() != n or not w.is_contiguous():
    raise ValueError("w must be a contiguous f32 [H*D] tensor")
  if mode != "none":
    want = (b, s, n) if mode == "interleaved" else (b, heads, s, d // 2)
    for name, t in (("cos", cos), ("sin", sin)):
      if t is None or tuple(t.shape) != want or t.dtype != torch.float32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous f32 tensor of shape {want} for mode={mode!r}")
  g = _grad_view(g, (b, s, heads, d), "g")
  dx = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=x.device)
  dw = torch.empty(n, dtype=torch.float32, device=x.device)
  ws, nws = _bwd_workspace(b * s, n, x.device)
  st = _strides(g)
  rc = _lib.load().mdattn_norm_rope_rows_bwd(
      _stream(), _ptr(x), int(x.dtype == torch.float32), _ptr(g), _ptr(dx), _ptr(w), _ptr(dw), _ptr(cos if mode != "none" else None),
      _ptr(sin if mode != "none" else None), modes[mode], b, s, heads, d, eps, x.stride(0), x.stride(1), dx.stride(0), dx.stride(1),
      ctypes.byref(st), _ptr(ws), nws)
  _lib.check(rc, "mdattn_norm_rope_rows_bwd")
  return dx, dw


def key_mask_bias(keep: torch.Tensor, masked_value: float = -math.inf) -> torch.Tensor:
  """[B,Skv] keep-mask (bool / uint8) -> additive key bias f32 [B, Skv rounded up to 32] for `flash_attention`."""
  _check_dev(keep)
  if keep.dim() != 2:
    raise ValueError(f"keep mask must have shape [batch, kv_length], got {tuple(keep.shape)}")
  keep8 = keep.to(torch.uint8).contiguous() if keep.dtype != torch.uint8 else keep.contiguous()
  b, skv = keep8.shape
  stride = (skv + 31) // 32 * 32
  bias = torch.empty((b, stride), dtype=torch.float32, device=keep.device)
  rc = _lib.load().mdattn_key_mask_bias(_stream(), _ptr(keep8), _ptr(bias), b, skv, stride, float(masked_value))
  _lib.check(rc, "mdattn_key_mask_bias")
  return bias


def flash_attention(q, k, v, scale: float | None = None, return_lse: bool = False, out_layout: str = "bshd", out=None,
                    key_bias: torch.Tensor | None = None, *, heads: int | None = None, keep: torch.Tensor | None = None, q_mul: float = 1.0):
  """softmax(scale * q k^T [+ key_bias]) v, non-causal.  q [B,Sq,H,D], k/v [B,Skv,H,D] logical views, bf16.

  `key_bias` f32 [B, >= Skv rounded up to 32] (see `key_mask_bias`) is added to the scaled logits of each key;
  -inf excludes a key.  Returns out (logical [B,Sq,H,D] in `out_layout`) and, if asked, lse f32 [B,H,Sq] (natural log).

  The registry entries' form (`heads` given): q, k, v as the models hand them over, [B,S,H*D] or [B,H,S,D], with a
  [B,Skv] keep-mask and a factor `q_mul` rounded into q; returns [B,Sq,H*D], or None when an operand needs a conversion
  first (another dtype, a head dim to be padded, a mask to be copied).
  """
  if heads is not None:
    return _lib.host().flash(q, k, v, heads, scale, keep, q_mul)
  _check_dev(q, k, v)
  if not (q.dtype == k.dtype == v.dtype == torch.bfloat16):
    raise ValueError("flash_attention needs bf16 q, k, v")
  b, sq, h, d = q.shape
  if k.shape != v.shape or k.shape[0] != b or k.shape[2] != h or k.shape[3] != d:
    raise ValueError(f"inconsistent shapes q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
  skv = k.shape[1]
  if scale is None:
    scale = 1.0 / math.sqrt(d)
  if out is None:
    out = _alloc_like_layout(b, sq, h, d, out_layout, torch.bfloat16, q.device)
  lse = torch.empty((b, h, sq), dtype=torch.float32, device=q.device) if return_lse else None
  sq_, sk_, sv_, so_ = _strides(q), _strides(k), _strides(v), _strides(out)
  if key_bias is None:
    rc = _lib.load().mdattn_fwd_bf16(
        _stream(), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), b, h, sq, skv, d,
        ctypes.byref(sq_), ctypes.byref(sk_), ctypes.byref(sv_), ctypes.byref(so_), float(scale))
    _lib.check(rc, "mdattn_fwd_bf16")
  else:
    _check_dev(key_bias)
    if key_bias.dtype != torch.float32 or key_bias.dim() != 2 or key_bias.shape[0] != b or key_bias.stride(1) != 1:
      raise ValueError("key_bias must be an f32 [batch, padded kv_length] tensor with a contiguous last axis")
    if key_bias.shape[1] != (skv + 31) // 32 * 32:
      # a shorter bias whose padding still covers Skv would silently exclude the trailing keys
      raise ValueError(f"key_bias must have kv_length rounded up to 32 = {(skv + 31) // 32 * 32} columns (padding filled with "
                       f"the masked value), got {key_bias.shape[1]}")
    rc = _lib.load().mdattn_fwd_bf16_bias(
        _stream(), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), b, h, sq, skv, d,
        ctypes.byref(sq_), ctypes.byref(sk_), ctypes.byref(sv_), ctypes.byref(so_), float(scale),
        _ptr(key_bias), key_bias.stride(0))
    _lib.check(rc, "mdattn_fwd_bf16_bias")
  return (out, lse) if return_lse else out


def flash_attention_backward(q, k, v, out, dout, lse, scale: float | None = None, key_bias: torch.Tensor | None = None):
  """Gradients of `flash_attention`: q, out, dout [B,Sq,H,D]; k, v [B,Skv,H,D] logical views, bf16; lse f32 [B,H,Sq] as
  returned by the forward; `key_bias` the additive key bias the forward was given, if any.  Returns (dq, dk, dv) shaped
  and laid out like q, k, v."""
  _check_dev(q, k, v, out, dout, lse)
  if not all(t.dtype == torch.bfloat16 for t in (q, k, v, out, dout)):
    raise ValueError("flash_attention_backward needs bf16 q, k, v, out, dout")
  b, sq, h, d = q.shape
  skv = k.shape[1]
  if out.shape != q.shape or dout.shape != q.shape or k.shape != v.shape or tuple(lse.shape) != (b, h, sq):
    raise ValueError("inconsistent shapes")
  if dout.stride() != out.stride():  # the kernels walk out and dout with one set of strides: re-lay dout like out
    dout = torch.empty_strided(out.shape, out.stride(), dtype=dout.dtype, device=dout.device).copy_(dout)
  if scale is None:
    scale = 1.0 / math.sqrt(d)
  lse = lse.contiguous()
  dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
  if dq.stride() != q.stride() or dk.stride() != k.stride() or dv.stride() != v.stride():
    raise ValueError("q, k, v must be dense tensors (their gradients take the same strides)")
  lib = _lib.load()
  nws = lib.mdattn_bwd_split_workspace_floats(b, h, sq, skv, d) or lib.mdattn_bwd_workspace_floats(b, h, sq)
  ws = torch.empty(nws, dtype=torch.float32, device=q.device)
  sq_, sk_, sv_, so_ = _strides(q), _strides(k), _strides(v), _strides(out)
  args = (_stream(), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(dout), _ptr(lse), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), nws,
          b, h, sq, skv, d, ctypes.byref(sq_), ctypes.byref(sk_), ctypes.byref(sv_), ctypes.byref(so_), float(scale))
  if key_bias is None:
    _lib.check(lib.mdattn_bwd_bf16(*args), "mdattn_bwd_bf16")
  else:
    _check_dev(key_bias)
    if key_bias.dtype != torch.float32 or tuple(key_bias.shape) != (b, (skv + 31) // 32 * 32) or key_bias.stride(1) != 1:
      raise ValueError("key_bias must be the f32 [batch, kv_length rounded up to 32] tensor the forward was given")
    _lib.check(lib.mdattn_bwd_bf16_bias(*args, _ptr(key_bias), key_bias.stride(0)), "mdattn_bwd_bf16_bias")
  return dq, dk, dv


def flash_attention_backward_static(q, k, v, out, dout, lse, dq, dk, dv, scale: float | None = None):
  """`flash_attention_backward` into caller-provided dq, dk, dv (strides of q, k, v) through the entry point that
  allocates nothing: its scratch (lse / delta and, where they fit, the partial gradients of a split pass) is a static
  device array of the library (32 MiB per GPU), so the call can sit in code that must not allocate (HIP graph capture).  Raises MdattnError (code E_TOOBIG) when B*H*ceil32(Sq)
  exceeds 4,194,304 rows.  Calls that overlap on one GPU share the scratch and race."""
  _check_dev(q, k, v, out, dout, lse, dq, dk, dv)
  if not all(t.dtype == torch.bfloat16 for t in (q, k, v, out, dout, dq, dk, dv)):
    raise ValueError("flash_attention_backward_static needs bf16 tensors")
  b, sq, h, d = q.shape
  if out.shape != q.shape or dout.shape != q.shape or k.shape != v.shape or tuple(lse.shape) != (b, h, sq) or not lse.is_contiguous():
    raise ValueError("inconsistent shapes")
  if dout.stride() != out.stride() or dq.stride() != q.stride() or dk.stride() != k.stride() or dv.stride() != v.stride():
    raise ValueError("dout must share out's strides and dq, dk, dv those of q, k, v")
  if dq.shape != q.shape or dk.shape != k.shape or dv.shape != v.shape:
    raise ValueError("dq, dk, dv must be shaped like q, k, v")
  if scale is None:
    scale = 1.0 / math.sqrt(d)
  sq_, sk_, sv_, so_ = _strides(q), _strides(k), _strides(v), _strides(out)
  rc = _lib.load().mdattn_bwd_bf16_static(
      _stream(), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(dout), _ptr(lse), _ptr(dq), _ptr(dk), _ptr(dv),
      b, h, sq, k.shape[1], d, ctypes.byref(sq_), ctypes.byref(sk_), ctypes.byref(sv_), ctypes.byref(so_), float(scale))
  _lib.check(rc, "mdattn_bwd_bf16_static")
  return dq, dk, dv


def quant_e4m3(x: torch.Tensor, premul: float = 1.0, pow2_scale: bool = False):
  """Per-tensor absmax quantisation of a contiguous bf16 tensor -> (uint8 e4m3 bytes, f32[2] scale buffer).

  `premul` is multiplied into x before the single rounding (x * premul ~= x8 * scale[0]); `pow2_scale` rounds the
  scale up to a power of two.  q with premul=folded_q_mul(D) and pow2_scale=True, k with pow2_scale=True and
  flash_attention_fp8(..., scale=FOLDED_SCALE) let the fp8 kernel apply the whole logit scale inside its MFMAs."""
  _check_dev(x)
  if x.dtype != torch.bfloat16 or not x.is_contiguous():
    raise ValueError("quant_e4m3 needs a contiguous bf16 tensor")
  x8 = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
  scale = torch.empty(2, dtype=torch.float32, device=x.device)
  rc = _lib.load().mdattn_quant_e4m3(_stream(), _ptr(x), _ptr(x8), _ptr(scale), x.numel(), float(premul), int(bool(pow2_scale)))
  _lib.check(rc, "mdattn_quant_e4m3")
  return x8, scale


FP8_SOFTMAX_MODES = {"exp2": 0, "byte_grid": 1}


def flash_attention_fp8(q8, k8, v8, q_scale, k_scale, v_scale, scale: float | None = None, return_lse: bool = False,
                        out_layout: str = "bshd", softmax: str = "exp2", key_bias: torch.Tensor | None = None):
  """fp8-e4m3 variant: q8/k8/v8 uint8 logical [B,S,H,D] views, *_scale device f32 tensors (element 0 is used).

  softmax="exp2": exact exponentials; the lse is the logsumexp of the quantised logits and the pair (out, lse) can be
  merged like a bf16 partial.  softmax="byte_grid": with power-of-two q and k scales and the softmax scale carried by
  q (see `quant_e4m3`) P is a piecewise-linear exponential read off the e4m3 byte grid (12 % faster; out keeps its
  accuracy, the lse is only good to about 0.08); with any other scales it is the same as "exp2".
  `key_bias` (see `key_mask_bias`): additive per-key bias, -inf excludes a key; always the exact-exponential softmax."""
  if softmax not in FP8_SOFTMAX_MODES:
    raise ValueError(f"softmax={softmax!r} not supported. Choose between 'exp2' and 'byte_grid'.")
  _check_dev(q8, k8, v8, q_scale, k_scale, v_scale)
  b, sq, h, d = q8.shape
  skv = k8.shape[1]
  if scale is None:
    scale = 1.0 / math.sqrt(d)
  out = _alloc_like_layout(b, sq, h, d, out_layout, torch.bfloat16, q8.device)
  lse = torch.empty((b, h, sq), dtype=torch.float32, device=q8.device) if return_lse else None
  sq_, sk_, sv_, so_ = _strides(q8), _strides(k8), _strides(v8), _strides(out)
  args = (_stream(), _ptr(q8), _ptr(k8), _ptr(v8), _ptr(out), _ptr(lse), b, h, sq, skv, d,
          ctypes.byref(sq_), ctypes.byref(sk_), ctypes.byref(sv_), ctypes.byref(so_), float(scale),
          _ptr(q_scale), _ptr(k_scale), _ptr(v_scale))
  if key_bias is None:
    _lib.check(_lib.load().mdattn_fwd_fp8(*args, FP8_SOFTMAX_MODES[softmax]), "mdattn_fwd_fp8")
  else:
    _check_dev(key_bias)
    if key_bias.dtype != torch.float32 or tuple(key_bias.shape) != (b, (skv + 31) // 32 * 32) or key_bias.stride(1) != 1:
      raise ValueError(f"key_bias must be an f32 [batch, kv_length rounded up to 32] = [{b}, {(skv + 31) // 32 * 32}] tensor")
    _lib.check(_lib.load().mdattn_fwd_fp8_bias(*args, _ptr(key_bias), key_bias.stride(0)), "mdattn_fwd_fp8_bias")
  return (out, lse) if return_lse else out


def new_merge_state(b, s, h, d, device, layout: str = "bshd"):
  """(o_run f32 zeros as a logical [B,S,H,D] view, lse_run f32 [B,H,S] filled with -1e30)."""
  o = _alloc_like_layout(b, s, h, d, layout, torch.float32, device)
  o.zero_()
  lse = torch.full((b, h, s), LSE_INIT, dtype=torch.float32, device=device)
  return o, lse


def merge_partial(o_run, lse_run, o_cur, lse_cur):
  """In-place LSE-space merge of (o_cur, lse_cur) into (o_run, lse_run)."""
  _check_dev(o_run, lse_run, o_cur, lse_cur)
  b, s, h, d = o_run.shape
  if o_run.dtype != torch.float32 or o_cur.shape != o_run.shape or o_cur.dtype not in (torch.bfloat16, torch.float32):
    raise ValueError("o_run must be f32 and o_cur bf16/f32 of the same logical shape")
  for t in (lse_run, lse_cur):
    if t.dtype != torch.float32 or tuple(t.shape) != (b, h, s) or not t.is_contiguous():
      raise ValueError("lse tensors must be contiguous f32 [B,H,S]")
  sr, sc = _strides(o_run), _strides(o_cur)
  rc = _lib.load().mdattn_merge(
      _stream(), _ptr(o_run), _ptr(lse_run), _ptr(o_cur), _ptr(lse_cur), int(o_cur.dtype == torch.float32),
      b, h, s, d, ctypes.byref(sr), ctypes.byref(sc))
  _lib.check(rc, "mdattn_merge")
  return o_run, lse_run


def flash_attention_merge(q, k, v, o_run, lse_run, scale: float | None = None):
  """One ring step in one launch: attention of q [B,Sq,H,D] against the chunk k/v [B,Skv,H,D] (bf16 logical views),
  merged in place into (o_run f32 logical [B,Sq,H,D], lse_run f32 [B,H,Sq]) as `merge_partial` would merge the
  result of `flash_attention`; the chunk's own output is never stored."""
  if q.is_cuda and _lib.host().flash_merge(q, k, v, o_run, lse_run, 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale):
    return o_run, lse_run
  _check_dev(q, k, v, o_run, lse_run)
  if not (q.dtype == k.dtype == v.dtype == torch.bfloat16):
    raise ValueError("flash_attention_merge needs bf16 q, k, v")
  b, sq, h, d = q.shape
  if k.shape != v.shape or k.shape[0] != b or k.shape[2] != h or k.shape[3] != d:
    raise ValueError(f"inconsistent shapes q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
  if o_run.dtype != torch.float32 or tuple(o_run.shape) != (b, sq, h, d):
    raise ValueError("o_run must be an f32 logical [B,Sq,H,D] view")
  if lse_run.dtype != torch.float32 or tuple(lse_run.shape) != (b, h, sq) or not lse_run.is_contiguous():
    raise ValueError("lse_run must be contiguous f32 [B,H,Sq]")
  if scale is None:
    scale = 1.0 / math.sqrt(d)
  sq_, sk_, sv_, sr_ = _strides(q), _strides(k), _strides(v), _strides(o_run)
  rc = _lib.load().mdattn_fwd_bf16_merge(
      _stream(), _ptr(q), _ptr(k), _ptr(v), _ptr(o_run), _ptr(lse_run), b, h, sq, k.shape[1], d,
      ctypes.byref(sq_), ctypes.byref(sk_), ctypes.byref(sv_), ctypes.byref(sr_), float(scale))
  _lib.check(rc, "mdattn_fwd_bf16_merge")
  return o_run, lse_run


def finalize(o_run: torch.Tensor) -> torch.Tensor:
  """f32 -> bf16 cast of a merged accumulator, same memory layout."""
  _check_dev(o_run)
  if o_run.dtype != torch.float32:
    raise ValueError("finalize needs an f32 tensor")
  out = torch.empty_like(o_run, dtype=torch.bfloat16)  # preserves strides of dense permuted views
  if out.stride() != o_run.stride():
    raise ValueError("finalize needs a dense tensor")
  rc = _lib.load().mdattn_finalize(_stream(), _ptr(o_run), _ptr(out), o_run.numel())
  _lib.check(rc, "mdattn_finalize")
  return out


# ------------------------------------------------------------------------------------------------ attention over packed sequences
def _packed_rows(t: torch.Tensor, group: int = 0) -> torch.Tensor:
  """t [rows, heads, D] as the kernels walk it (whole 16-byte pieces; strides below 2^23 between rows), copied if it is not.  group: heads of q
  or out whose strides the backward entry limits in sum."""
  row, head = _packed_strides(t)
  ok = (t.stride(2) == 1 or t.shape[2] == 1) and row % 8 == 0 and head % 8 == 0 and row < 1 << 23 and group * head < 1 << 29 and t.data_ptr() % 16 == 0
  return t if ok else t.clone(memory_format=torch.contiguous_format)


def _packed_strides(t):
  """Strides of rows and heads (an axis of one element may have any: 0)."""
  return (t.stride(0) if t.shape[0] > 1 else 0), (t.stride(1) if t.shape[1] > 1 else 0)


def _row_strides(t) -> Strides:
  return Strides(0, *_packed_strides(t))


def _packed(q, k, v, q_offsets, k_offsets, k_lengths, causal, max_q, max_k) -> _lib.Packed:
  """The checked mdattn_packed of a call."""
  _check_dev(q, k, v, q_offsets, k_offsets, k_lengths)
  for name, t in (("q", q), ("k", k), ("v", v)):
    if t.dim() != 3 or t.dtype != torch.bfloat16:
      raise ValueError(f"{name} must be a bf16 tensor of shape [rows, heads, head_dim], got {tuple(t.shape)} {t.dtype}")
  if k.shape != v.shape or q.shape[2] != k.shape[2] or k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
    raise ValueError(f"k and v must have one shape, q their head dim and a multiple of their heads, got q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
  if not 0 < q.shape[2] <= 128 or q.shape[2] % 8:
    raise ValueError(f"head_dim={q.shape[2]} not supported: a multiple of 8 up to 128.")
  n = q_offsets.numel() - 1
  for name, t, size in (("q_offsets", q_offsets, n + 1), ("k_offsets", k_offsets, n + 1), ("k_lengths", k_lengths, n)):
    if t is not None and (t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != size or n < 0 or not t.is_contiguous()):
      raise ValueError(f"{name} must be a contiguous int32 tensor of {size} elements, got {tuple(t.shape)} {t.dtype}")
  hint = lambda x: min(max(int(x or 0), 0), 2**31 - 1)
  p = lambda t: None if t is None else t.data_ptr()
  return _lib.Packed(p(q_offsets), p(k_offsets), p(k_lengths), n, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2], int(bool(causal)),
                     hint(max_q), hint(max_k))


def flash_attention_packed(q, k, v, q_offsets, k_offsets=None, *, k_lengths=None, causal: bool = True, scale: float | None = None,
                           max_q: int | None = None, max_k: int | None = None, return_lse: bool = False, return_rest: bool = False):
  """softmax(scale * q k^T) v over sequences that lie one behind the other.  q [Tq, H, D], k, v [Tk, Hkv, D], bf16, any strides of rows and heads;
  H a multiple of Hkv (head h of q meets head h // (H // Hkv)), D a multiple of 8 up to 128.

  q_offsets, k_offsets: int32 [B + 1] on the device, not decreasing: sequence i is the rows q_offsets[i] .. q_offsets[i + 1] of q and those of
  k_offsets (None: the same) of k and v.  k_lengths int32 [B]: only the first k_lengths[i] of them are keys (a cache with room).  causal: of a
  sequence with m queries and n keys, query i sees the keys up to i + n - m.  max_q, max_k: the longest sequence's queries and keys, if the
  caller knows them; they choose how the work is cut and no result depends on them but for its roundings.  Without them a call is planned for one
  sequence of all rows: 16 single tokens against caches of up to 4,096 keys, whose keys are cut only by the hints, take 49 us for 15.

  Returns out [Tq, H, D] and, if asked, lse f32 [H, Tq] (natural log) and what the rounding of out left (bf16, for the backward pass; rows of no
  sequence undefined).  Rows that see no key and rows of no sequence: 0 and -inf."""
  k_offsets = q_offsets if k_offsets is None else k_offsets
  p = _packed(q, k, v, q_offsets, k_offsets, k_lengths, causal, max_q, max_k)
  q, k, v = (_packed_rows(t) for t in (q, k, v))
  out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
  lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device) if return_lse else None
  rest = torch.empty_like(out) if return_rest else None
  lib = _lib.load()
  nws = lib.mdattn_fwd_bf16_packed_workspace_floats(ctypes.byref(p))
  ws = torch.empty(nws, dtype=torch.float32, device=q.device) if nws else None
  st = [ctypes.byref(_row_strides(t)) for t in (q, k, v, out)]
  rc = lib.mdattn_fwd_bf16_packed(_stream(), ctypes.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(rest), _ptr(lse), *st,
                                  float(q.shape[2]**-0.5 if scale is None else scale), _ptr(ws), nws)
  _lib.check(rc, "mdattn_fwd_bf16_packed")
  results = (out, *(t for t in (lse, rest) if t is not None))
  return results if len(results) > 1 else out


def flash_attention_packed_backward(q, k, v, out, dout, lse, q_offsets, k_offsets=None, *, rest=None, causal: bool = True, scale: float | None = None,
                                    max_q: int | None = None, max_k: int | None = None):
  """Backward of `flash_attention_packed`: its inputs, its out, lse and rest (None: gradients are further off where a key has most of a row's
  weight), and the gradient of out (bf16).  Returns (dq, dk, dv), bf16, dense; rows of no sequence get zeros."""
  k_offsets = q_offsets if k_offsets is None else k_offsets
  p = _packed(q, k, v, q_offsets, k_offsets, None, causal, max_q, max_k)
  _check_dev(q, out, dout, lse, rest)
  for name, t in (("out", out), ("dout", dout), *((("rest", rest),) if rest is not None else ())):
    if t.shape != q.shape or t.dtype != torch.bfloat16:
      raise ValueError(f"{name} must be bf16 and shaped like q, {tuple(q.shape)}, got {tuple(t.shape)} {t.dtype}")
  if lse.dtype != torch.float32 or tuple(lse.shape) != (q.shape[1], q.shape[0]) or not lse.is_contiguous():
    raise ValueError(f"lse must be a contiguous f32 tensor of shape {(q.shape[1], q.shape[0])}, got {tuple(lse.shape)} {lse.dtype}")
  group = q.shape[1] // k.shape[1]
  q, k, v = _packed_rows(q, group), _packed_rows(k), _packed_rows(v)
  out, dout = _packed_rows(out, group), _packed_rows(dout, group)
  rest = rest if rest is None else _packed_rows(rest, group)
  if any(t is not None and _packed_strides(t) != _packed_strides(out) for t in (dout, rest)):
    out, dout, rest = (t if t is None else t.contiguous() for t in (out, dout, rest))
  dq, dk, dv = (torch.empty(t.shape, dtype=torch.bfloat16, device=q.device) for t in (q, k, v))
  lib = _lib.load()
  nws = lib.mdattn_bwd_bf16_packed_workspace_floats(ctypes.byref(p))
  ws = torch.empty(max(nws, 4), dtype=torch.float32, device=q.device)
  st = [ctypes.byref(_row_strides(t)) for t in (q, k, v, out, dq, dk, dv)]
  rc = lib.mdattn_bwd_bf16_packed(_stream(), ctypes.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(rest), _ptr(dout), _ptr(lse), _ptr(dq), _ptr(dk),
                                  _ptr(dv), *st, float(q.shape[2]**-0.5 if scale is None else scale), _ptr(ws), nws)
  _lib.check(rc, "mdattn_bwd_bf16_packed")
  return dq, dk, dv


# ------------------------------------------------------------------------------------------------ the layers beside attention
def _float_kind(t, name):
  """1 for f32, 0 for bf16."""
  if t.dtype not in (torch.bfloat16, torch.float32):
    raise ValueError(f"{name} must be bf16 or f32, got {t.dtype}")
  return int(t.dtype == torch.float32)


def _norm_rows(x, name="x"):
  """(groups, rows of a group, C, stride of a group, stride of a row) of x [..., C]: the first axis and the ones between."""
  if x.dim() < 2 or (x.stride(-1) != 1 and x.shape[-1] > 1):
    raise ValueError(f"{name} must have shape [..., C] with a contiguous last axis, got {tuple(x.shape)} strides {x.stride()}")
  if x.dim() == 2:
    return 1, x.shape[0], x.shape[1], 0, x.stride(0)
  step = row_stride(x)
  if step is None:
    raise ValueError(f"the axes of {name} between the first and the last must be dense, got {tuple(x.shape)} strides {x.stride()}")
  return x.shape[0], math.prod(x.shape[1:-1]), x.shape[-1], x.stride(0), step


def row_stride(x):
  """The stride that all axes of x between the first and the last have together, None if there is none.  (An axis of one element may
  have any.)"""
  step = following = None
  for i in range(x.dim() - 2, 0, -1):
    if x.shape[i] == 1:
      continue
    if step is None:
      step = x.stride(i)
    elif x.stride(i) != following:
      return None
    following = x.stride(i) * x.shape[i]
  return x.shape[-1] if step is None else step


def _norm_vectors(weight, bias, groups, c):
  """(elements between the groups' vectors, is f32) of weight and bias, each [C], [B, C], [B, 1, C] or None."""
  stride, f32 = None, 0
  for name, t in (("weight", weight), ("bias", bias)):
    if t is None:
      continue
    shape = tuple(t.shape)
    if t.dim() == 3 and shape[1] == 1:
      shape = (shape[0], shape[2])
    if shape not in ((c,), (groups, c)) or not t.is_contiguous():
      raise ValueError(f"{name} must be a contiguous tensor of shape [{c}], [{groups}, {c}] or [{groups}, 1, {c}], got {tuple(t.shape)} strides {t.stride()}")
    mine = c if len(shape) == 2 else 0
    if stride is None:
      stride, f32 = mine, _float_kind(t, name)
    elif stride != mine or f32 != _float_kind(t, name):
      raise ValueError("weight and bias must agree in dtype, and in whether they are per batch element")
  return stride or 0, f32


def layer_norm(x, weight=None, bias=None, eps: float = 1e-6, weight_offset: float = 0.0, out_dtype=None):
  """h * (weight_offset + weight) + bias with h = (x - mean) / sqrt(var + eps) over the last axis of x [..., C], bf16 or f32.

  weight, bias: bf16 or f32, [C], or, for an x of three axes or more, one per element of its first axis, [B, C] or [B, 1, C] (adaLN's
  scale and shift, with weight_offset 1); None: h (+ bias), whatever weight_offset is, and h * (weight_offset + weight).  Statistics and arithmetic in f32, rounded once to out_dtype (x's)."""
  _check_dev(x, weight, bias)
  x_f32 = _float_kind(x, "x")
  groups, rows, c, sg, sr = _norm_rows(x)
  stride, wb_f32 = _norm_vectors(weight, bias, groups, c)
  out = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
  y_f32 = _float_kind(out, "out_dtype")
  if out.numel():
    rc = _lib.load().mdattn_layer_norm(_stream(), _ptr(x), x_f32, _ptr(out), y_f32, _ptr(weight), _ptr(bias), wb_f32, groups, rows, c, sg, sr,
                                       rows * c, c, stride, float(eps), float(weight_offset))
    _lib.check(rc, "mdattn_layer_norm")
  return out


def layer_norm_quant(x, weight=None, bias=None, eps: float = 1e-6, weight_offset: float = 0.0):
  """`layer_norm` with its unrounded rows quantised (`quant_block_e4m3`, blocks of 1 x 128) instead of stored: a BlockQuant of
  as many rows as x [..., C] has."""
  _check_dev(x, weight, bias)
  x_f32 = _float_kind(x, "x")
  groups, rows, c, sg, sr = _norm_rows(x)
  stride, wb_f32 = _norm_vectors(weight, bias, groups, c)
  out = _new_quant(groups * rows, c, 1, x.device)
  if x.numel():
    rc = _lib.load().mdattn_layer_norm_e4m3(_stream(), _ptr(x), x_f32, _ptr(out.values), _ptr(out.scales), _ptr(weight), _ptr(bias), wb_f32, groups,
                                            rows, c, sg, sr, stride, float(eps), float(weight_offset))
    _lib.check(rc, "mdattn_layer_norm_e4m3")
  return out


def layer_norm_backward(x, weight, bias, g, eps: float = 1e-6, weight_offset: float = 0.0, needs_vectors: bool = True):
  """Backward of `layer_norm`: x, weight, bias as the forward had them (of bias only whether there is one, its shape and dtype),
  g the gradient of its output, in x's dtype.  Returns (dx, dweight, dbias) in their tensors' shapes and dtypes, None for what
  there is not, or for the last two with needs_vectors False."""
  _check_dev(x, weight, bias, g)
  x_f32 = _float_kind(x, "x")
  groups, rows, c, sg, sr = _norm_rows(x)
  stride, wb_f32 = _norm_vectors(weight, bias, groups, c)
  if g.shape != x.shape or g.dtype != x.dtype:
    raise ValueError(f"g must be shaped and typed like x, {tuple(x.shape)} {x.dtype}, got {tuple(g.shape)} {g.dtype}")
  _, _, _, gg, gr = _norm_rows(g, "g")
  dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
  dw = torch.empty_like(weight) if weight is not None and needs_vectors else None
  db = torch.empty_like(bias) if bias is not None and needs_vectors else None
  if not x.numel():
    return dx, *(None if t is None else t.zero_() for t in (dw, db))
  lib = _lib.load()
  nws = lib.mdattn_layer_norm_bwd_workspace_floats(groups, rows, c) if dw is not None or db is not None else 0
  ws = torch.empty(nws, dtype=torch.float32, device=x.device) if nws else None
  rc = lib.mdattn_layer_norm_bwd(_stream(), _ptr(x), x_f32, _ptr(g), _ptr(dx), _ptr(weight), _ptr(dw), _ptr(db), wb_f32, groups, rows, c, sg, sr,
                                 gg, gr, rows * c, c, stride, float(eps), float(weight_offset), _ptr(ws), nws)
  _lib.check(rc, "mdattn_layer_norm_bwd")
  return dx, dw, db


def _residual(x, residual):
  """(is f32, stride of a group, stride of a row) of a residual beside x."""
  if residual is None:
    return 0, 0, 0
  r_f32 = _float_kind(residual, "residual")
  if residual.shape != x.shape or residual.device != x.device or r_f32 < (x.dtype == torch.float32):
    raise ValueError(f"residual must be shaped like x, {tuple(x.shape)}, and of its dtype, or f32 beside a bf16 x, got {tuple(residual.shape)} "
                     f"{residual.dtype} for {x.dtype}")
  return r_f32, *_norm_rows(residual, "residual")[3:]


def rms_norm(x, weight=None, bias=None, residual=None, eps: float = 1e-6, weight_offset: float = 0.0):
  """s = x + residual, y = s * (mean of s^2 over the last axis + eps)^-1/2 * (weight_offset + weight) + bias, for x [..., C], bf16 or f32.

  residual: of x's dtype, or f32 beside a bf16 x; None: s = x.  weight and bias as `layer_norm`'s.  Arithmetic in f32, the norm that of the unrounded
  sum.  Returns (y in x's dtype, s in the residual's), or y alone without a residual."""
  _check_dev(x, weight, bias, residual)
  x_f32 = _float_kind(x, "x")
  groups, rows, c, sg, sr = _norm_rows(x)
  r_f32, rg, rr = _residual(x, residual)
  stride, wb_f32 = _norm_vectors(weight, bias, groups, c)
  y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
  s = None if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device)
  if x.numel():
    rc = _lib.load().mdattn_rms_norm(_stream(), _ptr(x), x_f32, _ptr(residual), r_f32, _ptr(y), _ptr(s), _ptr(weight), _ptr(bias), wb_f32, groups, rows, c,
                                     sg, sr, rg, rr, rows * c, c, rows * c, c, stride, float(eps), float(weight_offset))
    _lib.check(rc, "mdattn_rms_norm")
  return y if residual is None else (y, s)


def rms_norm_quant(x, weight=None, bias=None, residual=None, eps: float = 1e-6, weight_offset: float = 0.0):
  """`rms_norm` with y's unrounded rows quantised (`quant_block_e4m3`, blocks of 1 x 128) instead of stored: (BlockQuant of as many rows as x
  has, s), or the BlockQuant alone without a residual."""
  _check_dev(x, weight, bias, residual)
  x_f32 = _float_kind(x, "x")
  groups, rows, c, sg, sr = _norm_rows(x)
  r_f32, rg, rr = _residual(x, residual)
  stride, wb_f32 = _norm_vectors(weight, bias, groups, c)
  q = _new_quant(groups * rows, c, 1, x.device)
  s = None if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device)
  if x.numel():
    rc = _lib.load().mdattn_rms_norm_e4m3(_stream(), _ptr(x), x_f32, _ptr(residual), r_f32, _ptr(q.values), _ptr(q.scales), _ptr(s), _ptr(weight), _ptr(bias),
                                          wb_f32, groups, rows, c, sg, sr, rg, rr, rows * c, c, stride, float(eps), float(weight_offset))
    _lib.check(rc, "mdattn_rms_norm_e4m3")
  return q if residual is None else (q, s)


def rms_norm_backward(s, weight, bias, g, gs=None, eps: float = 1e-6, weight_offset: float = 0.0, needs_vectors: bool = True, narrow: bool = False,
                      residual=None):
  """Backward of `rms_norm`: s as the forward returned it (x, where there was no residual; or x beside the forward's `residual`, both bf16, for
  gradients without s's rounding), weight and bias as it had them (of bias only
  whether there is one, its shape and dtype), g and gs the gradients of y and s (gs None: none), g in s's dtype or bf16 beside an f32 s.  Returns (ds, dx,
  dweight, dbias): the gradient of the residual, and of x, in s's dtype; the same in bf16 where `narrow` (x was bf16 beside an f32
  residual), else None; None for what there is not, or for the last two with needs_vectors False."""
  _check_dev(s, weight, bias, g, gs, residual)
  s_f32, g_f32 = _float_kind(s, "s"), _float_kind(g, "g")
  groups, rows, c, sg, sr = _norm_rows(s)
  stride, wb_f32 = _norm_vectors(weight, bias, groups, c)
  if g.shape != s.shape or g_f32 > s_f32 or (narrow and (g_f32 or not s_f32)):
    raise ValueError(f"g must be shaped like s, {tuple(s.shape)}, and of its dtype, or bf16 beside an f32 s (and there alone `narrow`), got {tuple(g.shape)} "
                     f"{g.dtype} for {s.dtype}")
  if gs is not None and (gs.shape != s.shape or gs.dtype != s.dtype):
    raise ValueError(f"gs must be shaped and typed like s, {tuple(s.shape)} {s.dtype}, got {tuple(gs.shape)} {gs.dtype}")
  if residual is not None and (s_f32 or residual.shape != s.shape or residual.dtype != s.dtype):
    raise ValueError(f"residual must be bf16 and shaped like s, which has to be bf16 beside it, got {tuple(residual.shape)} {residual.dtype} for "
                     f"{tuple(s.shape)} {s.dtype}")
  rg, rr = (0, 0) if residual is None else _norm_rows(residual, "residual")[3:]
  gg, gr = _norm_rows(g, "g")[3:]
  ug, ur = (0, 0) if gs is None else _norm_rows(gs, "gs")[3:]
  ds = torch.empty(s.shape, dtype=s.dtype, device=s.device)
  dx = torch.empty(s.shape, dtype=torch.bfloat16, device=s.device) if narrow else None
  dw = torch.empty_like(weight) if weight is not None and needs_vectors else None
  db = torch.empty_like(bias) if bias is not None and needs_vectors else None
  if not s.numel():
    return ds, dx, *(None if t is None else t.zero_() for t in (dw, db))
  lib = _lib.load()
  nws = lib.mdattn_rms_norm_bwd_workspace_floats(groups, rows, c) if dw is not None or db is not None else 0
  ws = torch.empty(nws, dtype=torch.float32, device=s.device) if nws else None
  rc = lib.mdattn_rms_norm_bwd(_stream(), _ptr(s), s_f32, _ptr(residual), _ptr(g), g_f32, _ptr(gs), _ptr(ds), _ptr(dx), _ptr(weight), _ptr(dw), _ptr(db), wb_f32,
                               groups, rows, c, sg, sr, rg, rr, gg, gr, ug, ur, stride, float(eps), float(weight_offset), _ptr(ws), nws)
  _lib.check(rc, "mdattn_rms_norm_bwd")
  return ds, dx, dw, db


class BlockQuant:
  """A matrix [rows, cols] held as e4m3 with one power-of-two scale per block of block_rows x 128.

  values: uint8 [rows, cols rounded up to 128], the padding zero (NaN in a block that is not finite).  scales: uint8 [ceil(rows / block_rows), blocks of a row
  rounded up to 4], the exponents with a bias of 127 (0xFF: a block that is not finite).  Both dense."""
  __slots__ = ("values", "scales", "rows", "cols", "block_rows")

  def __init__(self, values, scales, rows: int, cols: int, block_rows: int):
    want = ((rows, -(-cols // 128) * 128), (-(-rows // block_rows), -(-cols // 512) * 4)) if block_rows in (1, 128) else None
    if want is None or (tuple(values.shape), tuple(scales.shape)) != want or values.dtype != torch.uint8 or scales.dtype != torch.uint8 or \
        not values.is_contiguous() or not scales.is_contiguous():
      raise ValueError(f"a BlockQuant of {rows} x {cols} in blocks of {block_rows} x 128 (1 or 128) has dense uint8 values and scales of shapes "
                       f"{want}, got {tuple(values.shape)} {values.dtype} and {tuple(scales.shape)} {scales.dtype}")
    self.values, self.scales, self.rows, self.cols, self.block_rows = values, scales, rows, cols, block_rows

  def dequantize(self, dtype=torch.float32):
    """The numbers that it stands for, [rows, cols] (plain torch, for inspection)."""
    wide = torch.promote_types(dtype, torch.float32)  # (256 * 2^120, which f32's largest numbers round to, is no f32)
    v = self.values.view(torch.float8_e4m3fn).to(wide)
    s = torch.exp2(self.scales.to(wide) - 127).masked_fill_(self.scales == 255, math.nan)
    s = s.repeat_interleave(self.block_rows, 0)[:self.rows].repeat_interleave(128, 1)[:, :v.shape[1]]
    return (v * s)[:, :self.cols].to(dtype)


def _new_quant(rows, cols, block_rows, device):
  u8 = dict(dtype=torch.uint8, device=device)
  return BlockQuant(torch.empty((rows, -(-cols // 128) * 128), **u8), torch.empty((-(-rows // block_rows), -(-cols // 512) * 4), **u8), rows, cols,
                    block_rows)


def quant_block_e4m3(x, block_rows: int = 1, plain: bool = True, transposed: bool = False, sums: bool = False):
  """x [R, C] (bf16 or f32, C contiguous) to e4m3 with one power-of-two scale per block of block_rows x 128 (1 or 128): the smallest
  power of two, 2^-127 at least, with which a block's largest magnitude is at most 448.

  Returns what is asked for, one BlockQuant or a tuple: of x (`plain`), of its transpose [C, R] in blocks of block_rows x 128 of that
  (`transposed`), and f32 [ceil(R / 128), C], the sums of each column over 128 rows each (`sums`; see `sum_rows`)."""
  _check_dev(x)
  if x.dim() != 2 or (x.stride(1) != 1 and x.shape[1] > 1):
    raise ValueError(f"quant_block_e4m3 needs a matrix with contiguous rows, got {tuple(x.shape)} strides {x.stride()}")
  if block_rows not in (1, 128):
    raise ValueError(f"block_rows={block_rows!r} not supported. Choose between 1 and 128.")
  if not plain and not transposed:
    raise ValueError("neither the matrix nor its transpose is asked for")
  x_f32 = _float_kind(x, "x")
  r, c = x.shape
  q = _new_quant(r, c, block_rows, x.device) if plain else None
  qt = _new_quant(c, r, block_rows, x.device) if transposed else None
  part = torch.empty((-(-r // 128), c), dtype=torch.float32, device=x.device) if sums else None
  if x.numel():
    rc = _lib.load().mdattn_quant_block_e4m3(_stream(), _ptr(x), x_f32, r, c, x.stride(0), block_rows, _ptr(q.values if q else None),
                                             _ptr(q.scales if q else None), _ptr(qt.values if qt else None), _ptr(qt.scales if qt else None), _ptr(part))
    _lib.check(rc, "mdattn_quant_block_e4m3")
  out = tuple(t for t in (q, qt, part) if t is not None)
  return out[0] if len(out) == 1 else out


def sum_rows(rows, out_dtype=torch.float32):
  """f32 [n, C] -> [C], summed in a fixed order."""
  _check_dev(rows)
  if rows.dim() != 2 or rows.dtype != torch.float32 or not rows.is_contiguous():
    raise ValueError("sum_rows needs a contiguous f32 matrix")
  out = torch.empty(rows.shape[1], dtype=out_dtype, device=rows.device)
  kind = _float_kind(out, "out_dtype")
  if not rows.numel():
    return out.zero_()
  _lib.check(_lib.load().mdattn_sum_rows(_stream(), _ptr(rows), rows.shape[0], rows.shape[1], _ptr(out), kind), "mdattn_sum_rows")
  return out


def matmul_fp8_block(a: BlockQuant, b: BlockQuant, bias=None):
  """a b^T + bias in bf16: a [M, K] in blocks of 1 x 128, b [N, K] in blocks of 1 x 128 or 128 x 128; bias bf16 or f32 [N] or None.
  Sums in f32 on the matrix cores, whose 8-bit products are added eight at a time with 14 bits below the largest of them; rounded once."""
  return matmul_fp8_block_as(a, b, bias, (a.rows,))


def matmul_fp8_block_as(a, b, bias, rows_shape):
  """`matmul_fp8_block` with the rows in several axes, [*rows_shape, N].  (A view of [M, N] would be one that autograd forbids to change in
  place where it is made without gradients or inside a node.)"""
  _check_dev(a.values, a.scales, b.values, b.scales, bias)
  if a.block_rows != 1:
    raise ValueError("the first operand's blocks must be 1 x 128")
  if a.cols != b.cols:
    raise ValueError(f"inner dims differ: {a.cols} and {b.cols}")
  if bias is not None and (bias.dim() != 1 or bias.shape[0] != b.rows or not bias.is_contiguous()):
    raise ValueError(f"bias must be a contiguous tensor of shape [{b.rows}], got {tuple(bias.shape)}")
  bias_f32 = 0 if bias is None else _float_kind(bias, "bias")
  m, n, k = a.rows, b.rows, a.cols
  out = torch.empty((*rows_shape, n), dtype=torch.bfloat16, device=a.values.device)
  if not out.numel():
    return out
  if not k:
    return out.zero_() if bias is None else out.copy_(bias.expand(out.shape))
  lib = _lib.load()
  nws = lib.mdattn_matmul_fp8_block_workspace_floats(m, n, k)
  ws = torch.empty(nws, dtype=torch.float32, device=out.device) if nws else None
  rc = lib.mdattn_matmul_fp8_block(_stream(), _ptr(a.values), _ptr(a.scales), _ptr(b.values), _ptr(b.scales), b.block_rows, _ptr(bias), bias_f32,
                                   _ptr(out), n, m, n, k, _ptr(ws), nws)
  _lib.check(rc, "mdattn_matmul_fp8_block")
  return out
