"""The layers beside attention without a GPU: requests whose grids the card cannot count, and what the host side says of unusual arguments."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import layer_inputs
from maxdiffusion_amd import _lib, attention_op, layer_op, ops

P = ctypes.c_void_p
FAKE = P(0x1000)  # never dereferenced: every call below must be refused before it launches anything


def test_grids_past_2_32_threads_are_refused_before_a_launch(lib):
  """A launch of 2^32 threads or more is taken by the runtime and runs modulo 2^32."""
  norm = lambda groups, c: lib.mdattn_layer_norm(None, FAKE, 1, FAKE, 1, FAKE, None, 1, groups, 1, c, c, c, c, c, c, 1e-6, 0.0)
  assert norm(2**32 // 64, 1) == norm(2**32 // 1024, 16384) == _lib.E_UNSUPPORTED
  blocks = lambda groups, c: lib.mdattn_layer_norm_e4m3(None, FAKE, 1, FAKE, FAKE, FAKE, None, 1, groups, 1, c, c, c, c, 1e-6, 0.0)
  assert blocks(2**32 // 64, 1) == _lib.E_UNSUPPORTED

  def backward(groups, c, vectors):
    nws = lib.mdattn_layer_norm_bwd_workspace_floats(groups, 1, c)
    d = FAKE if vectors else None
    return lib.mdattn_layer_norm_bwd(None, FAKE, 1, FAKE, FAKE, FAKE, d, d, 1, groups, 1, c, c, c, c, c, c, c, c, 1e-6, 0.0, FAKE, nws)

  assert backward(2**32 // 1024, 64, True) == backward(2**31 // 1024, 65, True) == _lib.E_UNSUPPORTED  # the sums' grid
  assert backward(2**32 // 256, 1, False) == _lib.E_UNSUPPORTED
  assert lib.mdattn_sum_rows(None, FAKE, 1, 2**28, FAKE, 1) == _lib.E_UNSUPPORTED
  quant = lambda r: lib.mdattn_quant_block_e4m3(None, FAKE, 0, r, 1, 1, 1, FAKE, FAKE, None, None, None)
  assert quant(2**31) == _lib.E_UNSUPPORTED


def test_every_launch_asks_whether_its_grid_can_be_counted(lib):
  """An older entry, whose own checks know nothing of it."""
  assert lib.mdattn_host_copy(None, FAKE, FAKE, None, None, ctypes.c_int64(2**24 * 256 * 16)) == _lib.E_UNSUPPORTED


# ------------------------------------------------------------------------------------------------ second derivatives
class Square(torch.autograd.Function):
  """A node as the package's: its gradient comes from code that autograd does not see."""

  @staticmethod
  def forward(ctx, x, y):
    ctx.save_for_backward(x)
    return x * x

  @staticmethod
  @_lib.first_order
  def backward(ctx, g):
    (x,) = ctx.saved_tensors
    return torch.from_numpy((2 * x * g).detach().numpy()), None


def test_second_derivatives_are_refused():
  x = torch.arange(1.0, 4.0, requires_grad=True)
  (dx,) = torch.autograd.grad(Square.apply(x, None).sum(), x)
  assert torch.equal(dx, 2 * x) and not dx.requires_grad
  (dx,) = torch.autograd.grad(Square.apply(x, None).sum(), x, create_graph=True)  # recorded, and as right
  assert torch.equal(dx, 2 * x) and dx.requires_grad
  for penalty in (dx.square().sum(), dx.square().sum() + x.sum()):  # also where x is reached beside it
    with pytest.raises(NotImplementedError, match="second derivatives"):
      torch.autograd.grad(penalty, x, retain_graph=True)
  with pytest.raises(NotImplementedError, match="second derivatives"):
    dx.sum().backward()
  g = torch.ones(3, requires_grad=True)  # along the incoming gradient alone
  (dx,) = torch.autograd.grad(Square.apply(x, None), x, g, create_graph=True)
  with pytest.raises(NotImplementedError, match="second derivatives"):
    torch.autograd.grad(dx.sum(), g)
  y = torch.ones(3, requires_grad=True)  # a gradient that nothing differentiates is left alone
  (dy,) = torch.autograd.grad((Square.apply(x, None) * y).sum(), y, create_graph=True)
  assert torch.equal(torch.autograd.grad(dy.sum(), x)[0], 2 * x)


def test_tangents_are_refused():
  x, w = torch.zeros(2, 100), ops.BlockQuant(torch.zeros((130, 128), dtype=torch.uint8), torch.zeros((2, 4), dtype=torch.uint8), 130, 100, 128)
  context = dict(heads=1, scale=1.0)
  with forward_ad.dual_level():
    d = forward_ad.make_dual(x, torch.ones_like(x))
    q, v = d.view(1, 2, 100), torch.zeros(100)
    for call in (lambda: layer_op.hip_layer_norm(d), lambda: layer_op.hip_layer_norm(x, d[0]), lambda: layer_op.hip_linear_fp8(d, w),
                 lambda: layer_op.hip_linear_fp8(x, d), lambda: layer_op.hip_layer_norm_linear_fp8(d, None, None, w), lambda: layer_op.hip_linear_fp8(x, x, d[:, 0]),
                 lambda: attention_op.hip_flash_kernel(q, q, q, context), lambda: attention_op.hip_flash_fp8_kernel(q, q, q, context),
                 lambda: attention_op.hip_norm_rope(q, q, v, v, None, 1), lambda: attention_op.hip_norm_rope_ltx2(q, q, v, v, 1),
                 lambda: attention_op.hip_norm_rope_qkv(torch.cat((q, q, q), -1), v, v, None, 1)):
      with pytest.raises(NotImplementedError, match="tangents"):
        call()


# ------------------------------------------------------------------------------------------------ arguments
def test_an_empty_inner_axis_is_no_error_of_its_own():
  w = ops.BlockQuant(torch.zeros((4, 0), dtype=torch.uint8), torch.zeros((1, 0), dtype=torch.uint8), 4, 0, 128)
  for weight in (w, torch.zeros(4, 0, dtype=torch.bfloat16)):
    with pytest.raises(ValueError, match="device memory"):
      layer_op.hip_linear_fp8(torch.zeros(2, 3, 0, dtype=torch.bfloat16), weight)


def test_tensors_without_axes_are_refused():
  x, one = torch.zeros(2, 0), torch.zeros(())
  w = ops.BlockQuant(torch.zeros((4, 0), dtype=torch.uint8), torch.zeros((1, 0), dtype=torch.uint8), 4, 0, 128)
  for call in (lambda: layer_op.hip_layer_norm(one), lambda: layer_op.hip_layer_norm(torch.zeros(3)), lambda: layer_op.hip_linear_fp8(one, w),
               lambda: layer_op.hip_linear_fp8(one, x), lambda: layer_op.hip_linear_fp8(x, one), lambda: layer_op.hip_layer_norm_linear_fp8(one, None, None, w),
               lambda: layer_op.quantize_weight(one)):
    with pytest.raises(ValueError):
      call()


def test_tensors_of_another_device_are_refused(monkeypatch):
  class On:
    is_cuda = True

    def __init__(self, device):
      self.get_device = lambda: device

  monkeypatch.setattr(ops, "_current_device", lambda: 1)
  ops._check_dev(On(1), None, On(1))
  for ts in ((On(1), On(0)), (On(0),), (None, On(0), On(0))):
    with pytest.raises(ValueError, match="current device"):
      ops._check_dev(*ts)


def test_dequantized_in_64_bits():
  """f32's largest numbers round up to 2^128, the smallest block's last place is 2^-136."""
  values = torch.zeros((3, 128), dtype=torch.uint8)
  values[0, 0], values[1, 0], values[2, 0] = 0x78, 0x01, 0x7E  # 256, 2^-9, 448
  q = ops.BlockQuant(values, torch.tensor([[247, 0, 0, 0], [0, 0, 0, 0], [127, 0, 0, 0]], dtype=torch.uint8), 3, 1, 1)
  assert q.dequantize(torch.float64)[:, 0].tolist() == [2.0**128, 2.0**-136, 448.0]
  assert q.dequantize()[:, 0].tolist() == [float("inf"), 2.0**-136, 448.0]


# ------------------------------------------------------------------------------------------------ what the tests of the product can see
def test_exact_operands_show_a_wrong_scale_and_a_rounded_sum():
  """Mistakes planted in a plain product of the operands that the GPU tests use."""
  a, b, want = layer_inputs.cancelling(5, 7, 4096, "cpu")
  for kept, steps in ((torch.float32, 0.0), (torch.bfloat16, 0.9), (torch.float16, 0.4)):  # (the share of results that come out wrong, at least)
    s = torch.zeros(5, 7, dtype=kept)
    for i in range(0, 4096, 128):
      s = (s.double() + a[:, i : i + 128].double() @ b[:, i : i + 128].double().t()).to(kept)
    wrong = (s.float() != want).float().mean()
    assert wrong == 0 if kept == torch.float32 else wrong >= steps, kept
  a, b, want = layer_inputs.scaled(300, 300, 900, "cpu")
  assert torch.equal(a @ b.t(), want)
  blocks = lambda t, by: torch.cat([t[:, i : i + 128] * (2.0 if i // 128 == by else 1.0) for i in range(0, 900, 128)], 1)
  assert not torch.equal(blocks(a, 3) @ b.t(), want) and not torch.equal(blocks(a, 7) @ b.t(), want)
  exps = lambda t: torch.frexp(t[:, :896].reshape(300, 7, 128).abs().amax(2))[1]
  for t in (a, b):  # bytes that differ between a row's blocks and between a block's rows
    assert len(exps(t)[0].unique()) > 3 and len(exps(t)[:, 0].unique()) > 2
