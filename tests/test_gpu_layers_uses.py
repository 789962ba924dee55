"""The layers beside attention as programs use them: calls past what a grid can count, outputs that are changed in place, hooks, autograd's
other modes, arguments that the usual path leaves aside.  Tolerances as in the tests of the kernels: bit for bit where nothing is said."""
import importlib.util
import os

import pytest
import torch
from torch.autograd import forward_ad

import layer_inputs
from maxdiffusion_amd import attention_op as A
from maxdiffusion_amd import layer_op as L
from maxdiffusion_amd import ops

from test_gpu_layers import assert_quant, blocks64, close, half_ulp, norm64, plain_block

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def rand(dev, *shape, seed=0, dtype=F32, std=1.0):
  gen = torch.Generator(device=dev).manual_seed(seed)
  return (torch.randn(shape, generator=gen, device=dev) * std).to(dtype)


# ------------------------------------------------------------------------------------------------ grids past 2^32 threads
def test_one_row_against_very_many_columns(dev):
  """More rows of b than workgroups of 16 of them can be launched."""
  n = 134_300_000  # 8,393,750 workgroups of 512 threads: 2^32 is 8,388,608
  values = torch.zeros((n, 128), dtype=torch.uint8, device=dev)
  values[:, 0] = torch.arange(n, device=dev, dtype=torch.int32).remainder_(64).add_(8).to(torch.uint8)
  b = ops.BlockQuant(values, torch.full((n, 4), 127, dtype=torch.uint8, device=dev), n, 1, 1)
  a = ops.quant_block_e4m3(torch.ones((1, 1), dtype=BF16, device=dev))
  got = ops.matmul_fp8_block(a, b)
  assert torch.equal(got[0], values[:, 0].contiguous().view(torch.float8_e4m3fn).to(BF16))


def test_quantising_very_many_blocks(dev):
  """More blocks than the kernel of rows alone can be launched for."""
  n = 1_080_000_000  # 16,875,000 workgroups of 256 threads: 2^32 is 16,777,216
  x = torch.arange(n, dtype=torch.int32, device=dev).remainder_(250).add_(1).to(BF16).view(n, 1)
  q = ops.quant_block_e4m3(x)
  some = ops.quant_block_e4m3(x[:250].contiguous())
  for i in range(0, n, 60_000_000):  # (a whole number of periods)
    assert torch.equal(q.values[i : i + 60_000_000, 0].view(-1, 250), some.values[:, 0].expand(240_000, 250))
    assert torch.equal(q.scales[i : i + 60_000_000, 0].view(-1, 250), some.scales[:, 0].expand(240_000, 250))
  assert not bool(q.values[-1000:, 1:].any())


# ------------------------------------------------------------------------------------------------ outputs that are changed in place
LAYOUTS = {"dense": lambda x: x, "apart": lambda x: torch.cat((x, x), -1)[..., : x.shape[-1]]}  # (the second one goes through the Python node)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("shape", [(5, 256), (2, 5, 256), (2, 1, 5, 256)])
def test_outputs_take_terms_in_place(dev, layout, shape):
  """A residual added in place, to a layer in training and, as a term that wants a gradient, to a frozen one."""
  x = LAYOUTS[layout](rand(dev, *shape, seed=1, dtype=BF16))
  w, v, g = rand(dev, 130, 256, seed=2, dtype=BF16), rand(dev, 256, seed=3), rand(dev, *shape[:-1], 130, seed=4, dtype=BF16)
  w8 = L.quantize_weight(w)
  term = rand(dev, *shape[:-1], 130, seed=5, dtype=BF16).requires_grad_(True)
  for frozen in (lambda: L.hip_linear_fp8(x, w8), lambda: L.hip_layer_norm_linear_fp8(x, v, None, w8)):
    y, want = frozen(), frozen() + term
    assert not y._is_view()
    y += term
    assert torch.equal(y, want) and torch.equal(torch.autograd.grad(y, term, g)[0], g)
  xr, wr = x.detach().requires_grad_(True), w.clone().requires_grad_(True)
  y = L.hip_linear_fp8(xr, wr)
  want = torch.autograd.grad(y, (xr, wr), g)
  y = L.hip_linear_fp8(xr, wr)
  y += term
  for a, b in zip(torch.autograd.grad(y, (xr, wr, term), g), (*want, g)):
    assert torch.equal(a, b)
  vr, g = v.clone().requires_grad_(True), rand(dev, *shape, seed=6, dtype=BF16)
  y = L.hip_layer_norm(xr, vr)
  y += 1.0
  assert torch.equal(torch.autograd.grad(y, vr, g)[0], torch.autograd.grad(L.hip_layer_norm(xr, vr), vr, g)[0])


# ------------------------------------------------------------------------------------------------ saved-tensor hooks
@pytest.mark.parametrize("xt", [BF16, F32])
def test_saved_tensor_hooks(dev, xt):
  """What a hook hands back is used where it is what was saved (a copy, as an offloading hook returns it), and refused where its dtype
  is another one."""
  x, w, v = rand(dev, 2, 5, 256, seed=1, dtype=xt), rand(dev, 256, seed=2), rand(dev, 130, 256, seed=3, dtype=BF16)
  x, w, v = (t.requires_grad_(True) for t in (x, w, v))
  norm_python = lambda: L.hip_layer_norm(torch.cat((x, x), -1)[..., :256].transpose(0, 1)[:, :, None], torch.cat((w, w))[::2], None)
  calls = {"norm": (lambda: L.hip_layer_norm(x, w), (x, w)), "norm, plain": (lambda: L.hip_layer_norm(x), (x,)), "norm, Python node": (norm_python, (x, w))}
  if xt == BF16:
    calls["linear"] = (lambda: L.hip_linear_fp8(x, v), (x, v))
    calls["linear, Python node"] = (lambda: L.hip_linear_fp8(torch.cat((x, x), -1)[..., :256], v), (x, v))
  swaps = {BF16: F32, F32: BF16, torch.uint8: F32}
  for name, (call, leaves) in calls.items():
    print(name, flush=True)
    loss = lambda y: y.float().square().sum()
    want = torch.autograd.grad(loss(call()), leaves)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(dev)):
      out = call()
    for a, b in zip(torch.autograd.grad(loss(out), leaves), want):
      assert torch.equal(a, b), name
    for which in {t.dtype for t in leaves}:  # x alone, the weight alone, or both where they are of one type
      lossy = lambda t: t.to(swaps[t.dtype]) if t.dtype == (torch.uint8 if name.startswith("linear") else which) else t
      with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lossy):
        out = call()
      with pytest.raises(ValueError):
        torch.autograd.grad(out, leaves, torch.ones_like(out))


# ------------------------------------------------------------------------------------------------ autograd's other modes
def test_second_derivatives_are_refused(dev):
  """A penalty on gradients fails, and does not come out as a constant."""
  x, w, v = rand(dev, 2, 5, 256, seed=1, dtype=BF16), rand(dev, 256, seed=2), rand(dev, 128, 256, seed=3, dtype=BF16)
  x, w, v = (t.requires_grad_(True) for t in (x, w, v))
  apart = lambda: torch.cat((x, x), -1)[..., :256]
  op = A.AttentionOp(attention_kernel="hip_flash", scale=0.125, heads=4, dim_head=64, dtype=BF16)
  hw = torch.ones(256, dtype=BF16, device=dev, requires_grad=True)
  calls = {"norm": lambda: L.hip_layer_norm(x, w), "norm, Python node": lambda: L.hip_layer_norm(apart().transpose(0, 1)[:, :, None], torch.cat((w, w))[::2]),
           "linear": lambda: L.hip_linear_fp8(x, v), "linear, Python node": lambda: L.hip_linear_fp8(apart(), v),
           "attention": lambda: op.apply_attention(x, x, x), "prologue": lambda: A.hip_norm_rope(x, x, hw, hw, None, 4)[0]}
  for name, call in calls.items():
    print(name, flush=True)
    loss = lambda: call().float().square().sum()
    (plain,) = torch.autograd.grad(loss(), x)
    (dx,) = torch.autograd.grad(loss(), x, create_graph=True)
    assert torch.equal(dx, plain) and dx.requires_grad and not plain.requires_grad
    with pytest.raises(NotImplementedError, match="second derivatives"):
      torch.autograd.grad(dx.float().square().sum() + x.float().sum(), x)


@pytest.mark.parametrize("recording", [True, False])
def test_tangents_are_refused(dev, recording):
  """Forward-mode differentiation fails, and does not lose its tangent."""
  x, w, v = rand(dev, 2, 5, 256, seed=1, dtype=BF16), rand(dev, 256, seed=2), rand(dev, 128, 256, seed=3, dtype=BF16)
  w8, hw = L.quantize_weight(v), rand(dev, 256, seed=4, dtype=BF16)
  op = A.AttentionOp(attention_kernel="hip_flash", scale=0.125, heads=4, dim_head=64, dtype=BF16)
  with forward_ad.dual_level(), torch.set_grad_enabled(recording):
    d, e, f = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w, v))
    for call in (lambda: L.hip_layer_norm(d), lambda: L.hip_layer_norm(x, e), lambda: L.hip_linear_fp8(d, w8), lambda: L.hip_linear_fp8(x, f),
                 lambda: L.hip_layer_norm_linear_fp8(d, w, None, w8), lambda: L.hip_layer_norm_linear_fp8(x, e, None, w8),
                 lambda: op.apply_attention(d, x, x), lambda: op.apply_attention(x, x, d), lambda: A.hip_norm_rope(d, x, hw, hw, None, 4),
                 lambda: A.hip_norm_rope_ltx2(d, x, w, w, 4), lambda: A.hip_norm_rope_ltx2(x, x, e, w, 4)):
      with pytest.raises(NotImplementedError, match="tangents"):
        call()


# ------------------------------------------------------------------------------------------------ arguments
@pytest.mark.parametrize("offset", [1.0, -1.0, 1e8, 3e38, float("inf")])
def test_the_weight_offset_is_the_weights(dev, offset):
  """Without a weight the factor is 1, whatever the offset."""
  x, b, g = rand(dev, 2, 5, 200, seed=1), rand(dev, 200, seed=2), rand(dev, 2, 5, 200, seed=3)
  for bias in (None, b):
    assert torch.equal(ops.layer_norm(x, None, bias, weight_offset=offset), ops.layer_norm(x, None, bias))
    got, want = ops.layer_norm_quant(x, None, bias, weight_offset=offset), ops.layer_norm_quant(x, None, bias)
    assert torch.equal(got.values, want.values) and torch.equal(got.scales[:, :2], want.scales[:, :2])
    for p, q in zip(ops.layer_norm_backward(x, None, bias, g, 1e-6, offset), ops.layer_norm_backward(x, None, bias, g)):
      assert (p is None and q is None) or torch.equal(p, q)


@pytest.mark.parametrize("shape", [(3, 0), (2, 3, 0), (2, 0, 0), (0,)])
def test_linear_over_an_empty_axis(dev, shape):
  """A sum over nothing: the bias alone, and gradients of no elements."""
  x, g = torch.empty(shape, dtype=BF16, device=dev), rand(dev, *shape[:-1], 4, seed=1, dtype=BF16)
  w, b = torch.empty((4, 0), dtype=BF16, device=dev), rand(dev, 4, seed=2, dtype=BF16)
  want = b.expand(*shape[:-1], 4)
  assert torch.equal(L.hip_linear_fp8(x, w, b), want) and torch.equal(L.hip_linear_fp8(x, L.quantize_weight(w), b), want)
  assert torch.equal(L.hip_linear_fp8(x, w), torch.zeros_like(want))
  x, w, b = (t.requires_grad_(True) for t in (x, w, b))
  y = L.hip_linear_fp8(x, w, b)
  dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
  assert torch.equal(y, want) and dx.shape == x.shape and dw.shape == w.shape
  if len(shape) > 1:
    assert torch.equal(db, g.float().reshape(-1, 4).sum(0).to(BF16))
    w8 = L.quantize_weight(w.detach())
    assert torch.equal(L.hip_layer_norm_linear_fp8(x.detach(), None, None, w8, b.detach()), want)


def test_tensors_without_axes_are_refused(dev):
  x, one = rand(dev, 2, 3, 64, seed=1), torch.ones((), device=dev)
  w8 = L.quantize_weight(rand(dev, 8, 64, seed=2))
  for call in (lambda: L.hip_layer_norm(one), lambda: L.hip_layer_norm(x, one), lambda: L.hip_layer_norm(x, None, one), lambda: L.hip_linear_fp8(one, w8),
               lambda: L.hip_linear_fp8(x, w8, one), lambda: L.hip_linear_fp8(x, one), lambda: L.hip_layer_norm_linear_fp8(x, one, None, w8)):
    with pytest.raises(ValueError):
      call()


# ------------------------------------------------------------------------------------------------ every form of the product
# (few rows; tiles of 128 and of 256; either with K split, which only its workspace says; whole rounds of tiles and what they leave)
FORMS = [(7, 300, 4100, 0), (30, 1501, 1000, 0), (130, 300, 4096, 128), (700, 900, 4096, 128), (333, 520, 1000, None), (2900, 1507, 15759, 256), (2900, 1504, 15759, 256),
         (4200, 3800, 900, None), (3900, 4051, 1100, None), (4300, 4096, 4100, 128)]


def test_forms_are_the_ones_that_are_meant(lib):
  for m, n, k, tile in FORMS:
    floats = lib.mdattn_matmul_fp8_block_workspace_floats(m, n, k)
    if not tile:
      assert floats == 0
      continue
    rows = m if m < 4300 else m - 4096  # (whole rounds of 16 x 16 tiles of 256 go first)
    area = -(-rows // tile) * tile * -(-n // tile) * tile
    assert floats >= 2 * area and floats % area == 0
    if tile == 256:  # and not of 128
      assert floats % (-(-rows // 128) * 128 * -(-n // 128) * 128) != 0


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("m,n,k,tile", FORMS)
def test_product_by_every_form(dev, m, n, k, tile, block_rows):
  """Scale bytes that differ between rows and blocks, sums that need f32: exact, with a bias and without."""
  for make in (layer_inputs.scaled, layer_inputs.cancelling):
    a, b, want = make(m, n, k, dev, seed=m + block_rows)
    qa, qb = ops.quant_block_e4m3(a), ops.quant_block_e4m3(b, block_rows)
    assert torch.equal(qa.dequantize(), a) and torch.equal(qb.dequantize(), b)  # (blocks hold them as they are)
    assert torch.equal(ops.matmul_fp8_block(qa, qb).float(), want)
    bias = torch.randint(-4, 5, (n,), device=dev).float()
    for t in (bias, bias.to(BF16)):
      assert torch.equal(ops.matmul_fp8_block(qa, qb, t).float(), (want + bias).to(BF16).float())


# ------------------------------------------------------------------------------------------------ the norm
@pytest.mark.parametrize("xt", [BF16, F32])
@pytest.mark.parametrize("c", [6145, 6200, 8191, 8192, 12288, 12289, 16383, 16384])
def test_wide_norm_into_blocks(dev, c, xt):
  """Teams of 512 and 1,024 threads, with a last block that the row ends in: values, scale bytes and the zeros behind the row."""
  x = rand(dev, 2, 37, c, seed=c, dtype=xt) + 0.5
  w, b = (rand(dev, 2, c, seed=i, std=0.3) for i in (2, 3))
  got = ops.layer_norm_quant(x, w, b, weight_offset=1.0)
  rows = ops.layer_norm(x, w, b, weight_offset=1.0, out_dtype=F32)
  want, _, _, _, size = norm64(x, w, b, 1e-6, 1.0)
  close(rows, want, half_ulp(want, F32) + 16 * 2.0**-24 * size, str(c))
  assert_quant(got, rows.view(-1, c), 1, str(c))
  assert not bool(got.values[:, c:].any())


@pytest.mark.parametrize("xt", [BF16, F32])
def test_norm_by_views_of_a_modulation(dev, xt):
  """adaLN's scale and shift as a model has them, chunks of [B, 6, C]: the results of dense copies, and the gradient of the whole."""
  x, g = rand(dev, 3, 50, 264, seed=1, dtype=xt), rand(dev, 3, 50, 264, seed=2, dtype=xt)
  m = rand(dev, 3, 6, 264, seed=3).requires_grad_(True)
  shift, scale = m.chunk(6, dim=1)[:2]
  s, t = (v.detach().contiguous().requires_grad_(True) for v in (scale, shift))
  w8 = L.quantize_weight(rand(dev, 130, 264, seed=4))
  with torch.no_grad():
    assert torch.equal(L.hip_layer_norm(x, scale, shift, weight_offset=1.0), L.hip_layer_norm(x, s, t, weight_offset=1.0))
    assert torch.equal(L.hip_layer_norm_linear_fp8(x, scale, shift, w8, weight_offset=1.0), L.hip_layer_norm_linear_fp8(x, s, t, w8, weight_offset=1.0))
  x = x.requires_grad_(True)
  dx, dm = torch.autograd.grad(L.hip_layer_norm(x, scale, shift, weight_offset=1.0), (x, m), g)
  wx, ws, wt = torch.autograd.grad(L.hip_layer_norm(x, s, t, weight_offset=1.0), (x, s, t), g)
  assert torch.equal(dx, wx) and torch.equal(dm, torch.cat((wt, ws, torch.zeros(3, 4, 264, device=dev)), 1))


# ------------------------------------------------------------------------------------------------ all of them in one block
def test_gradients_of_the_example_block(dev):
  """Each weight's gradient against that of the block in 64 bits on the CPU, its dense layers' operands as blocks of e4m3 hold them and rounding
  passed through.  Left is what the kernels round beside: the output gradients, and x along the tokens, to e4m3 (2^-4 of a value at most, 2^-5
  of a vector's length), in up to four products between the loss and a weight, a tenth in all if none cancels, and bf16 between the layers;
  attention's backward subtracts, which is allowed to double it, and the sum of both to grow by a quarter."""
  path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "wan_block_fp8.py")
  spec = importlib.util.spec_from_file_location("wan_block_fp8", path)
  ex = importlib.util.module_from_spec(spec)
  spec.loader.exec_module(ex)
  heads, grid = 2, (3, 6, 7)
  block = ex.make_block(heads, dev)
  x, modulation, freqs = rand(dev, 2, 126, 256, seed=1, dtype=BF16), rand(dev, 6, 2, 256, seed=2, std=0.1), ex.rotary_table(*grid, dev)

  class Held(torch.autograd.Function):
    @staticmethod
    def forward(ctx, t, block_rows):
      v, byte = blocks64(t, block_rows)
      scale = torch.exp2(byte.double() - 127).repeat_interleave(block_rows, 0)[: t.shape[0]].repeat_interleave(128, 1)
      return (v.view(torch.float8_e4m3fn).double() * scale)[:, : t.shape[1]]

    @staticmethod
    def backward(ctx, g):
      return g, None

  plain = {n: t.cpu().double().requires_grad_(True) for n, t in block.items()}
  y = plain_block(plain, x.cpu(), modulation.cpu(), freqs.cpu(), heads, Held.apply)
  want = torch.autograd.grad(y.square().mean(), list(plain.values()))
  leaves = [t.requires_grad_(True) for t in block.values()]
  z = ex.run_block(block, x, modulation, freqs, heads)
  for name, g, w in zip(block, torch.autograd.grad(z.float().square().mean(), leaves), want):
    off = (g.cpu().double() - w).norm() / w.norm()
    print(f"{name}: {off.item():.4f}")
    assert off <= 0.25, name
