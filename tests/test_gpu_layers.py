"""Layer norm, quantisation in blocks of 128 and products of such operands, against plain implementations in 64 bits.

Tolerances.  u = 2^-24, f32's unit roundoff.  A norm's output: one rounding to its type, and f32 arithmetic whose error is a few u of
the sizes that meet in it, |w h| + |b| and, through the mean, |w| r max|x|: 16 u of their sum.  A sum of n terms in f32: (sqrt(n) + 8) u of the
sum of magnitudes would be the likely error; 2 sqrt(n) + 16 is allowed.  A product of e4m3 operands: a group of eight products is
cut at 2^-14 of its largest, at most 8 * 2^-14 = 2^-11 of the sum of magnitudes, and bf16, of 8 significant bits, rounds by 2^-8 at most.  Quantised values and
whole numbers are equal, bit for bit."""
import math

import pytest
import torch

from maxdiffusion_amd import _lib, layer_op as L
from maxdiffusion_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0**-24
BF16, F32 = torch.bfloat16, torch.float32


def rand(dev, *shape, seed=0, dtype=F32, std=1.0, mean=0.0):
  gen = torch.Generator(device=dev).manual_seed(seed)
  return (torch.randn(shape, generator=gen, device=dev) * std + mean).to(dtype)


def half_ulp(t, dtype):
  return t.abs() * (2.0**-8 if dtype == BF16 else U) + 1e-38


def close(got, want, tol, what):
  off = (got.double() - want).abs()
  assert got.shape == want.shape
  assert bool((off <= tol).all()), f"{what}: {(off - tol).max().item():.3g} over, {off.max().item():.3g} off"


# ------------------------------------------------------------------------------------------------ layer norm
def vector(v, x):
  return v.double() if v.dim() == 1 else v.double().reshape(v.shape[0], *([1] * (x.dim() - 2)), v.shape[-1])


def norm64(x, w, b, eps, off):
  x = x.double()
  mean = x.mean(-1, keepdim=True)
  r = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
  h = (x - mean) * r
  m = 1.0 if w is None else off + vector(w, x)
  y = h * m + (0.0 if b is None else vector(b, x))
  size = (h * m).abs() + (0.0 if b is None else vector(b, x).abs()) + (r * x.abs().amax(-1, keepdim=True)) * (m if w is None else m.abs())
  return y, h, r, m, size


SHAPES = [(1, 1, 1), (1, 1, 8), (2, 3, 7), (1, 126, 512), (2, 5, 513), (3, 1, 1001), (1, 9, 1024), (1, 7, 1025), (2, 33, 1536), (1, 5, 5120),
          (1, 3, 8184), (1, 2, 16384), (4, 700, 64), (1, 4097, 72)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("xt,wt,per_batch,off", [(BF16, F32, True, 1.0), (F32, BF16, False, 0.0)])
def test_norm_forward(dev, shape, xt, wt, per_batch, off):
  b, s, c = shape
  x = rand(dev, *shape, seed=1, dtype=xt, mean=0.3)
  w, v = (rand(dev, *((b, c) if per_batch else (c,)), seed=i, dtype=wt, std=0.5) for i in (2, 3))
  for weight, bias in ((w, v), (None, None), (w, None), (None, v)):
    for out in (BF16, F32):
      got = ops.layer_norm(x, weight, bias, 1e-6, off, out_dtype=out)
      want, _, _, _, size = norm64(x, weight, bias, 1e-6, off)
      close(got, want, half_ulp(want, out) + 16 * U * size, f"{shape} {out}")
      assert torch.equal(got, ops.layer_norm(x, weight, bias, 1e-6, off, out_dtype=out))


@pytest.mark.parametrize("c", [512, 2048, 5120])
def test_norm_of_rows_far_from_zero(dev, c):
  """A mean of 1,000 deviations: the squares are summed around it, nothing cancels."""
  x = rand(dev, 1, 40, c, seed=4, mean=1000.0)
  want, _, _, _, size = norm64(x, None, None, 1e-6, 0.0)
  close(ops.layer_norm(x), want, 16 * U * size, "far")


def test_norm_of_equal_values_and_of_what_is_not_finite(dev):
  x = torch.full((3, 640), 7.0, device=dev)
  assert torch.equal(ops.layer_norm(x), torch.zeros_like(x))  # no deviation: h is 0
  x = rand(dev, 4, 640, seed=5)
  x[1, 100] = math.inf
  x[2, 3] = math.nan
  y = ops.layer_norm(x)
  assert bool(y[1].isnan().all()) and bool(y[2].isnan().all()) and bool(y[[0, 3]].isfinite().all())
  q = ops.layer_norm_quant(x)
  assert bool((q.scales[[1, 2], :5] == 255).all()) and bool(q.dequantize()[[0, 3]].isfinite().all())


@pytest.mark.parametrize("xt", [BF16, F32])
@pytest.mark.parametrize("c", [64, 1001, 1536])
def test_norm_walks_strides_and_odd_addresses(dev, xt, c):
  big = rand(dev, 3, 11, 2 * c + 3, seed=6, dtype=xt)
  x = big[:, 1:, 1:1 + c]  # rows apart, one element off
  g = rand(dev, 3, 10, c + 5, seed=7, dtype=xt)[..., 3:3 + c]
  w, b = (rand(dev, 3, c + 1, seed=i)[:, 1:].contiguous() for i in (8, 9))
  assert torch.equal(ops.layer_norm(x, w, b), ops.layer_norm(x.contiguous(), w, b))
  flat = torch.zeros(c * 3 + 1, device=dev)
  flat[1:] = w.reshape(-1)
  assert torch.equal(ops.layer_norm(x, flat[1:].view(3, c), b), ops.layer_norm(x, w, b))
  for a, d in zip(ops.layer_norm_backward(x, w, b, g), ops.layer_norm_backward(x.contiguous(), w, b, g.contiguous())):
    assert torch.equal(a, d)
  assert torch.equal(L.hip_layer_norm(big.transpose(0, 1)[1:, :, 1:1 + c]), ops.layer_norm(x.transpose(0, 1).contiguous()))


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("xt,wt,per_batch,off", [(BF16, F32, True, 1.0), (F32, F32, False, 0.0), (BF16, BF16, False, 0.0)])
def test_norm_backward(dev, shape, xt, wt, per_batch, off):
  b, s, c = shape
  x, g = rand(dev, *shape, seed=1, dtype=xt, mean=0.3), rand(dev, *shape, seed=2, dtype=xt)
  w, v = (rand(dev, *((b, c) if per_batch else (c,)), seed=i, dtype=wt, std=0.5) for i in (3, 4))
  eps = 1e-3 if c < 8 else 1e-6  # (of few channels h and its gradient are all cancellation)
  dx, dw, db = ops.layer_norm_backward(x, w, v, g, eps, off)
  _, h, r, m, _ = norm64(x, w, v, eps, off)
  gd = g.double()
  a = gd * m
  c1, c2 = a.mean(-1, keepdim=True), (a * h).mean(-1, keepdim=True)
  want = r * (a - c1 - h * c2)
  # the sizes that meet: a, its means over the row, and h with the error that the mean's rounding leaves in it
  mag = a.abs().mean(-1, keepdim=True)
  hx = h.abs() + r * x.double().abs().amax(-1, keepdim=True)
  size = r * (a.abs() + mag + hx * (a * h).abs().mean(-1, keepdim=True) + h.abs() * (a.abs() * hx).mean(-1, keepdim=True))
  close(dx, want, half_ulp(want, xt) + 32 * U * size, f"dx {shape}")
  over = 1 if per_batch else (0, 1)
  n = s if per_batch else b * s
  slack = (2 * math.sqrt(n) + 16) * U
  want_w, want_b = (gd * h).sum(over), gd.sum(over)
  close(dw, want_w, half_ulp(want_w, wt) + slack * (gd.abs() * hx).sum(over), f"dw {shape}")
  close(db, want_b, half_ulp(want_b, wt) + slack * gd.abs().sum(over), f"db {shape}")
  for p, q in zip((dx, dw, db), ops.layer_norm_backward(x, w, v, g, eps, off)):
    assert torch.equal(p, q)  # fixed order of every sum
  only, none_w, none_b = ops.layer_norm_backward(x, w, v, g, eps, off, needs_vectors=False)
  assert torch.equal(only, dx) and none_w is None and none_b is None
  dx0, n0, db0 = ops.layer_norm_backward(x, None, v, g, eps, off)
  assert n0 is None and torch.equal(db0, db) and bool(dx0.isfinite().all())


def test_norm_gradient_against_differences(dev):
  """The kernel's gradient against central differences of the formula in 64 bits, along directions in x, w and b."""
  x, g = rand(dev, 2, 6, 200, seed=11), rand(dev, 2, 6, 200, seed=12)
  w, b = rand(dev, 2, 200, seed=13, std=0.3), rand(dev, 2, 200, seed=14)
  grads = ops.layer_norm_backward(x, w, b, g, 1e-6, 1.0)
  loss = lambda x, w, b: (norm64(x, w, b, 1e-6, 1.0)[0] * g.double()).sum()
  at = [x.double(), w.double(), b.double()]
  for i, grad in enumerate(grads):
    d = rand(dev, *grad.shape, seed=20 + i).double()
    step = 1e-4
    hi, lo = ([a + (k * step * d if j == i else 0) for j, a in enumerate(at)] for k in (1, -1))
    want = (loss(*hi) - loss(*lo)) / (2 * step)  # (third derivatives of order one: an error of 1e-8)
    got = (grad.double() * d).sum()
    assert abs(got - want) <= 1e-6 * (grad.double() * d).abs().sum()


def test_norm_through_autograd_with_expanded_gradients(dev):
  x = rand(dev, 2, 50, 96, seed=1, dtype=BF16).requires_grad_(True)
  w, b = (rand(dev, 2, 1, 96, seed=i).requires_grad_(True) for i in (2, 3))
  y = L.hip_layer_norm(x, w, b, weight_offset=1.0)
  dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))  # the gradient is one value, expanded
  want = ops.layer_norm_backward(x.detach(), w.detach(), b.detach(), torch.ones_like(x), 1e-6, 1.0)
  for p, q in zip((dx, dw, db), want):
    assert p.shape == q.shape and p.dtype == q.dtype and torch.equal(p, q)
  (only,) = torch.autograd.grad(L.hip_layer_norm(x, w.detach(), b.detach(), weight_offset=1.0).sum(), (x,))
  assert torch.equal(only, dx)


# ------------------------------------------------------------------------------------------------ quantisation
def blocks64(x, block_rows):
  """(values, scale bytes) of the definition in 64 bits; no infinities or NaN."""
  r, c = x.shape
  x = torch.nn.functional.pad(x.double(), (0, -c % 128, 0, -r % block_rows))
  t = x.reshape(x.shape[0] // block_rows, block_rows, x.shape[1] // 128, 128)
  m = t.abs().amax((1, 3))
  frac, exp = torch.frexp(m)
  e = torch.where(m > 0, exp - 9 + (frac > 0.875), torch.full_like(exp, -127)).clamp(min=-127)
  q = torch.ldexp(t, -e[:, None, :, None]).float().to(torch.float8_e4m3fn).view(torch.uint8).reshape(x.shape)
  return q[:r], (e + 127).to(torch.uint8)


def assert_quant(got, x, block_rows, what):
  q, s = blocks64(x, block_rows)
  assert (got.rows, got.cols, got.block_rows) == (*x.shape, block_rows)
  assert torch.equal(got.scales[:, :s.shape[1]], s), f"{what}: scales"
  same = (got.values == q) | ((got.values | q) == 0x80)  # (a zero's sign: the reference goes through f32)
  assert bool(same.all()), f"{what}: {int((~same).sum())} values"


QUANT = [(1, 1), (1, 128), (3, 129), (127, 64), (128, 512), (130, 1000), (333, 333), (257, 1280), (4097, 136)]


@pytest.mark.parametrize("shape", QUANT)
@pytest.mark.parametrize("xt", [BF16, F32])
def test_quantisation(dev, shape, xt):
  x = rand(dev, *shape, seed=1, dtype=xt) * torch.exp2(rand(dev, shape[0], 1, seed=2, std=6).round()).to(xt)
  x[:, ::7] = 0
  assert_quant(ops.quant_block_e4m3(x), x, 1, "rows")
  for br in (1, 128):
    q, qt, sums = ops.quant_block_e4m3(x, br, transposed=True, sums=True)
    assert_quant(q, x, br, f"blocks of {br}")
    assert_quant(qt, x.t(), br, f"transposed blocks of {br}")
    only = ops.quant_block_e4m3(x, br, plain=False, transposed=True)
    assert torch.equal(only.values, qt.values)
    want = x.double().sum(0)
    for out in (BF16, F32):
      close(ops.sum_rows(sums, out), want, half_ulp(want, out) + (2 * math.sqrt(shape[0]) + 16) * U * x.double().abs().sum(0), "sums")


def test_quantisation_walks_strides_and_odd_addresses(dev):
  big = rand(dev, 140, 300, seed=3, dtype=BF16)
  x = big[1:, 3:200]
  for br in (1, 128):
    a, at = ops.quant_block_e4m3(x, br, transposed=True)
    b, bt = ops.quant_block_e4m3(x.contiguous(), br, transposed=True)
    assert torch.equal(a.values, b.values) and torch.equal(at.values, bt.values) and torch.equal(a.scales[:, :2], b.scales[:, :2])
  assert torch.equal(ops.quant_block_e4m3(x).values, ops.quant_block_e4m3(x.contiguous()).values)


def test_quantisation_at_the_edges_of_the_range(dev):
  x = torch.zeros(8, 128, device=dev)
  x[1, 5] = 3.4e38
  x[2, 5] = 1e-45  # below every normal number
  x[3, 5] = 448.0
  x[4, 5] = 448.0000305  # the next f32: one scale up
  x[5, 5], x[5, 6] = 1.75 * 2.0**-118, -1e-38  # the smallest scale that is not clamped
  x[6, 5] = math.inf
  x[7, 5], x[7, 6] = math.nan, 3.0
  q = ops.quant_block_e4m3(x)
  assert q.scales[:6, 0].tolist() == [0, 247, 0, 127, 128, 1]
  assert_quant(q.__class__(q.values[:6].contiguous(), q.scales[:6].contiguous(), 6, 128, 1), x[:6], 1, "edges")
  assert q.scales[6:, 0].tolist() == [255, 255] and bool(q.dequantize()[6:].isnan().all())
  t = ops.quant_block_e4m3(x, 128)  # one block: not finite as a whole
  assert t.scales[0, 0] == 255


def test_norm_into_blocks(dev):
  """The quantised output is the quantisation of the rows that the f32 form of the norm stores."""
  for shape in ((1, 3, 64), (2, 70, 1001), (1, 40, 1536), (1, 5, 5120)):
    for xt in (BF16, F32):
      x = rand(dev, *shape, seed=1, dtype=xt)
      w, b = (rand(dev, shape[0], shape[2], seed=i, std=0.3) for i in (2, 3))
      got = ops.layer_norm_quant(x, w, b, weight_offset=1.0)
      rows = ops.layer_norm(x, w, b, weight_offset=1.0, out_dtype=F32).view(-1, shape[2])
      assert_quant(got, rows, 1, str(shape))


# ------------------------------------------------------------------------------------------------ products
PRODUCTS = [(1, 1, 1), (1, 7, 100), (1, 640, 5120), (2, 130, 128), (16, 1000, 512), (17, 48, 1000), (33, 333, 640), (64, 2048, 1536), (111, 333, 1000),
            (128, 128, 4096), (129, 129, 129), (257, 1280, 640), (300, 520, 8192), (512, 512, 512), (1000, 70, 2048), (2674, 1536, 256)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("block_rows", [1, 128])
def test_product(dev, m, n, k, block_rows):
  a = ops.quant_block_e4m3(rand(dev, m, k, seed=1) * torch.exp2(rand(dev, m, 1, seed=3, std=3).round()))
  b = ops.quant_block_e4m3(rand(dev, n, k, seed=2, std=k**-0.5), block_rows)
  ad, bd = a.dequantize(torch.float64), b.dequantize(torch.float64)
  want, size = ad @ bd.t(), ad.abs() @ bd.abs().t()
  for bias in (None, rand(dev, n, seed=4), rand(dev, n, seed=4, dtype=BF16)):
    got = ops.matmul_fp8_block(a, b, bias)
    w = want if bias is None else want + bias.double()
    # (half an ulp of the rounded sum, which may lie a little above the exact one)
    close(got, w, 2.0**-8 * w.abs() + (1 + 2.0**-8) * 2.0**-11 * size + 1e-38, f"{m} {n} {k}")
    assert torch.equal(got, ops.matmul_fp8_block(a, b, bias))


@pytest.mark.parametrize("m,n,k", [(5, 48, 384), (130, 300, 1152), (300, 300, 640)])
def test_product_of_whole_numbers_is_exact(dev, m, n, k):
  """Small whole numbers, sums below 256: every step is exact, at any split and in any order."""
  gen = torch.Generator(device=dev).manual_seed(0)
  pick = lambda r: torch.randint(-2, 3, (r, k), generator=gen, device=dev) * (torch.rand((r, k), generator=gen, device=dev) < 0.2)
  a, b = pick(m), pick(n)
  want = (a.double() @ b.double().t())
  assert want.abs().max() < 256
  got = ops.matmul_fp8_block(ops.quant_block_e4m3(a.to(BF16)), ops.quant_block_e4m3(b.to(BF16), 128))
  assert torch.equal(got.double(), want)


def test_product_with_blocks_that_are_not_finite(dev):
  x, w = rand(dev, 200, 512, seed=1), rand(dev, 150, 512, seed=2)
  x[7, 300] = math.nan
  x[150, 0] = math.inf
  y = ops.matmul_fp8_block(ops.quant_block_e4m3(x), ops.quant_block_e4m3(w, 128))
  assert bool(y[[7, 150]].isnan().all()) and int(y.isnan().any(1).sum()) == 2
  one = ops.matmul_fp8_block(ops.quant_block_e4m3(x[7:8].contiguous()), ops.quant_block_e4m3(w, 128))
  assert bool(one.isnan().all())


def test_product_into_wider_rows_leaves_what_is_between(dev, lib):
  """The C entry's output stride, odd, at an odd address."""
  import ctypes

  P = ctypes.c_void_p
  a, b = ops.quant_block_e4m3(rand(dev, 140, 256, seed=1)), ops.quant_block_e4m3(rand(dev, 130, 256, seed=2), 128)
  out = torch.full((140 * 151 + 1,), 7.0, dtype=BF16, device=dev)
  rc = lib.mdattn_matmul_fp8_block(P(torch.cuda.current_stream().cuda_stream), P(a.values.data_ptr()), P(a.scales.data_ptr()), P(b.values.data_ptr()),
                                   P(b.scales.data_ptr()), 128, None, 0, P(out.data_ptr() + 2), 151, 140, 130, 256, None, 0)
  assert rc == _lib.E_OK
  rows = out[1:].view(140, 151)
  assert torch.equal(rows[:, :130], ops.matmul_fp8_block(a, b)) and bool((rows[:, 130:] == 7).all()) and out[0] == 7


@pytest.mark.parametrize("shape,n", [((1, 1, 512), 200), ((2, 65, 200), 130), ((300, 640), 384)])
def test_linear_gradients(dev, shape, n):
  """Each product against the same in 64 bits of the operands as they are quantised."""
  k = shape[-1]
  x = rand(dev, *shape, seed=1, dtype=BF16).requires_grad_(True)
  w = rand(dev, n, k, seed=2, dtype=BF16, std=k**-0.5).requires_grad_(True)
  b = rand(dev, n, seed=3, dtype=BF16).requires_grad_(True)
  dy = rand(dev, *shape[:-1], n, seed=4, dtype=BF16, std=1e-3)
  y = L.hip_linear_fp8(x, w, b)
  grads = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
  xs, ws, gs = x.detach().reshape(-1, k), w.detach(), dy.reshape(-1, n)
  held = lambda t, br=1: ops.quant_block_e4m3(t.contiguous(), br).dequantize(torch.float64)
  pairs = [(y.detach().reshape(-1, n), held(xs), held(ws, 128).t(), b.detach().double()), (grads[0].reshape(-1, k), held(gs), held(ws, 128), 0.0),
           (grads[1], held(gs.t()), held(xs.t()).t(), 0.0)]
  for got, p, q, add in pairs:
    want = p @ q + add
    close(got, want, 2.0**-8 * want.abs() + (1 + 2.0**-8) * 2.0**-11 * (p.abs() @ q.abs()) + 1e-38, f"{shape} {n}")
  want = gs.double().sum(0)
  close(grads[2], want, half_ulp(want, BF16) + (2 * math.sqrt(len(gs)) + 16) * U * gs.double().abs().sum(0), "db")
  for i, t in enumerate((x, w, b)):  # each alone
    (one,) = torch.autograd.grad(L.hip_linear_fp8(*(s if j == i else s.detach() for j, s in enumerate((x, w, b)))), (t,), dy)
    assert torch.equal(one, grads[i])
  with torch.no_grad():
    assert torch.equal(L.hip_linear_fp8(x, w, b), y) and torch.equal(L.hip_linear_fp8(x, L.quantize_weight(w), b), y)


def test_linear_gradient_against_differences(dev):
  """Whole numbers, which quantisation leaves as they are: the layer is linear in each argument, and differences are exact."""
  gen = torch.Generator(device=dev).manual_seed(1)
  pick = lambda *s: (torch.randint(-2, 3, s, generator=gen, device=dev) * (torch.rand(s, generator=gen, device=dev) < 0.2)).to(BF16)
  x, w, dy = pick(60, 150), pick(70, 150), pick(60, 70)
  xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
  dx, dw = torch.autograd.grad(L.hip_linear_fp8(xr, wr), (xr, wr), dy)
  d = pick(60, 150)
  with torch.no_grad():
    up, down = L.hip_linear_fp8(x + d, w), L.hip_linear_fp8(x - d, w)
    assert ((up.double() - down.double()) / 2 * dy.double()).sum() == (dx.double() * d.double()).sum()
    e = pick(70, 150)
    up, down = L.hip_linear_fp8(x, w + e), L.hip_linear_fp8(x, w - e)
    assert ((up.double() - down.double()) / 2 * dy.double()).sum() == (dw.double() * e.double()).sum()


def test_norm_and_linear_together(dev):
  for shape, n in (((1, 1, 512), 700), ((2, 77, 1001), 130), ((1, 300, 1536), 512)):
    x = rand(dev, *shape, seed=1, dtype=BF16)
    w, b = (rand(dev, shape[0], shape[2], seed=i, std=0.3) for i in (2, 3))
    w8, ob = L.quantize_weight(rand(dev, n, shape[2], seed=4)), rand(dev, n, seed=5, dtype=BF16)
    got = L.hip_layer_norm_linear_fp8(x, w, b, w8, ob, weight_offset=1.0)
    rows = ops.layer_norm(x, w, b, weight_offset=1.0, out_dtype=F32)
    assert torch.equal(got, L.hip_linear_fp8(rows, w8, ob))


# ------------------------------------------------------------------------------------------------ sizes of nothing, streams, graphs
def test_no_rows(dev):
  x = torch.empty((2, 0, 64), dtype=BF16, device=dev)
  w = rand(dev, 64, seed=1).requires_grad_(True)
  xr = x.clone().requires_grad_(True)
  y = L.hip_layer_norm(xr, w, w)
  assert y.shape == x.shape
  dx, dw = torch.autograd.grad(y, (xr, w), torch.empty_like(y))
  assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))
  w8 = L.quantize_weight(rand(dev, 40, 64, seed=2, dtype=BF16))
  assert L.hip_linear_fp8(x, w8).shape == (2, 0, 40) and L.hip_layer_norm_linear_fp8(x, None, None, w8).shape == (2, 0, 40)
  wr, br = rand(dev, 40, 64, seed=2, dtype=BF16).requires_grad_(True), rand(dev, 40, seed=3, dtype=BF16).requires_grad_(True)
  y = L.hip_linear_fp8(xr, wr, br)
  dx, dw, db = torch.autograd.grad(y, (xr, wr, br), torch.empty_like(y))
  assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(wr)) and torch.equal(db, torch.zeros_like(br))


def step(s):
  y = L.hip_layer_norm(s["x"], s["w"], s["b"], weight_offset=1.0)
  z = L.hip_linear_fp8(y, s["p"], s["q"])
  return (z,) + torch.autograd.grad(z, (s["x"], s["w"], s["b"], s["p"], s["q"]), s["dz"])


def inputs(dev, seed):
  s = dict(x=rand(dev, 2, 150, 640, seed=seed, dtype=BF16), w=rand(dev, 2, 640, seed=seed + 1), b=rand(dev, 2, 640, seed=seed + 2),
           p=rand(dev, 384, 640, seed=seed + 3, dtype=BF16), q=rand(dev, 384, seed=seed + 4, dtype=BF16), dz=rand(dev, 2, 150, 384, seed=seed + 5, dtype=BF16))
  return {n: t.requires_grad_(n != "dz") for n, t in s.items()}


def test_another_stream(dev):
  s = inputs(dev, 1)
  want = step(s)
  torch.cuda.synchronize()
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    got = step(s)
  side.synchronize()
  assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_in_a_graph(dev):
  """Captured once, replayed over other inputs, with eager work between the replays."""
  s = inputs(dev, 1)
  w8 = L.quantize_weight(s["p"].detach())
  call = lambda: (L.hip_layer_norm_linear_fp8(s["x"], s["w"], s["b"], w8, s["q"], weight_offset=1.0), L.hip_layer_norm(s["x"], s["w"], s["b"]),
                  L.hip_linear_fp8(s["x"][:1, :1], w8), *ops.layer_norm_backward(s["x"], s["w"], s["b"], s["x"]))
  with torch.no_grad():
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      got = call()
    for seed in (10, 20, 30):
      for n, t in inputs(dev, seed).items():
        if n in ("x", "w", "b"):
          s[n].copy_(t)
      graph.replay()
      torch.cuda.synchronize()
      assert all(torch.equal(p, q) for p, q in zip(got, call()))


# ------------------------------------------------------------------------------------------------ all of them in one block
def plain_block(block, x, modulation, freqs, heads, held):
  """The example's block in 64 bits.  held(t, block_rows): a matrix as the dense layers' products see it."""
  shift1, scale1, gate1, shift2, scale2, gate2 = modulation.double()
  b = {n: t.double() for n, t in block.items()}

  def norm(h, scale, shift):
    return norm64(h, None, None, 1e-6, 0.0)[0] * (1 + scale[:, None]) + shift[:, None]

  def dense(h, name, bias=True):
    y = held(h.reshape(-1, h.shape[-1]), 1) @ held(b[name], 128).t()
    return y.reshape(*h.shape[:-1], -1) + (b[name + "_bias"] if bias else 0.0)

  def prologue(t, w):
    t = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
    t = torch.view_as_complex(t.reshape(*t.shape[:-1], heads, -1, 2)) * freqs[0, 0][None, :, None].to(torch.complex128)
    return torch.view_as_real(t).flatten(-2).transpose(1, 2)

  q, k, v = dense(norm(x.double(), scale1, shift1), "qkv").chunk(3, dim=-1)
  q, k = prologue(q, b["norm_q"]), prologue(k, b["norm_k"])
  v = v.reshape(*v.shape[:-1], heads, -1).transpose(1, 2)
  att = torch.softmax(q @ k.transpose(-1, -2).contiguous() * q.shape[-1] ** -0.5, dim=-1) @ v
  x = x.double() + gate1[:, None] * dense(att.transpose(1, 2).flatten(2), "out")
  h = torch.nn.functional.gelu(dense(norm(x, scale2, shift2), "up"), approximate="tanh")
  return x + gate2[:, None] * dense(h, "down")


def test_example_block(dev):
  """The example's block on a small clip, ragged against every tile: inference and training give one output, as near to 64 bits as
  operands that are rounded to bf16 between the layers and then to e4m3 can be (2^-4 of a value at most in the dense layers' inputs, which
  a sum over many of them averages out: a few hundredths of a half's output), and every weight gets a gradient."""
  import importlib.util
  import os

  path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "wan_block_fp8.py")
  spec = importlib.util.spec_from_file_location("wan_block_fp8", path)
  ex = importlib.util.module_from_spec(spec)
  spec.loader.exec_module(ex)
  heads, grid = 2, (3, 6, 7)
  block = ex.make_block(heads, dev)
  x = rand(dev, 2, 126, 256, seed=1, dtype=BF16)
  modulation, freqs = rand(dev, 6, 2, 256, seed=2, std=0.1), ex.rotary_table(*grid, dev)
  with torch.no_grad():
    y = ex.run_block(ex.quantize(block), x, modulation, freqs, heads)
  same = plain_block(block, x, modulation, freqs, heads, lambda t, br: ops.quant_block_e4m3(t.float().contiguous(), br).dequantize(torch.float64))
  full = plain_block(block, x, modulation, freqs, heads, lambda t, br: t)
  part = (full - x.double()).norm()  # what the block adds
  assert (y.double() - same).norm() <= 0.05 * part and (same - full).norm() <= 0.1 * part
  leaves = [t.requires_grad_(True) for t in block.values()]
  z = ex.run_block(block, x, modulation, freqs, heads)
  assert (z.double() - same).norm() <= 0.05 * part
  for name, g, t in zip(block, torch.autograd.grad(z.float().square().mean(), leaves), leaves):
    assert g.shape == t.shape and bool(g.isfinite().all()) and bool((g != 0).any()), name


# ------------------------------------------------------------------------------------------------ many tiles, long tensors, in place
@pytest.mark.parametrize("m,n,k", [(4116, 4096, 4096), (4300, 4096, 8192), (8200, 4500, 384), (8000, 2600, 4096), (16500, 4100, 1300)])
def test_product_of_several_rounds_of_tiles(dev, m, n, k):
  """Whole rounds of tiles and what they leave: a few rows, a split over K, a last round with idle workgroups.  Sums of whole numbers below
  256 are exact; as few nonzeros as that needs."""
  gen = torch.Generator(device=dev).manual_seed(0)
  pick = lambda r: torch.randint(-2, 3, (r, k), generator=gen, device=dev) * (torch.rand((r, k), generator=gen, device=dev) < 3.0 * k**-0.5)
  a, b = pick(m).float(), pick(n).float()
  want = a @ b.t()
  assert want.abs().max() < 256
  qa, qb = ops.quant_block_e4m3(a.to(BF16)), ops.quant_block_e4m3(b.to(BF16), 128)
  got = ops.matmul_fp8_block(qa, qb)
  assert torch.equal(got.float(), want)
  bias = torch.randint(-2, 3, (n,), generator=gen, device=dev).float()
  assert torch.equal(ops.matmul_fp8_block(qa, qb, bias).float(), (want + bias).to(BF16).float())


LONG = 430_000  # rows of 5,120: 2.2e9 elements, past 2^31


def test_norm_past_2_31_elements(dev):
  x = rand(dev, 1, LONG, 5120, seed=1, dtype=BF16)
  w, b = rand(dev, 5120, seed=2), rand(dev, 5120, seed=3)
  at = [0, 1, LONG // 2, 2**31 // 5120 - 1, 2**31 // 5120, LONG - 1]
  some = x[:, at].contiguous()
  y = ops.layer_norm(x, w, b, 1e-6, 0.0)
  want, _, _, _, size = norm64(some, w, b, 1e-6, 0.0)
  close(y[:, at], want, half_ulp(want, BF16) + 16 * U * size, "norm")
  dx, _, db = ops.layer_norm_backward(x, w, b, y, 1e-6, 0.0)
  _, h, r, m, _ = norm64(some, w, b, 1e-6, 0.0)
  a = y[:, at].double() * m
  want = r * (a - a.mean(-1, keepdim=True) - h * (a * h).mean(-1, keepdim=True))
  hx = h.abs() + r * some.double().abs().amax(-1, keepdim=True)
  size = r * (a.abs() + a.abs().mean(-1, keepdim=True) + hx * (a * h).abs().mean(-1, keepdim=True) + h.abs() * (a.abs() * hx).mean(-1, keepdim=True))
  close(dx[:, at], want, half_ulp(want, BF16) + 32 * U * size, "dx")
  # db: the sum of g's columns (in pieces: a tensor of g in 64 bits has no place here)
  total, size = torch.zeros(5120, device=dev, dtype=torch.float64), torch.zeros(5120, device=dev, dtype=torch.float64)
  for part in y[0].split(43_000):
    total += part.double().sum(0)
    size += part.double().abs().sum(0)
  close(db, total, half_ulp(total, F32) + (2 * math.sqrt(LONG) + 16) * U * size, "db")


def test_blocks_and_products_past_2_31_elements(dev):
  x = rand(dev, LONG, 5120, seed=1, dtype=BF16)
  at = [0, 2**31 // 5120 - 1, 2**31 // 5120, LONG - 1]
  q = ops.quant_block_e4m3(x)
  some = ops.quant_block_e4m3(x[at].contiguous())
  assert torch.equal(q.values[at], some.values) and torch.equal(q.scales[at], some.scales)
  q128, t128 = ops.quant_block_e4m3(x, 1, transposed=True)
  assert torch.equal(q128.values[at], some.values)
  last = x[LONG // 128 * 128 - 256 :]  # whole blocks of the transposed rows
  _, tail_t = ops.quant_block_e4m3(last, 1, transposed=True)
  assert torch.equal(t128.values[:, LONG // 128 * 128 - 256 : LONG], tail_t.values[:, : last.shape[0]])
  del t128, q128, x
  # rows of a, rows of b and rows of c past 2^31 bytes and elements
  b = ops.quant_block_e4m3(rand(dev, 5120, 5120, seed=2, std=5120**-0.5), 128)
  want, size = some.dequantize(torch.float64) @ b.dequantize(torch.float64).t(), some.dequantize(torch.float64).abs() @ b.dequantize(torch.float64).abs().t()
  tol = 2.0**-8 * want.abs() + (1 + 2.0**-8) * 2.0**-11 * size + 1e-38
  close(ops.matmul_fp8_block(q, b)[at], want, tol, "rows of a and of c")
  few = ops.quant_block_e4m3(rand(dev, 40, 5120, seed=4))
  want = few.dequantize(torch.float64) @ some.dequantize(torch.float64).t()
  size = few.dequantize(torch.float64).abs() @ some.dequantize(torch.float64).abs().t()
  tol = 2.0**-8 * want.abs() + (1 + 2.0**-8) * 2.0**-11 * size + 1e-38
  close(ops.matmul_fp8_block(few, q)[:, at], want, tol, "rows of b")
  one = ops.quant_block_e4m3(rand(dev, 40, 5120, seed=4)[:1].contiguous())
  close(ops.matmul_fp8_block(one, q)[:, at], want[:1], tol[:1], "rows of b, one row of a")


@pytest.mark.parametrize("c", [7, 512, 5120])
def test_norm_in_place_at_the_c_entry(dev, lib, c):
  import ctypes

  P = ctypes.c_void_p
  x = rand(dev, 2, 33, c, seed=1, dtype=BF16)
  want = ops.layer_norm(x, None, None, 1e-6)
  rc = lib.mdattn_layer_norm(P(torch.cuda.current_stream().cuda_stream), P(x.data_ptr()), 0, P(x.data_ptr()), 0, None, None, 1, 2, 33, c, 33 * c, c,
                             33 * c, c, 0, 1e-6, 0.0)
  assert rc == _lib.E_OK
  assert torch.equal(x, want)


# ------------------------------------------------------------------------------------------------ axes of one element, many groups
@pytest.mark.parametrize("shape,strides", [((1, 1, 1), (0, 0, 0)), ((1, 1, 5, 64), (9, 7, 64, 1)), ((2, 1, 3, 64), (192, 5, 64, 1)),
                                           ((1, 4, 1, 72), (3, 72, 11, 1)), ((3, 1), (1, 9)), ((1, 2, 3, 1), (0, 3, 1, 0))])
def test_norm_of_axes_of_one_element_with_any_stride(dev, shape, strides):
  """Such strides mean nothing, and `contiguous` leaves them as they are."""
  size = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
  x, g = (rand(dev, size, seed=i, dtype=BF16).as_strided(shape, strides) for i in (1, 2))
  plain_x, plain_g = (t.clone().reshape(-1).view(shape) for t in (x, g))
  w = rand(dev, shape[-1], seed=3)
  results = []
  for a, b in ((x, g), (plain_x, plain_g)):
    a, v = a.detach().requires_grad_(), w.clone().requires_grad_()
    y = L.hip_layer_norm(a, v, None, 1e-3)
    results.append((y, *torch.autograd.grad(y, (a, v), b)))
    ops_y = ops.layer_norm(a.detach(), w, None, 1e-3)
    assert torch.equal(ops_y, y)
  for p, q in zip(*results):
    assert torch.equal(p, q)


@pytest.mark.parametrize("per_group", [False, True])
def test_norm_of_very_many_groups(dev, per_group):
  b, s, c = 70_001, 2, 64
  x, g = rand(dev, b, s, c, seed=1, dtype=BF16), rand(dev, b, s, c, seed=2, dtype=BF16)
  w, v = (rand(dev, *((b, c) if per_group else (c,)), seed=i, std=0.5) for i in (3, 4))
  want, h, r, m, size = norm64(x, w, v, 1e-6, 1.0)
  close(ops.layer_norm(x, w, v, 1e-6, 1.0), want, half_ulp(want, BF16) + 16 * U * size, "y")
  dx, dw, db = ops.layer_norm_backward(x, w, v, g, 1e-6, 1.0)
  a = g.double() * m
  want = r * (a - a.mean(-1, keepdim=True) - h * (a * h).mean(-1, keepdim=True))
  hx = h.abs() + r * x.double().abs().amax(-1, keepdim=True)
  size = r * (a.abs() + a.abs().mean(-1, keepdim=True) + hx * (a * h).abs().mean(-1, keepdim=True) + h.abs() * (a.abs() * hx).mean(-1, keepdim=True))
  close(dx, want, half_ulp(want, BF16) + 32 * U * size, "dx")
  over, n = (1, s) if per_group else ((0, 1), b * s)
  want_w, want_b = (g.double() * h).sum(over), g.double().sum(over)
  slack = (2 * math.sqrt(n) + 16) * U
  close(dw, want_w, half_ulp(want_w, F32) + slack * (g.double().abs() * hx).sum(over), "dw")
  close(db, want_b, half_ulp(want_b, F32) + slack * g.double().abs().sum(over), "db")


def test_norm_of_strided_groups_that_share_vectors(dev):
  """Groups that are not one after the other, next to the same rows dense."""
  big = rand(dev, 5, 9, 200, seed=1, dtype=BF16)
  w = rand(dev, 200, seed=2)
  for x in (big[:, 2:7], big[:, :1], big[::2], big[1:2, 3:]):
    assert torch.equal(ops.layer_norm(x, w), ops.layer_norm(x.contiguous(), w))
    assert torch.equal(ops.layer_norm_quant(x, w).values, ops.layer_norm_quant(x.contiguous(), w).values)
    for p, q in zip(ops.layer_norm_backward(x, w, None, x)[:1], ops.layer_norm_backward(x.contiguous(), w, None, x.contiguous())[:1]):
      assert torch.equal(p, q)
