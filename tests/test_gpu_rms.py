"""RMS norm with the residual's addition against 64 bits, forward, backward and into blocks of e4m3.

Tolerances.  u = 2^-24, f32's unit roundoff.  s: one rounding.  y: one rounding, and f32 arithmetic whose error is a few u of the sizes that meet
in it, |w h| + |b|: 16 u.  The backward pass has s as it was rounded, by v (2^-8 in bf16, u in f32) of an element at most: r is off by v of
itself, h by 2 v, mean(a h) by 2 v of mean |a h|."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from maxdiffusion_amd import layer_op as L
from maxdiffusion_amd import ops
from test_gpu_layers import BF16, F32, SHAPES, U, assert_quant, close, half_ulp, rand, vector

pytestmark = pytest.mark.gpu
TYPES = [(BF16, None), (BF16, BF16), (BF16, F32), (F32, F32), (F32, None)]
HALF = {BF16: 2.0**-8, F32: U}


def rms64(x, res, w, b, eps, off):
  s = x.double() if res is None else x.double() + res.double()
  r = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
  h = s * r
  m = torch.ones((), dtype=torch.float64, device=x.device) if w is None else off + vector(w, x)
  t = torch.zeros((), dtype=torch.float64, device=x.device) if b is None else vector(b, x)
  return h * m + t, s, h, r, m, (h * m).abs() + t.abs()


def both(out, res):
  return (out, None) if res is None else out


@pytest.mark.parametrize("shape", SHAPES + [(2, 3, 12288), (1, 2, 6200)])
@pytest.mark.parametrize("xt,rt", TYPES)
@pytest.mark.parametrize("wt,per_batch,off", [(F32, True, 1.0), (BF16, False, 0.0)])
def test_forward(dev, shape, xt, rt, wt, per_batch, off):
  n, _, c = shape
  x = rand(dev, *shape, seed=1, dtype=xt, mean=0.3)
  res = None if rt is None else rand(dev, *shape, seed=2, dtype=rt, std=3.0)
  w, v = (rand(dev, *((n, c) if per_batch else (c,)), seed=i, dtype=wt, std=0.5) for i in (3, 4))
  for weight, bias in ((w, v), (None, None), (w, None), (None, v)):
    y, s = both(ops.rms_norm(x, weight, bias, res, 1e-6, off), res)
    want, ws, _, _, _, size = rms64(x, res, weight, bias, 1e-6, off)
    close(y, want, half_ulp(want, xt) + 16 * U * size, f"y {shape}")
    assert y.dtype == xt
    if res is not None:
      assert s.dtype == rt and torch.equal(s, (x.float() + res.float()).to(rt))
    # what is rounded to e4m3 are the f32 rows: those of operands that are f32
    rows = both(ops.rms_norm(x.float(), weight, bias, None if res is None else res.float(), 1e-6, off), res)[0]
    q, s8 = both(ops.rms_norm_quant(x, weight, bias, res, 1e-6, off), res)
    assert_quant(q, rows.view(-1, c), 1, f"blocks {shape}")
    assert res is None or torch.equal(s8, s)


@pytest.mark.parametrize("shape", SHAPES + [(2, 3, 12288), (1, 2, 6200)])
@pytest.mark.parametrize("xt,rt", TYPES)
@pytest.mark.parametrize("wt,per_batch,off", [(F32, True, 1.0), (BF16, False, 0.0)])
def test_backward(dev, shape, xt, rt, wt, per_batch, off):
  n, rows, c = shape
  st = rt or xt
  x = rand(dev, *shape, seed=1, dtype=xt, mean=0.3)
  res = None if rt is None else rand(dev, *shape, seed=2, dtype=rt, std=3.0)
  w, v = (rand(dev, *((n, c) if per_batch else (c,)), seed=i, dtype=wt, std=0.5) for i in (3, 4))
  g, gs = rand(dev, *shape, seed=5, dtype=xt), rand(dev, *shape, seed=6, dtype=st)
  s = x if res is None else ops.rms_norm(x, w, v, res, 1e-6, off)[1]
  narrow = st != xt
  _, _, h, r, m, _ = rms64(x, res, w, v, 1e-6, off)
  a = g.double() * m
  mean, size = (a * h).mean(-1, keepdim=True), (a * h).abs().mean(-1, keepdim=True)
  # from s as it was rounded, and from x and the residual where both are bf16
  for up, again in ((None, False), (gs, False), *(((None, True), (gs, True)) if rt == BF16 else ())):
    v_s = 0.0 if res is None or again else HALF[st]
    inputs = dict(s=x, residual=res) if again else dict(s=s)
    call = lambda: ops.rms_norm_backward(weight=w, bias=v, g=g, gs=up, eps=1e-6, weight_offset=off, narrow=narrow, **inputs)
    ds, dx, dw, db = call()
    want = r * (a - h * mean) + (0 if up is None else up.double())
    err = 32 * U * (r * (a.abs() + h.abs() * size) + (0 if up is None else up.double().abs()))
    err = err + v_s * (r * (a - h * mean)).abs() + 1.02 * r * h.abs() * (2 * v_s * mean.abs() + 2 * v_s * size)
    close(ds, want, half_ulp(want, st) + err, f"ds {shape}")
    assert (dx is None) == (not narrow) and (dx is None or torch.equal(dx, ds.to(BF16)) or bool(((dx.double() - want).abs() <= half_ulp(want, BF16) + err).all()))
    over, terms = ((1,), rows) if per_batch else ((0, 1), n * rows)
    gh = (g.double() * h).abs()
    want_w, want_b = (g.double() * h).sum(over), g.double().sum(over)
    close(dw, want_w, half_ulp(want_w, wt) + (2 * v_s * 1.02 + (2 * math.sqrt(terms) + 32) * U) * gh.sum(over), f"dw {shape}")
    close(db, want_b, half_ulp(want_b, wt) + (2 * math.sqrt(terms) + 16) * U * g.double().abs().sum(over), f"db {shape}")
    assert all(p is q or torch.equal(p, q) for p, q in zip((ds, dx, dw, db), call()))
  ds, dx, dw, db = ops.rms_norm_backward(s, w, v, g, gs, 1e-6, off, narrow=narrow)
  alone = ops.rms_norm_backward(s, w, v, g, gs, 1e-6, off, needs_vectors=False, narrow=narrow)
  assert torch.equal(alone[0], ds) and alone[2] is None and alone[3] is None
  only = ops.rms_norm_backward(s, None, v, g, gs, 1e-6, off, narrow=narrow)
  assert only[2] is None and torch.equal(only[3], db)


def test_gradients_against_differences(dev):
  """The formula in 64 bits, moved along random directions: the kernel's gradients, of f32 operands, predict the change."""
  x, res, g, gs = (rand(dev, 2, 5, 72, seed=i) for i in range(4))
  w, b = rand(dev, 2, 72, seed=5), rand(dev, 2, 72, seed=6)
  leaves = [t.clone().requires_grad_(True) for t in (x, w, b, res)]
  y, s = L.hip_rms_norm(*leaves, weight_offset=1.0)
  grads = torch.autograd.grad((y, s), leaves, (g, gs))

  def loss(x, w, b, res):
    y, s, *_ = rms64(x, res, w, b, 1e-6, 1.0)
    return float((y * g.double()).sum() + (s * gs.double()).sum())

  at = [t.double() for t in (x, w, b, res)]
  for i, grad in enumerate(grads):
    u = rand(dev, *grad.shape, seed=10 + i).double()
    step = 2.0**-16
    ahead, behind = ([*at[:i], at[i] + d * u, *at[i + 1:]] for d in (step, -step))
    slope = (loss(*ahead) - loss(*behind)) / (2 * step)
    assert abs(float((grad.double() * u).sum()) - slope) <= 1e-5 * float((grad.double() * u).abs().sum())


def test_rows_that_are_zero_or_not_finite(dev):
  x = rand(dev, 5, 640, seed=5)
  x[0] = 0
  x[1, 100], x[2, 3] = math.inf, math.nan
  y = ops.rms_norm(x)
  assert not y[0].any() and bool(y[2].isnan().all()) and bool(y[3:].isfinite().all()) and bool(y[1, 100].isnan())
  y, s = ops.rms_norm(-x, residual=x)
  assert not y[[0, 3, 4]].any() and not s[[0, 3, 4]].any() and bool(y[[1, 2]].isnan().all())
  q = ops.rms_norm_quant(x)
  assert bool((q.scales[2, :5] == 255).all()) and bool(q.dequantize()[[0, 3, 4]].isfinite().all())
  ds, _, _, _ = ops.rms_norm_backward(x, None, None, torch.ones_like(x))
  assert bool(ds[[0, 3, 4]].isfinite().all()) and bool(ds[2].isnan().all())


@pytest.mark.parametrize("xt,rt", TYPES)
@pytest.mark.parametrize("c", [64, 1001, 1536])
def test_strides_and_odd_addresses(dev, xt, rt, c):
  def apart(seed, t):
    return None if t is None else rand(dev, 3, 11, 2 * c + 3, seed=seed, dtype=t)[:, 1:, 1:1 + c]

  x, res, g, gs = apart(1, xt), apart(2, rt), apart(3, xt), apart(4, rt or xt)
  w = rand(dev, 3, c + 1, seed=5)[:, 1:]
  dense = lambda t: None if t is None else t.contiguous()
  want = both(ops.rms_norm(dense(x), dense(w), None, dense(res)), res)
  for call in (lambda *a: both(ops.rms_norm(*a), res), lambda *a: both(L.hip_rms_norm(*a), res)):
    for p, q in zip(call(x, dense(w), None, res), want):
      assert p is q or torch.equal(p, q)
  assert torch.equal(both(L.hip_rms_norm(x, w, None, res), res)[0], want[0])  # (vectors that are copied)
  s = x if res is None else apart(6, rt)
  narrow = s.dtype != xt
  for p, q in zip(ops.rms_norm_backward(s, dense(w), None, g, gs, narrow=narrow), ops.rms_norm_backward(dense(s), dense(w), None, dense(g), dense(gs), narrow=narrow)):
    assert p is q or torch.equal(p, q)
  turned = lambda t: None if t is None else t.transpose(0, 1)
  p, q = both(L.hip_rms_norm(turned(x), None, None, turned(res)), res), both(ops.rms_norm(turned(dense(x)).contiguous(), None, None, dense(turned(res))), res)
  assert torch.equal(p[0], q[0])
  # a residual laid out otherwise than x
  if res is not None:
    other = dense(turned(res)).transpose(0, 1)
    assert torch.equal(L.hip_rms_norm(x, None, None, other)[1], L.hip_rms_norm(x, None, None, res)[1])


def leaves_of(dev, xt, rt, wt=F32, shape=(2, 7, 264), per_batch=False):
  n, _, c = shape
  x, res = rand(dev, *shape, seed=1, dtype=xt), rand(dev, *shape, seed=2, dtype=rt)
  w, b = (rand(dev, *((n, c) if per_batch else (c,)), seed=i, dtype=wt) for i in (3, 4))
  return [t.requires_grad_(True) for t in (x, w, b, res)]


@pytest.mark.parametrize("xt,rt", [t for t in TYPES if t[1]])
@pytest.mark.parametrize("python", [False, True])
def test_autograd(dev, xt, rt, python):
  """Every subset of gradients, of y alone, of s alone, of both; by the native node and by the Python one."""
  leaves = leaves_of(dev, xt, rt)
  x, w, b, res = leaves
  g, gs = rand(dev, 2, 7, 264, seed=5, dtype=xt), rand(dev, 2, 7, 264, seed=6, dtype=rt)

  def call():
    return L.hip_rms_norm(torch.cat((x, x), -1)[..., :264].transpose(0, 1)[:, :, None] if python else x, w, b,
                          res.transpose(0, 1)[:, :, None] if python else res)

  def flat(t):
    return t[:, :, 0].transpose(0, 1) if python else t

  s = ops.rms_norm(x.detach(), w.detach(), b.detach(), res.detach())[1]
  narrow = xt != rt

  def want(g, gs):
    again = rt == BF16 and w.dtype == F32  # x and the residual are kept, in place of s
    ds, dx, dw, db = ops.rms_norm_backward(x.detach() if again else s, w.detach(), b.detach(), torch.zeros_like(x) if g is None else g, gs, narrow=narrow,
                                           residual=res.detach() if again else None)
    return (ds if dx is None else dx, dw, db, ds)

  for up in ((g, None), (None, gs), (g, gs)):
    y, t = (flat(o) for o in call())
    outs = [o for o, u in zip((y, t), up) if u is not None]
    got = torch.autograd.grad(outs, leaves, [u for u in up if u is not None])
    for name, p, q in zip(("dx", "dw", "db", "dres"), got, want(*up)):
      if python and name in ("dw", "db"):  # (rows in another order)
        assert (p.double() - q.double()).abs().max() <= 2.0**-7 * q.double().abs().max()
      else:
        assert torch.equal(p, q), name
  for i in range(4):
    y, _ = call()
    (one,) = torch.autograd.grad(flat(y), leaves[i], g)
    assert one.shape == leaves[i].shape
  y = L.hip_rms_norm(x, w, b)
  assert torch.equal(torch.autograd.grad(y, x, g)[0], ops.rms_norm_backward(x.detach(), w.detach(), b.detach(), g)[0])


def test_gradients_of_both_terms_are_apart(dev):
  """x and the residual have one gradient: what is accumulated into one's .grad does not reach the other's."""
  x, _, _, res = leaves_of(dev, BF16, BF16)
  y, s = L.hip_rms_norm(x, residual=res)
  (y.float().sum() + s.float().sum()).backward()
  keep = res.grad.clone()
  x.grad.zero_()
  assert torch.equal(res.grad, keep) and keep.any()


def test_outputs_changed_in_place(dev):
  """y may change; s, which the backward reads, is refused once it has."""
  x, w, b, res = leaves_of(dev, BF16, BF16)
  want = torch.autograd.grad(L.hip_rms_norm(x, w, b, res)[0].sum(), (x, w))
  y, s = L.hip_rms_norm(x, w, b, res)
  y += 1.0
  for p, q in zip(torch.autograd.grad(y.sum(), (x, w)), want):
    assert torch.equal(p, q)
  y, s = L.hip_rms_norm(x, w, b, res)
  s += 1.0
  if w.dtype == F32:  # (x and the residual are kept, in place of s)
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], want[0])
  y, s = L.hip_rms_norm(x, w.to(BF16), b.to(BF16), res)
  s += 1.0
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    torch.autograd.grad(y.sum(), x)


@pytest.mark.parametrize("rt", [BF16, F32])
def test_hooks_and_checkpoints(dev, rt):
  leaves = leaves_of(dev, BF16, rt)
  loss = lambda out: sum(o.float().square().sum() for o in out)
  native = lambda x, w, b, res: L.hip_rms_norm(x, w, b, res)
  python = lambda x, w, b, res: L.hip_rms_norm(x, torch.cat((w, w))[:264], torch.stack((b, b), 1)[:, 0], res)
  for call in (native, python):
    want = torch.autograd.grad(loss(call(*leaves)), leaves)
    with torch.autograd.graph.save_on_cpu():
      out = call(*leaves)
    for p, q in zip(torch.autograd.grad(loss(out), leaves), want):
      assert torch.equal(p, q)
    out = torch.utils.checkpoint.checkpoint(call, *leaves, use_reentrant=False)
    for p, q in zip(torch.autograd.grad(loss(out), leaves), want):
      assert torch.equal(p, q)
    for t in {rt, F32}:  # what is saved: s, of the residual's type, and w
      with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda u: u.to({BF16: F32, F32: BF16}[t]) if u.dtype == t else u):
        out = L.hip_rms_norm(*leaves)
      with pytest.raises(ValueError):
        torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])


def test_what_has_no_derivative_is_refused(dev):
  x, w, b, res = leaves_of(dev, BF16, BF16)
  y, s = L.hip_rms_norm(x, w, b, res)
  (dx,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
  with pytest.raises(NotImplementedError, match="second derivatives"):
    torch.autograd.grad(dx.float().square().sum() + x.float().sum(), x)
  w8 = L.quantize_weight(rand(dev, 8, 264, seed=7))
  with pytest.raises(NotImplementedError, match="no backward"):
    L.hip_rms_norm_linear_fp8(x, w, b, w8, residual=res)
  with pytest.raises(NotImplementedError, match="no backward"):
    L.hip_rms_norm_linear_fp8(x.detach(), None, None, w8, residual=res)
  x, w, b, res = (t.detach() for t in (x, w, b, res))
  with forward_ad.dual_level():
    dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
    for args in ((dual(x), w, b, res), (x, dual(w), b, res), (x, w, b, dual(res))):
      with pytest.raises(NotImplementedError, match="tangents"):
        L.hip_rms_norm(*args)
      with pytest.raises(NotImplementedError, match="tangents"):
        L.hip_rms_norm_linear_fp8(args[0], args[1], args[2], w8, residual=args[3])


def test_arguments_are_checked(dev):
  x, res, w = rand(dev, 2, 3, 64, seed=1, dtype=BF16), rand(dev, 2, 3, 64, seed=2, dtype=BF16), rand(dev, 64, seed=3)
  w8 = L.quantize_weight(rand(dev, 8, 64, seed=4))
  for call in (L.hip_rms_norm, lambda x, w=None, b=None, residual=None: L.hip_rms_norm_linear_fp8(x, w, b, w8, residual=residual)):
    for args in ((x, w, None, res[:, :2]), (x, w, None, res[0]), (x.float(), w, None, res), (x, w, None, res.half()), (x.half(), w), (x, w[:5]), (x, w.half()),
                 (x, w, w.to(BF16)), (x, w.expand(3, 64)), (torch.ones((), device=dev), None), (x, w, None, res.cpu()), (x.cpu(), w)):
      with pytest.raises(ValueError):
        call(*args)
  s = x.float()
  for args in ((s, w, None, x[:1]), (x, w, None, s), (s, w, None, s, x), (s, w, None, s, s[:1])):
    with pytest.raises(ValueError):
      ops.rms_norm_backward(*args)
  with pytest.raises(ValueError):
    ops.rms_norm_backward(s, w, None, s, narrow=True)
  with pytest.raises(ValueError):
    ops.rms_norm_backward(x, w, None, x, narrow=True)


@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 64), (3, 0)])
def test_nothing_to_compute(dev, shape):
  x, res = (torch.empty(shape, dtype=BF16, device=dev).requires_grad_(True) for _ in range(2))
  w = torch.ones(shape[-1], device=dev).requires_grad_(True)
  y, s = L.hip_rms_norm(x, w, None, res)
  assert y.shape == s.shape == x.shape
  dx, dw, dr = torch.autograd.grad((y, s), (x, w, res), (torch.ones_like(y), torch.ones_like(s)))
  assert dx.shape == dr.shape == x.shape and not dw.any()


@pytest.mark.parametrize("xt,rt", TYPES)
@pytest.mark.parametrize("m,c,n", [(1, 264, 130), (37, 512, 256), (3, 5120, 64)])
def test_norm_and_product(dev, xt, rt, m, c, n):
  x, w, v = rand(dev, 2, m, c, seed=1, dtype=xt), rand(dev, c, seed=2), rand(dev, n, seed=4)
  res = None if rt is None else rand(dev, 2, m, c, seed=3, dtype=rt)
  w8 = L.quantize_weight(rand(dev, n, c, seed=5, std=c**-0.5))
  for bias, out_bias in ((None, None), (w, v)):
    y, s = both(L.hip_rms_norm_linear_fp8(x, w, bias, w8, out_bias, res, weight_offset=1.0), res)
    q, t = both(ops.rms_norm_quant(x, w, bias, res, weight_offset=1.0), res)
    assert torch.equal(y, ops.matmul_fp8_block(q, w8, out_bias).view(2, m, n)) and (res is None or torch.equal(s, t))
    turned = lambda t: None if t is None else t.transpose(0, 1)[:, :, None]
    y2, s2 = both(L.hip_rms_norm_linear_fp8(turned(x), w, bias, w8, out_bias, turned(res), weight_offset=1.0), res)
    assert torch.equal(y2, turned(y)) and (res is None or torch.equal(s2, turned(s)))
  empty = x[:, :0]
  out = L.hip_rms_norm_linear_fp8(empty, w, None, w8, residual=None if res is None else res[:, :0])
  assert both(out, res)[0].shape == (2, 0, n)


def test_in_place_through_the_c_interface(dev, lib):
  """s over the residual and y over x."""
  import ctypes

  x, res, w = rand(dev, 9, 520, seed=1, dtype=BF16), rand(dev, 9, 520, seed=2, dtype=BF16), rand(dev, 520, seed=3)
  y, s = ops.rms_norm(x, w, None, res)
  p = lambda t: ctypes.c_void_p(t.data_ptr())
  st = (0, 520)
  rc = lib.mdattn_rms_norm(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), p(x), 0, p(res), 0, p(x), p(res), p(w), None, 1, 1, 9, 520, *st, *st, *st, *st,
                           0, 1e-6, 0.0)
  assert rc == 0 and torch.equal(x, y) and torch.equal(res, s)


def test_captured_and_on_another_stream(dev):
  leaves = leaves_of(dev, BF16, BF16, per_batch=True)
  g = rand(dev, 2, 7, 264, seed=5, dtype=BF16)

  def step():
    y, s = L.hip_rms_norm(*leaves, weight_offset=1.0)
    return (y.detach(), s.detach(), *torch.autograd.grad((y, s), leaves, (g, g)))

  want = [t.clone() for t in step()]
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    for p, q in zip(step(), want):
      assert torch.equal(p, q)
  torch.cuda.current_stream().wait_stream(side)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = step()
  for rep in range(3):
    for t in captured:
      t.fill_(rep + 0.5)
    for p, q in zip(step(), want):
      assert torch.equal(p, q)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for p, q in zip(captured, want):
      assert torch.equal(p, q)


def test_many_rows(dev):
  """Rows whose offsets pass 32 bits."""
  n = 1_100_000
  x = torch.empty((n, 2048), dtype=BF16, device=dev)
  x[:] = rand(dev, 1, 2048, seed=1, dtype=BF16)
  some = rand(dev, 50, 2048, seed=2, dtype=BF16)
  x[-50:] = some
  y, s = L.hip_rms_norm(x, residual=x)
  want, ws = L.hip_rms_norm(some, residual=some)
  assert torch.equal(y[-50:], want) and torch.equal(s[-50:], ws) and torch.equal(y[0], y[n // 2])
