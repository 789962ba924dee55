"""Attention over packed sequences as programs use it: long caches, pieces, layouts, autograd's modes, graphs, streams, and what is refused."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from maxdiffusion_amd import attention_op as A
from maxdiffusion_amd import ops
from packed_reference import assert_within, attention, starts
from test_gpu_packed import BF16, ints, make

pytestmark = pytest.mark.gpu


def check_forward(dev, q, k, v, qo, ko, kl=None, causal=True, **hints):
  want = attention(q, k, v, qo, ko, kl, causal)
  out, lse = ops.flash_attention_packed(q, k, v, ints(dev, qo), ints(dev, ko), k_lengths=None if kl is None else ints(dev, kl), causal=causal, return_lse=True,
                                        **hints)
  assert_within(out, want["out"], want["out_err"], f"out {hints}")
  none = want["lse"] == -math.inf
  assert torch.equal(lse == -math.inf, none) and not out.transpose(0, 1)[none].any()
  if not none.all():
    assert (lse - want["lse"])[~none].abs().max() <= 1e-4
  return out, lse


# ------------------------------------------------------------------------------------------------ few rows against many keys
@pytest.mark.parametrize("h,hkv,d", [(8, 2, 128), (4, 4, 64), (5, 1, 80)])
@pytest.mark.parametrize("m,n", [([1], [20000]), ([1, 1, 1, 1], [5000, 1, 0, 777]), ([3, 0, 7], [4097, 300, 2049]), ([200], [3000]), ([40, 100], [6000, 10])])
def test_keys_in_pieces(dev, m, n, h, hkv, d):
  qo, ko = starts(m), starts(n)
  q, k, v, _ = make(dev, qo[-1], ko[-1], h, hkv, d, seed=3)
  for causal in (True, False):
    print(m, n, h, hkv, d, causal, flush=True)
    check_forward(dev, q, k, v, qo, ko, causal=causal)
    check_forward(dev, q, k, v, qo, ko, causal=causal, max_q=max(m), max_k=max(n))
    check_forward(dev, q, k, v, qo, ko, causal=causal, max_q=1, max_k=700)  # (the last piece takes the rest)


@pytest.mark.parametrize("room,filled", [(300, [0, 1, 300, 299, 32]), (4096, [4096, 1, 1500, 0]), (64, [64] * 200)])
def test_tokens_against_a_cache_with_room(dev, room, filled):
  """What stands behind the filled part of a cache has no say, NaNs included."""
  b = len(filled)
  q, k, v, _ = make(dev, b, b * room, 8, 2, 128, seed=4)
  for i, n in enumerate(filled):
    k[i * room + n:(i + 1) * room] = math.nan
    v[i * room + n:(i + 1) * room] = math.nan
  qo, ko = list(range(b + 1)), [i * room for i in range(b + 1)]
  out, _ = check_forward(dev, q, k, v, qo, ko, filled, max_q=1, max_k=max(filled))
  with torch.no_grad():
    for hints in ({}, dict(max_q=1, max_k=room)):
      got = A.hip_flash_packed(q, k, v, ints(dev, qo), ints(dev, ko), k_lengths=ints(dev, filled), **hints)
      assert_within(got, *(attention(q, k, v, qo, ko, filled)[x] for x in ("out", "out_err")), "hip_flash_packed")
  # lengths past a sequence's room, and negative ones, are brought into it
  clipped = [room if n == room else n for n in filled]
  k2, v2 = k.nan_to_num(1.0), v.nan_to_num(1.0)
  wild = [n + 1000 if n == room else -5 if n == 0 else n for n in filled]
  a = ops.flash_attention_packed(q, k2, v2, ints(dev, qo), ints(dev, ko), k_lengths=ints(dev, wild))
  b = ops.flash_attention_packed(q, k2, v2, ints(dev, qo), ints(dev, ko), k_lengths=ints(dev, clipped))
  assert torch.equal(a, b)


def test_a_cache_whose_offsets_pass_32_bits(dev):
  rows, n = 2_200_000, 3000  # 8 heads of 128: element 2^31 is in row 2,097,152
  k, v = (torch.empty((rows, 8, 128), dtype=BF16, device=dev) for _ in range(2))
  q, ks, vs, _ = make(dev, 2, n, 16, 8, 128, seed=5)
  k[-n:], v[-n:] = ks, vs
  lens = [1000, 2000]
  want = attention(q, ks, vs, [0, 1, 2], starts(lens))
  for hints in ({}, dict(max_q=1, max_k=2000)):
    out = ops.flash_attention_packed(q, k, v, ints(dev, [0, 1, 2]), ints(dev, starts(lens, rows - n)), **hints)
    assert_within(out, want["out"], want["out_err"], "out")


def test_more_heads_than_a_die_has_and_large_groups(dev):
  for h, hkv in ((64, 2), (40, 1), (36, 12)):
    q, k, v, g = make(dev, 75, 75, h, hkv, 64, seed=6)
    want = attention(q, k, v, [0, 70, 75], [0, 70, 75], dout=g, rest=False)
    out, lse = check_forward(dev, q, k, v, [0, 70, 75], [0, 70, 75])
    for name, t in zip(("dq", "dk", "dv"), ops.flash_attention_packed_backward(q, k, v, out, g, lse, ints(dev, [0, 70, 75]))):
      assert_within(t, want[name], want[name + "_err"], name)


# ------------------------------------------------------------------------------------------------ the backward pass
@pytest.mark.parametrize("h,hkv,d", [(8, 2, 128), (2, 2, 64), (6, 1, 72)])
@pytest.mark.parametrize("m,n", [([1500, 700, 1], None), ([2000], [130]), ([129], [3000])])
def test_rows_in_pieces(dev, m, n, h, hkv, d):
  qo, ko = starts(m), starts(n or m)
  q, k, v, g = make(dev, qo[-1], ko[-1], h, hkv, d, seed=7, lean=0.5)
  for causal in (True, False):
    want = attention(q, k, v, qo, ko, causal=causal, dout=g, rest=False)
    out, lse = ops.flash_attention_packed(q, k, v, ints(dev, qo), ints(dev, ko), causal=causal, return_lse=True)
    for hints in ({}, dict(max_q=max(m), max_k=max(n or m)), dict(max_q=200, max_k=10)):
      got = [ops.flash_attention_packed_backward(q, k, v, out, g, lse, ints(dev, qo), ints(dev, ko), causal=causal, **hints) for _ in range(2)]
      for name, t, again in zip(("dq", "dk", "dv"), *got):
        assert_within(t, want[name], want[name + "_err"], f"{name} {causal} {hints}")
        assert torch.equal(t, again)  # no sum depends on which workgroup was first


def test_gradients_against_differences(dev):
  """The loss of packed attention in 64 bits, moved along random directions: the kernels' gradients predict the change."""
  qo = [0, 50, 51, 120]
  q, k, v, g = make(dev, 120, 120, 4, 2, 64, seed=8, lean=0.5)
  leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
  grads = torch.autograd.grad(A.hip_flash_packed(*leaves, ints(dev, qo)), leaves, g)
  bounds = attention(q, k, v, qo, qo, dout=g)
  loss = lambda *t: float((attention(*t, qo, qo)["out"] * g.double()).sum())
  step = 2.0**-20
  for i, (name, grad) in enumerate(zip(("dq", "dk", "dv"), grads)):
    u = torch.randn(q.shape if i == 0 else k.shape, generator=torch.Generator(device=dev).manual_seed(i), device=dev, dtype=torch.float64)
    at = [t.double() for t in (q, k, v)]
    ahead, behind = ([*at[:i], at[i] + s * u, *at[i + 1:]] for s in (step, -step))
    slope = (loss(*ahead) - loss(*behind)) / (2 * step)
    room = float((1.02 * bounds[name + "_err"] * u.abs()).sum()) + 1e-4 * abs(slope)
    assert abs(float((grad.double() * u).sum()) - slope) <= room


# ------------------------------------------------------------------------------------------------ rows of no sequence, values that are not finite
@pytest.mark.parametrize("m", [[40, 3, 100], [], [0, 0]])
def test_rows_of_no_sequence_are_zero(dev, m):
  front, back = 37, 150
  qo = starts(m, front)
  t = qo[-1] + back
  q, k, v, g = make(dev, t, t, 4, 2, 128, seed=9)
  inside = torch.zeros(t, dtype=torch.bool, device=dev)
  inside[front:qo[-1]] = True
  want = attention(q, k, v, qo, qo, dout=g, rest=False)
  for x in (q, k, v, g):
    x[~inside] = math.nan
  for hints in ({}, dict(max_q=1, max_k=100)):
    out, lse = ops.flash_attention_packed(q, k, v, ints(dev, qo), return_lse=True, **hints)
    assert not out[~inside].any() and bool((lse[:, ~inside] == -math.inf).all())
    got = ops.flash_attention_packed_backward(q, k, v, out, g, lse, ints(dev, qo), **hints)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *got)):
      assert not x[~inside].any(), name
      if m and sum(m):
        assert_within(x, want[name], want[name + "_err"], name)


def test_a_split_call_leaves_rows_of_no_sequence_zero(dev):
  q, k, v, _ = make(dev, 5, 9000, 4, 1, 128, seed=10)
  q[0] = q[4] = math.nan
  out, lse = ops.flash_attention_packed(q, k, v, ints(dev, [1, 2, 4]), ints(dev, [10, 4000, 8990]), max_q=2, max_k=5000, return_lse=True)
  want = attention(q, k, v, [1, 2, 4], [10, 4000, 8990])
  assert not out[[0, 4]].any() and bool((lse[:, [0, 4]] == -math.inf).all())
  assert_within(out, want["out"], want["out_err"], "out")


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_sequence_that_is_not_finite_spoils_no_other(dev, bad):
  qo = [0, 45, 100, 163]
  q, k, v, g = make(dev, 163, 163, 4, 2, 128, seed=11)
  want = attention(q, k, v, qo, qo, dout=g, rest=False)
  spoilt = slice(45, 100)
  for x in (q, k, v, g):
    x[spoilt] = bad
  out, lse = ops.flash_attention_packed(q, k, v, ints(dev, qo), return_lse=True)
  got = ops.flash_attention_packed_backward(q, k, v, out, g, lse, ints(dev, qo))
  assert not torch.isfinite(out[spoilt]).any()
  keep = torch.ones(163, dtype=torch.bool, device=dev)
  keep[spoilt] = False
  for name, x in zip(("out", "dq", "dk", "dv"), (out, *got)):
    assert_within(x[keep], want[name][keep], want[name + "_err"][keep], name)


@pytest.mark.parametrize("order", ["up", "down", "spike"])
def test_logits_of_every_size(dev, order):
  """Logits that climb by hundreds, fall by hundreds, or jump to thousands: the reference point of the softmax moves."""
  n, d = 300, 128
  q, k, v, g = make(dev, n, n, 2, 1, d, seed=12, lean=0.0)
  ramp = torch.linspace(-300, 300, n, device=dev)
  size = {"up": ramp, "down": -ramp, "spike": torch.where(torch.arange(n, device=dev) % 97 == 50, 3000.0, 0.0)}[order]
  q[:, :, 0], k[:, :, 0] = d**0.5, size[:, None].to(BF16)
  want = attention(q, k, v, [0, n], [0, n])
  out, lse = ops.flash_attention_packed(q, k, v, ints(dev, [0, n]), return_lse=True)
  # A logit is a sum over 128 channels that passes through the accumulators of eight matrix instructions in turn, each rounded to the last place of the
  # sum (2^-23 of it at most); its factor, the reference point and the sum of the logarithm are three roundings more.  The probabilities are
  # off by as much of themselves.
  scale = want["lse"].abs().max() * 11 * 2.0**-23
  assert_within(out, want["out"], want["out_err"] + 2 * scale * attention(q, k, v.abs(), [0, n], [0, n])["out"], "out")
  assert (lse - want["lse"]).abs().max() <= scale + 1e-4


def test_scales(dev):
  q, k, v, g = make(dev, 90, 90, 2, 2, 64, seed=13)
  for scale in (1e-20, 0.01, 1.0, math.log(2.0)):
    want = attention(q, k, v, [0, 90], [0, 90], scale=scale, dout=g, rest=False)
    out, lse = ops.flash_attention_packed(q, k, v, ints(dev, [0, 90]), scale=scale, return_lse=True)
    assert_within(out, want["out"], want["out_err"], f"out {scale}")
    if scale > 1e-3:
      for name, x in zip(("dq", "dk", "dv"), ops.flash_attention_packed_backward(q, k, v, out, g, lse, ints(dev, [0, 90]), scale=scale)):
        assert_within(x, want[name], want[name + "_err"], f"{name} {scale}")


def test_offsets_that_decrease_or_point_outside_touch_nothing_else(dev):
  """Brought into the tensors: where the offsets increase, the sequences that lie inside keep their results; where they decrease, nothing is said."""
  q, k, v, g = make(dev, 200, 200, 4, 2, 64, seed=14)
  good = ops.flash_attention_packed(q, k, v, ints(dev, [0, 64]))[:64]
  for o in ([0, 64, 10**9], [-(2**31), 64], [0, 64, 2**31 - 1, -7], [0, 64, 30, 200]):
    out, lse = ops.flash_attention_packed(q, k, v, ints(dev, o), return_lse=True)
    if o == sorted(o):
      assert torch.equal(out[:64], good)
    ops.flash_attention_packed_backward(q, k, v, out, g, lse, ints(dev, o))
  torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ layouts
def test_layouts(dev):
  h, hkv, d, t = 6, 2, 64, 150
  o = ints(dev, [0, 100, 150])
  q, k, v, g = make(dev, t, t, h, hkv, d, seed=15)
  want = A.hip_flash_packed(q, k, v, o)
  fused = torch.cat((q.flatten(1), k.flatten(1), v.flatten(1)), 1)
  views = [x.unflatten(1, (-1, d)) for x in fused.split([h * d, hkv * d, hkv * d], 1)]
  by_head = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
  odd = [torch.cat((x.new_zeros(1), x.flatten()))[1:].view(x.shape) for x in (q, k, v)]  # at an address that is 2 mod 16
  ragged = [torch.cat((x, x[..., :4]), 2)[..., :d] for x in (q, k, v)]                      # strides that 8 does not divide
  back = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]                # the head dim is not the last in memory
  for form in (views, by_head, odd, ragged, back):
    assert torch.equal(A.hip_flash_packed(*form, o), want)
    leaves = [x.detach().requires_grad_(True) for x in form]
    y = A.hip_flash_packed(*leaves, o)
    assert torch.equal(y, want) and y.is_contiguous()
    grads = torch.autograd.grad(y, leaves, g)
    dense = [x.clone().requires_grad_(True) for x in (q, k, v)]
    for a, b in zip(grads, torch.autograd.grad(A.hip_flash_packed(*dense, o), dense, g)):
      assert torch.equal(a, b)
  # heads that are one tensor, read with stride 0
  one = k[:, :1]
  assert torch.equal(A.hip_flash_packed(q, one.expand(t, hkv, d), v, o), A.hip_flash_packed(q, one.repeat(1, hkv, 1), v, o))


def test_gradients_that_arrive_in_other_forms(dev):
  q, k, v, g = make(dev, 70, 70, 4, 2, 64, seed=16)
  o = ints(dev, [0, 30, 70])

  def grads(leaves, y, dout):
    return torch.autograd.grad(y, leaves, dout)

  def run(dout):
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    return grads(leaves, A.hip_flash_packed(*leaves, o), dout)

  row = g[:1, :1, :]
  for odd, plain in ((row.expand_as(g), row.repeat(70, 4, 1)), (g.transpose(0, 1).contiguous().transpose(0, 1), g),
                     (torch.cat((g.new_zeros(1), g.flatten()))[1:].view(g.shape), g)):
    for a, b in zip(run(odd), run(plain)):
      assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ autograd's modes
def test_which_gradients_are_asked_for(dev):
  q, k, v, g = make(dev, 64, 64, 4, 2, 128, seed=17)
  o = ints(dev, [0, 64])
  leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
  every = torch.autograd.grad(A.hip_flash_packed(*leaves, o), leaves, g)
  for i in range(3):
    some = [x.clone().requires_grad_(j == i) for j, x in enumerate((q, k, v))]
    assert torch.equal(torch.autograd.grad(A.hip_flash_packed(*some, o), some[i], g)[0], every[i])
  shared = q[:, :2].clone().requires_grad_(True)  # one tensor as k and v
  (d,) = torch.autograd.grad(A.hip_flash_packed(q, shared, shared, o), shared, g)
  a, b = (shared.detach().clone().requires_grad_(True) for _ in range(2))
  da, db = torch.autograd.grad(A.hip_flash_packed(q, a, b, o), (a, b), g)
  assert torch.equal(d, da + db)


def test_hooks_checkpoints_and_changes_in_place(dev):
  q, k, v, g = make(dev, 64, 64, 4, 2, 128, seed=18)
  o = ints(dev, [0, 10, 64])
  leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
  want = torch.autograd.grad(A.hip_flash_packed(*leaves, o), leaves, g)
  with torch.autograd.graph.save_on_cpu():
    y = A.hip_flash_packed(*leaves, o)
  for a, b in zip(torch.autograd.grad(y, leaves, g), want):
    assert torch.equal(a, b)
  y = torch.utils.checkpoint.checkpoint(lambda *t: A.hip_flash_packed(*t, o), *leaves, use_reentrant=False)
  for a, b in zip(torch.autograd.grad(y, leaves, g), want):
    assert torch.equal(a, b)
  with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.float() if t.dtype == BF16 else t):
    y = A.hip_flash_packed(*leaves, o)
    with pytest.raises(ValueError):
      torch.autograd.grad(y, leaves, g)
  y = A.hip_flash_packed(*leaves, o)
  o.add_(0)
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    torch.autograd.grad(y, leaves, g)
  y = A.hip_flash_packed(*leaves, o)
  y.mul_(1)  # the output, which the backward reads
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    torch.autograd.grad(y, leaves, g)


def test_what_has_no_derivative_is_refused(dev):
  q, k, v, g = make(dev, 64, 64, 4, 2, 128, seed=19)
  o = ints(dev, [0, 64])
  q.requires_grad_(True)
  with pytest.raises(NotImplementedError, match="k_lengths"):
    A.hip_flash_packed(q, k, v, o, k_lengths=ints(dev, [64]))
  (dq,) = torch.autograd.grad(A.hip_flash_packed(q, k, v, o).float().square().sum(), q, create_graph=True)
  with pytest.raises((NotImplementedError, RuntimeError)):
    torch.autograd.grad(dq.float().sum(), q)
  with forward_ad.dual_level():
    dual = forward_ad.make_dual(q.detach(), torch.ones_like(q))
    with pytest.raises(NotImplementedError, match="tangents"):
      A.hip_flash_packed(dual, k, v, o)


def test_arguments_are_checked(dev):
  q, k, v, g = make(dev, 64, 64, 4, 2, 128, seed=20)
  o = ints(dev, [0, 64])
  for call in (A.hip_flash_packed, ops.flash_attention_packed):
    for args in ((q.float(), k, v, o), (q[0], k, v, o), (q, k[:, :1], v, o), (q[:, :3], k, v, o), (q, k[..., :64], v[..., :64], o), (q, k, v[:63], o),
                 (q[..., :20], k[..., :20], v[..., :20], o), (q, k, v, o.long()), (q, k, v, o[None]), (q, k, v, o, ints(dev, [0, 1, 64])),
                 (q, k, v, o[:0]), (torch.cat((q, q), 2), torch.cat((k, k), 2), torch.cat((v, v), 2), o), (q.cpu(), k, v, o), (q, k, v, o.cpu())):
      with pytest.raises(ValueError):
        call(*args)
    with pytest.raises(ValueError):
      call(q, k, v, o, k_lengths=ints(dev, [1, 2]))
  out, lse = ops.flash_attention_packed(q, k, v, o, return_lse=True)
  for bad in (dict(out=out.float()), dict(dout=g[:5]), dict(lse=lse[:, :5]), dict(lse=lse.double())):
    with pytest.raises(ValueError):
      ops.flash_attention_packed_backward(**{**dict(q=q, k=k, v=v, out=out, dout=g, lse=lse, q_offsets=o), **bad})


def test_nothing_to_compute(dev):
  q, k, v, g = make(dev, 5, 7, 4, 2, 128, seed=21)
  none = ints(dev, [0, 0])
  assert A.hip_flash_packed(q[:0], k, v, none, ints(dev, [0, 7])).shape == (0, 4, 128)
  assert not A.hip_flash_packed(q, k[:0], v[:0], ints(dev, [0, 5]), none).any()
  assert not A.hip_flash_packed(q, k, v, ints(dev, [0]), ints(dev, [0])).any()
  for a, b in ((0, 7), (5, 0), (0, 0)):
    leaves = [x.clone().requires_grad_(True) for x in (q[:a], k[:b], v[:b])]
    y = A.hip_flash_packed(*leaves, ints(dev, [0, a]), ints(dev, [0, b]))
    for t, x in zip(torch.autograd.grad(y, leaves, g[:a]), leaves):
      assert t.shape == x.shape and not t.any()


# ------------------------------------------------------------------------------------------------ graphs and streams
def test_a_captured_call_follows_the_offsets(dev):
  """One graph, replayed on sequences of other lengths; single tokens against a cache that grows; a training pass."""
  q, k, v, g = make(dev, 300, 300, 8, 2, 128, seed=22)
  o, kl = ints(dev, [0, 100, 300]), ints(dev, [5, 60])
  tq = q[:2]

  def step():
    out, lse = ops.flash_attention_packed(q, k, v, o, return_lse=True, max_q=300, max_k=300)
    return (out, lse, *ops.flash_attention_packed_backward(q, k, v, out, g, lse, o, max_q=300, max_k=300),
            ops.flash_attention_packed(tq, k, v, ints_one, o, k_lengths=kl, max_q=1, max_k=3000))

  ints_one = ints(dev, [0, 1, 2])
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step()
  torch.cuda.current_stream().wait_stream(side)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = step()
  for rep, (lengths, filled) in enumerate([([0, 100, 300], [5, 60]), ([0, 1, 300], [1, 299]), ([20, 20, 250], [0, 7]), ([0, 100, 300], [5, 60])]):
    o.copy_(ints(dev, lengths))
    kl.copy_(ints(dev, filled))
    want = [t.clone() for t in step()]
    for t in captured:
      t.fill_(rep + 0.25)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(captured, want)):
      assert torch.equal(a, b), (rep, i)


def test_a_captured_training_step(dev):
  """Forward and backward through autograd in one graph, beside eager passes of other leaves."""
  q, k, v, g = make(dev, 200, 200, 4, 2, 64, seed=23)
  o = ints(dev, [0, 150, 200])
  leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]

  def step():
    return torch.autograd.grad(A.hip_flash_packed(*leaves, o), leaves, g)

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    want = [t.clone() for t in step()]
  torch.cuda.current_stream().wait_stream(side)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    captured = step()
  for rep in range(3):
    for t in captured:
      t.fill_(rep + 0.5)
    other = [x.clone().requires_grad_(True) for x in (q, k, v)]
    eager = torch.autograd.grad(A.hip_flash_packed(*other, o), other, g)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(captured, want, eager):
      assert torch.equal(a, b) and torch.equal(c, b)


def test_two_streams_at_once(dev):
  """Calls that need workspaces, on two streams: each has its own."""
  o, ko = ints(dev, [0, 1]), ints(dev, [0, 30000])
  sets = [make(dev, 1, 30000, 8, 2, 128, seed=s) for s in (24, 25)]
  want = [ops.flash_attention_packed(q, k, v, o, ko) for q, k, v, _ in sets]
  streams = [torch.cuda.Stream() for _ in sets]
  for s in streams:
    s.wait_stream(torch.cuda.current_stream())
  got = [[] for _ in sets]
  for _ in range(20):
    for i, (q, k, v, _) in enumerate(sets):
      with torch.cuda.stream(streams[i]):
        got[i].append(ops.flash_attention_packed(q, k, v, o, ko))
  torch.cuda.synchronize()
  for g, w in zip(got, want):
    assert all(torch.equal(t, w) for t in g)


def test_gradients_of_rows_with_one_heavy_key(dev):
  """Short sequences whose first key has most of the weight: dS is far smaller than dP and delta there, and delta from the rounded out alone would be
  off by as much.  The autograd node keeps what the rounding left."""
  m = [3] * 40 + [2] * 40 + [8] * 20
  o = starts(m)
  off = []
  for h, hkv, d in ((8, 2, 128), (4, 4, 64), (6, 2, 72)):
    q, k, v, g = make(dev, o[-1], o[-1], h, hkv, d, seed=d, lean=0.0)
    k[[a for a in o[:-1]]] += (q[[a + 1 for a in o[:-1]]].view(-1, hkv, h // hkv, d).float().mean(2) * 0.5).to(BF16)
    want = attention(q, k, v, o, o, dout=g)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    for name, t in zip(("dq", "dk", "dv"), torch.autograd.grad(A.hip_flash_packed(*leaves, ints(dev, o)), leaves, g)):
      assert_within(t, want[name], want[name + "_err"], f"{name} {h} {d}")
      off.append(float((t.double() - want[name]).norm() / want[name].norm()))
  # dS and the result are rounded, each by 2^-8 of an element at most and less than 0.43 of that in the root mean square; without the rest 6 to 8e-3
  assert max(off) < 2.0**-8
