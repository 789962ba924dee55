"""Packed attention in every form that the plan knows, each test saying which form it runs: waves that share keys, orders of the tiles, walks in pieces;
and calls whose sequences have room for more keys than they hold, with fewer queries than keys, and with more."""
import ctypes
import math

import pytest
import torch

from maxdiffusion_amd import _lib
from maxdiffusion_amd import attention_op as A
from maxdiffusion_amd import ops
from packed_reference import U, assert_within, attention, starts
from test_gpu_packed import BF16, ints, make
from test_packed_plans import Plan

pytestmark = pytest.mark.gpu


def plans(lib, q, k, sequences, causal, hints):
  """(forward, backward) of the call."""
  p = _lib.Packed(0x1000, 0x1000, None, sequences, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2], int(causal), hints.get("max_q", 0), hints.get("max_k", 0))
  fwd, bwd = Plan(), Plan()
  assert lib.mdattn_host_packed_fwd_plan(ctypes.byref(p), ctypes.byref(fwd)) == lib.mdattn_host_packed_bwd_plan(ctypes.byref(p), ctypes.byref(bwd)) == _lib.E_OK
  return fwd, bwd


# ------------------------------------------------------------------------------------------------ forward and backward
LENGTHS = [1, 33, 0, 97, 300, 2, 513, 130, 64]
# sequences without rows behind the others, heads, heads of k and v, hints; the forward's waves and orders (causal, not), the backward's orders and
# whether its walks are cut (where that does not go by the head dim)
FORMS = {
    "four": (0, 4, 2, dict(max_q=1, max_k=1), 4, (0, 0), (0, 0), False),
    "four, the backward's walks cut": (0, 4, 2, {}, 4, (0, 0), (0, 0), True),
    "two, more sequences than are sorted": (69, 4, 2, {}, 2, (0, 0), (0, 0), True),
    "two, sorted where causal": (20, 4, 4, {}, 2, (1, 0), (0, 0), False),
    "one, as they come": (0, 4, 2, dict(max_k=1), 1, (0, 0), (0, 0), True),
    "one, sorted, the backward too": (40, 8, 8, {}, 1, (1, 2), (1, 2), False),
    "one, sorted, the backward too, its walks cut": (40, 64, 8, {}, 1, (1, 2), (1, 2), True),
}


@pytest.mark.parametrize("d", [64, 40, 80, 128, 104])
@pytest.mark.parametrize("form", FORMS)
def test_forms(dev, lib, form, d):
  empty, h, hkv, hints, waves, fwd_orders, bwd_orders, cut = FORMS[form]
  o = starts(LENGTHS + [0] * empty)
  q, k, v, g = make(dev, o[-1], o[-1], h, hkv, d, seed=len(form), lean=0.5)
  offsets = ints(dev, o)
  for i, causal in enumerate((True, False)):
    print(form, d, causal, flush=True)
    fwd, bwd = plans(lib, q, k, len(o) - 1, causal, hints)
    assert (fwd.waves, fwd.order, fwd.pieces, bwd.order, bwd.pieces > 1) == (waves, fwd_orders[i], 1, bwd_orders[i], cut)
    want = attention(q, k, v, o, o, causal=causal, dout=g)
    out, lse, rest = ops.flash_attention_packed(q, k, v, offsets, causal=causal, return_lse=True, return_rest=True, **hints)
    assert_within(out, want["out"], want["out_err"], f"out {form} {d} {causal}")
    assert (lse - want["lse"]).abs().max() <= 1e-4  # f32 logits up to some 20
    for name, t in zip(("dq", "dk", "dv"), ops.flash_attention_packed_backward(q, k, v, out, g, lse, offsets, rest=rest, causal=causal, **hints)):
      assert_within(t, want[name], want[name + "_err"], f"{name} {form} {d} {causal}")


# ------------------------------------------------------------------------------------------------ fewer queries than keys, and more, in caches with room
QUERIES = [5, 1, 40, 0, 64, 3, 130]
# room of each, filled, sequences without rows behind the others, heads of k and v, hints; waves, orders, whether the keys are cut
CACHES = {
    "four": (320, [77, 300, 20, 50, 64, 0, 200], 0, 1, dict(max_q=1, max_k=1), 4, (0, 0), False),
    "four, keys cut": (1500, [700, 1500, 20, 50, 64, 0, 901], 0, 1, dict(max_q=1, max_k=1500), 4, (0, 0), True),
    "two": (320, [77, 300, 20, 50, 64, 0, 200], 60, 2, {}, 2, (0, 0), False),
    "two, sorted where causal": (320, [77, 300, 20, 50, 64, 0, 200], 23, 5, {}, 2, (1, 0), False),
    "one": (320, [77, 300, 20, 50, 64, 0, 200], 0, 1, dict(max_k=1), 1, (0, 0), False),
    "one, sorted": (320, [77, 300, 20, 50, 64, 0, 200], 40, 8, dict(max_k=320), 1, (1, 2), False),
}


@pytest.mark.parametrize("d", [64, 40, 80, 128])
@pytest.mark.parametrize("form", CACHES)
def test_queries_against_caches_with_room(dev, lib, form, d):
  """Several queries against keys of which they are the last, against more and against fewer; what stands behind the filled part has no say."""
  room, filled, empty, hkv, hints, waves, orders, cut = CACHES[form]
  filled = filled + [0] * empty
  qo, ko = starts(QUERIES + [0] * empty), [min(i, len(QUERIES)) * room for i in range(len(QUERIES) + empty + 1)]
  q, k, v, _ = make(dev, qo[-1], ko[-1], 2 * hkv, hkv, d, seed=len(form))
  for i, n in enumerate(filled[:len(QUERIES)]):
    k[i * room + n:(i + 1) * room] = math.nan
    v[i * room + n:(i + 1) * room] = math.nan
  for i, causal in enumerate((True, False)):
    print(form, d, causal, flush=True)
    fwd, _ = plans(lib, q, k, len(filled), causal, hints)
    assert (fwd.waves, fwd.order, fwd.pieces > 1) == (waves, orders[i], cut)
    want = attention(q, k, v, qo, ko, filled, causal)
    out, lse = ops.flash_attention_packed(q, k, v, ints(dev, qo), ints(dev, ko), k_lengths=ints(dev, filled), causal=causal, return_lse=True, **hints)
    assert_within(out, want["out"], want["out_err"], f"out {form} {d} {causal}")
    none = want["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, none) and not out.transpose(0, 1)[none].any()
    assert (lse - want["lse"])[~none].abs().max() <= 1e-4
    with torch.no_grad():
      assert torch.equal(A.hip_flash_packed(q, k, v, ints(dev, qo), ints(dev, ko), k_lengths=ints(dev, filled), causal=causal, **hints), out)


# ------------------------------------------------------------------------------------------------ what the join of pieces leaves for the backward pass
PIECES = [([1], [5000]), ([3], [700]), ([7, 1, 3], [2049, 700, 5000]), ([2, 0, 4], [600, 900, 1])]


def spoil(like):
  """Blocks of `like`'s size that the next allocations get, full of NaN."""
  torch.cuda.synchronize()
  blocks = [torch.full_like(like, math.nan) for _ in range(8)]
  torch.cuda.synchronize()
  del blocks


@pytest.mark.parametrize("h,hkv,d", [(8, 2, 128), (4, 4, 64), (3, 1, 80), (4, 2, 40)])
@pytest.mark.parametrize("m,n", PIECES)
def test_rest_of_keys_in_pieces(dev, lib, m, n, h, hkv, d):
  """Queries of zeros: every probability is one, the sums are exact but for their f32 rounding, and out and rest together are the mean of the keys seen."""
  qo, ko = starts(m), starts(n)
  q, k, v, _ = make(dev, qo[-1], ko[-1], h, hkv, d, seed=len(n))
  q.zero_()
  hints = dict(max_q=max(m), max_k=max(n))
  for causal in (True, False):
    assert plans(lib, q, k, len(m), causal, hints)[0].pieces > 1
    want = attention(q, k, v, qo, ko, causal=causal)["out"]
    spoil(q)
    out, rest = ops.flash_attention_packed(q, k, v, ints(dev, qo), ints(dev, ko), causal=causal, return_rest=True, **hints)
    # a sum of n terms: 2 sqrt(n) roundings of 2^-24 of the values' size, below 8 in bf16 randn; of rest its own rounding, 2^-8 of 2^-8 of out
    room = U * U * want.abs() + (2 * math.sqrt(max(n)) + 8) * 2.0**-24 * 8
    got = out.double() + rest.double()
    assert bool(((got - want).abs() <= room).all()), float(((got - want).abs() - room).max())
    assert bool((rest.double().abs() <= 1.01 * U * out.double().abs()).all()) and bool(rest.any())


@pytest.mark.parametrize("h,hkv,d", [(8, 2, 128), (4, 4, 64), (3, 1, 80), (4, 2, 40)])
@pytest.mark.parametrize("m,n", PIECES)
def test_gradients_where_the_forward_cuts_its_keys(dev, lib, m, n, h, hkv, d):
  qo, ko = starts(m), starts(n)
  q, k, v, g = make(dev, qo[-1], ko[-1], h, hkv, d, seed=len(n) + 1, lean=0.5)
  hints = dict(max_q=max(m), max_k=max(n))
  for causal in (True, False):
    print(m, n, h, hkv, d, causal, flush=True)
    assert plans(lib, q, k, len(m), causal, hints)[0].pieces > 1
    want = attention(q, k, v, qo, ko, causal=causal, dout=g)
    spoil(q)
    out, lse, rest = ops.flash_attention_packed(q, k, v, ints(dev, qo), ints(dev, ko), causal=causal, return_lse=True, return_rest=True, **hints)
    got = ops.flash_attention_packed_backward(q, k, v, out, g, lse, ints(dev, qo), ints(dev, ko), rest=rest, causal=causal, **hints)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    spoil(q)
    y = A.hip_flash_packed(*leaves, ints(dev, qo), ints(dev, ko), causal=causal, **hints)
    assert_within(y, want["out"], want["out_err"], "out")
    for name, t, u in zip(("dq", "dk", "dv"), got, torch.autograd.grad(y, leaves, g)):
      assert_within(t, want[name], want[name + "_err"], name)
      assert torch.equal(t, u), name
