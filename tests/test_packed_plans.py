"""How calls of packed attention are launched, as the library plans it on the host, and what its Python entry points refuse: no GPU needed."""
import ctypes
import random

import pytest
import torch

from maxdiffusion_amd import _lib, attention_op, ops


class Plan(ctypes.Structure):
  """mdattn_host_packed_plan"""
  _fields_ = [("waves", ctypes.c_int), ("order", ctypes.c_int), ("pieces", ctypes.c_int), ("each", ctypes.c_int), ("items", ctypes.c_int64)]


def packed(**kw):
  d = dict(q_offsets=0x1000, k_offsets=0x1000, k_lengths=None, sequences=2, q_rows=300, k_rows=300, heads=8, kv_heads=2, head_dim=128, causal=1, max_q=0, max_k=0)
  d.update(kw)
  return _lib.Packed(**d)


def fwd_plan(lib, **kw):
  p, plan = packed(**kw), Plan()
  assert lib.mdattn_host_packed_fwd_plan(ctypes.byref(p), ctypes.byref(plan)) == _lib.E_OK
  return plan


def list_length(offsets, k_offsets, rows, k_rows, group, kv_heads, block, pieces, each):
  """Tiles of `block` rows with their pieces, of all heads, as the kernels' search counts them: the rows in front of the first sequence and behind the
  last among them."""
  clip = lambda x, most: min(max(x, 0), most)
  q = [0] + [clip(x, rows) for x in offsets] + [rows]
  k = [0] + [clip(x, k_rows) for x in k_offsets] + [k_rows]
  total = 0
  for i, (a, b, c, e) in enumerate(zip(q, q[1:], k, k[1:])):
    inside = 0 < i <= len(offsets) - 1
    total += -(-max(b - a, 0) * group // block) * (max(min(-(-max(e - c, 0) // each), pieces), 1) if inside else 1)
  return total * kv_heads


def test_offsets_that_rise_stay_within_the_list(lib):
  """What a call works on at most is never less than what offsets that do not decrease make."""
  rng = random.Random(1)
  for _ in range(2000):
    rows, k_rows, sequences = rng.choice([0, 1, 31, 300, 5000]), rng.choice([0, 1, 700, 40000]), rng.choice([0, 1, 3, 70, 400])
    kv_heads, group = rng.choice([1, 2, 8]), rng.choice([1, 3, 4, 16])
    hints = dict(max_q=rng.choice([0, 1, 2, 40, rows]), max_k=rng.choice([0, 1, 600, k_rows]))
    plan = fwd_plan(lib, sequences=sequences, q_rows=rows, k_rows=k_rows, heads=kv_heads * group, kv_heads=kv_heads, head_dim=rng.choice([8, 64, 128]),
                    causal=rng.randrange(2), **hints)
    assert plan.waves in (1, 2, 4) and plan.pieces >= 1 and (plan.waves == 4 or plan.pieces == 1)
    offsets = sorted(rng.choice([rng.randrange(rows + 1), 0, rows]) for _ in range(sequences + 1))
    k_offsets = sorted(rng.choice([rng.randrange(k_rows + 1), 0, k_rows]) for _ in range(sequences + 1))
    block = {1: 128, 2: 64, 4: 32}[plan.waves]
    assert list_length(offsets, k_offsets, rows, k_rows, group, kv_heads, block, plan.pieces, plan.each) <= plan.items


def test_offsets_that_go_back_do_not_lengthen_the_list(lib):
  """The walk over the list ends where offsets that rise would end at the latest, and below 2^31, whatever the offsets hold: theirs may be longer than
  31 bits count."""
  rows, sequences, group = 80000, 250000, 8
  plan = fwd_plan(lib, sequences=sequences, q_rows=rows, k_rows=rows, heads=group, kv_heads=1, head_dim=8, max_q=1)
  assert plan.waves == 4
  offsets = [0, rows] * (sequences // 2) + [0]
  assert list_length(offsets, offsets, rows, rows, group, 1, 32, plan.pieces, plan.each) >= 2**31
  assert plan.items == (rows * group // 32 + sequences + 2) * plan.pieces
  for kw in (dict(sequences=1 << 18, q_rows=1 << 18, k_rows=1 << 20, heads=16, kv_heads=1, max_q=1, max_k=1 << 20), dict(sequences=1, q_rows=1, k_rows=1 << 27, heads=8, kv_heads=1),
             dict(sequences=1, q_rows=1, k_rows=1, heads=1 << 23, kv_heads=1 << 23, head_dim=8)):
    assert fwd_plan(lib, **kw).items < 2**31


def test_plans_of_sizes_that_are_refused(lib):
  plan = Plan()
  assert lib.mdattn_host_packed_fwd_plan(None, ctypes.byref(plan)) == _lib.E_BADARG
  assert lib.mdattn_host_packed_fwd_plan(ctypes.byref(packed(head_dim=100)), ctypes.byref(plan)) == _lib.E_UNSUPPORTED


def test_an_empty_head_dim_is_refused_as_others_are(lib):
  q, o = torch.zeros(4, 2, 0, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
  for call in (attention_op.hip_flash_packed, ops.flash_attention_packed):
    with pytest.raises(ValueError):
      call(q, q, q, o)
