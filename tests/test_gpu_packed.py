"""Attention over packed sequences on the GPU, forward, backward and by single tokens, against 64 bits.  The bounds count the roundings to bf16
that the kernels make (packed_reference.py)."""
import math

import pytest
import torch

from maxdiffusion_amd import attention_op as A
from maxdiffusion_amd import ops
from packed_reference import assert_within, attention, starts

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def make(dev, tq, tk, h, hkv, d, seed=0, lean=1.0):
  gen = torch.Generator(device=dev).manual_seed(seed)
  r = lambda *s: torch.randn(s, generator=gen, device=dev)
  q, k, v, g = r(tq, h, d), r(tk, hkv, d), r(tk, hkv, d), r(tq, h, d)
  u = r(1, 1, d) * lean * d**-0.25  # logits that reach far from 0
  return [t.to(BF16) for t in (q + u, k + u, v, g)]


def ints(dev, x):
  return torch.tensor(x, dtype=torch.int32, device=dev)


# lengths of q, lengths of k (None: the same)
BATCHES = {
    "one": ([1], None),
    "tile": ([128], None),
    "odd": ([1, 33, 0, 97, 2, 31, 32, 130], None),
    "long": ([700], None),
    "two": ([257, 300], None),
    "more_keys": ([1, 5, 64], [77, 5, 200]),
    "fewer_keys": ([40, 3, 9], [7, 0, 9]),  # rows that see no key, and a sequence without keys
    "keys_only": ([0, 12], [50, 12]),       # a sequence without rows
    "many": ([3] * 70 + [0] * 5 + [17], None),  # more sequences than a wave looks at together
}
SHAPES = [(1, 1, 128), (4, 1, 128), (6, 2, 64), (5, 1, 64), (3, 3, 80), (8, 8, 128), (2, 1, 8), (4, 2, 120), (12, 4, 40), (10, 2, 96)]


@pytest.mark.parametrize("h,hkv,d", SHAPES)
@pytest.mark.parametrize("batch", BATCHES)
def test_forward(dev, batch, h, hkv, d):
  m, n = BATCHES[batch]
  qo, ko = starts(m), starts(n or m)
  q, k, v, _ = make(dev, qo[-1], ko[-1], h, hkv, d, seed=len(batch))
  for causal in (True, False):
    print(batch, h, hkv, d, causal, flush=True)
    want = attention(q, k, v, qo, ko, causal=causal)
    for hint in (None, max(m), 1):
      out, lse = ops.flash_attention_packed(q, k, v, ints(dev, qo), ints(dev, ko), causal=causal, max_q=hint, max_k=hint and max(n or m), return_lse=True)
      assert_within(out, want["out"], want["out_err"], f"out {batch} {h} {hkv} {d} {causal} {hint}")
      none = want["lse"] == -math.inf
      assert torch.equal(lse == -math.inf, none) and not out.transpose(0, 1)[none].any()
      assert (lse - want["lse"])[~none].abs().max() <= 1e-4  # f32 logits up to some 20


@pytest.mark.parametrize("h,hkv,d", SHAPES)
@pytest.mark.parametrize("batch", BATCHES)
def test_backward(dev, batch, h, hkv, d):
  m, n = BATCHES[batch]
  qo, ko = starts(m), starts(n or m)
  q, k, v, g = make(dev, qo[-1], ko[-1], h, hkv, d, seed=len(batch) + 1, lean=0.5)
  for causal in (True, False):
    print(batch, h, hkv, d, causal, flush=True)
    want = attention(q, k, v, qo, ko, causal=causal, dout=g)
    out, lse, rest = ops.flash_attention_packed(q, k, v, ints(dev, qo), ints(dev, ko), causal=causal, return_lse=True, return_rest=True)
    for hint in (None, 1):
      got = ops.flash_attention_packed_backward(q, k, v, out, g, lse, ints(dev, qo), ints(dev, ko), rest=rest, causal=causal, max_q=hint, max_k=hint)
      for name, t in zip(("dq", "dk", "dv"), got):
        assert_within(t, want[name], want[name + "_err"], f"{name} {batch} {h} {hkv} {d} {causal} {hint}")
