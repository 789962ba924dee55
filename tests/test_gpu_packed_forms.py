"""Attention over packed sequences in each of its forms -- four waves that share the keys of 32 rows, two those of 64, none those of 128 -- and orders of
the tiles, which sizes and hints choose, against 64 bits."""
import math

import pytest
import torch

from maxdiffusion_amd import attention_op as A
from maxdiffusion_amd import layer_op as L
from maxdiffusion_amd import ops
from packed_reference import assert_within, attention, starts
from test_gpu_packed import ints, make

pytestmark = pytest.mark.gpu
LENGTHS = [1, 33, 0, 97, 300, 2, 513, 130, 64]

# sequences without rows behind the others, heads, heads of k and v, the longest lengths as the call gives them
FORMS = {
    "shared by four": (0, 4, 2, (1, 1)),
    "shared by four, several tiles": (0, 2, 1, (None, None)),
    "shared by two": (60, 2, 1, (None, None)),         # 86 tiles of 128 rows at most, of more sequences than are sorted
    "shared by two, sorted": (20, 4, 4, (None, None)),
    "shared by two, both ends": (0, 15, 15, (None, None)),  # 17 tiles of 64 rows for the first round of the heads, the others from the other end
    "not shared": (0, 4, 2, (None, 1)),
    "not shared, sorted": (10, 16, 16, (None, None)),
    "not shared, both ends": (0, 32, 32, (None, None)),
    "not shared, many": (100, 12, 4, (None, None)),
}


@pytest.mark.parametrize("d", [64, 40, 80, 128, 104])
@pytest.mark.parametrize("form", FORMS)
def test_forms(dev, form, d):
  empty, h, hkv, (max_q, max_k) = FORMS[form]
  lengths = LENGTHS + [0] * empty
  o = starts(lengths)
  q, k, v, g = make(dev, o[-1], o[-1], h, hkv, d, seed=len(form), lean=0.5)
  offsets = ints(dev, o)
  for causal in (True, False):
    print(form, d, causal, flush=True)
    want = attention(q, k, v, o, o, causal=causal, dout=g)
    out, lse, rest = ops.flash_attention_packed(q, k, v, offsets, causal=causal, max_q=max_q, max_k=max_k, return_lse=True, return_rest=True)
    assert_within(out, want["out"], want["out_err"], f"out {form} {d} {causal}")
    assert (lse - want["lse"]).abs().max() <= 1e-4  # f32 logits up to some 20
    for name, t in zip(("dq", "dk", "dv"), ops.flash_attention_packed_backward(q, k, v, out, g, lse, offsets, rest=rest, causal=causal, max_q=max_q, max_k=max_k)):
      assert_within(t, want[name], want[name + "_err"], f"{name} {form} {d} {causal}")


def test_other_lengths_of_the_keys_in_each_order(dev):
  """Rows that see no key, keys that no row sees, and sequences of one side alone, sorted by what they meet."""
  m, n = [40, 0, 300, 7, 129, 64, 1], [7, 50, 300, 0, 1000, 3, 257]
  qo, ko = starts(m, 3), starts(n, 5)
  for h, hkv, d in ((32, 32, 64), (48, 24, 128), (12, 12, 96)):
    q, k, v, g = make(dev, qo[-1] + 9, ko[-1] + 2, h, hkv, d, seed=d, lean=0.5)
    for causal in (True, False):
      print(h, hkv, d, causal, flush=True)
      want = attention(q, k, v, qo, ko, causal=causal, dout=g)
      out, lse, rest = ops.flash_attention_packed(q, k, v, ints(dev, qo), ints(dev, ko), causal=causal, return_lse=True, return_rest=True)
      assert_within(out, want["out"], want["out_err"], f"out {h} {causal}")
      assert torch.equal(lse == -math.inf, want["lse"] == -math.inf)
      for name, t in zip(("dq", "dk", "dv"), ops.flash_attention_packed_backward(q, k, v, out, g, lse, ints(dev, qo), ints(dev, ko), rest=rest, causal=causal)):
        assert_within(t, want[name], want[name + "_err"], f"{name} {h} {causal}")


def test_a_capture_beside_an_older_graph_of_the_same_leaves_is_refused(dev):
  q, k, v, g = make(dev, 64, 64, 4, 2, 64, seed=3)
  o = ints(dev, [0, 64])
  x, w = torch.randn(8, 256, device=dev), torch.ones(256, device=dev)
  cases = [([q, k, v], lambda t: A.hip_flash_packed(*t, o), g), ([x, w], lambda t: L.hip_rms_norm(t[0], t[1]), torch.randn(8, 256, device=dev))]
  for tensors, call, grad in cases:
    leaves = [t.clone().requires_grad_(True) for t in tensors]
    step = lambda: torch.autograd.grad(call(leaves), leaves, grad)
    want = step()
    older = call(leaves)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      torch.zeros(1, device=dev)
      with pytest.raises(RuntimeError, match="another stream"):
        call(leaves)
    del older
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      got = step()
    for _ in range(2):
      for t in got:
        t.fill_(0.5)
      graph.replay()
      torch.cuda.synchronize()
      for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_thousands_of_sequences(dev):
  """More sequences than a workgroup looks through at once: short ones, and single tokens against caches of which a few are long."""
  gen = torch.Generator().manual_seed(5)
  m = torch.randint(0, 4, (4500,), generator=gen).tolist()
  m[4400] = 150
  o = starts(m)
  q, k, v, g = make(dev, o[-1], o[-1], 2, 1, 64, seed=6, lean=0.5)
  want = attention(q, k, v, o, o, dout=g)
  for hints in ({}, dict(max_q=1, max_k=1), dict(max_q=150, max_k=150)):
    out, lse, rest = ops.flash_attention_packed(q, k, v, ints(dev, o), return_lse=True, return_rest=True, **hints)
    assert_within(out, want["out"], want["out_err"], f"out {hints}")
    for name, t in zip(("dq", "dk", "dv"), ops.flash_attention_packed_backward(q, k, v, out, g, lse, ints(dev, o), rest=rest, **hints)):
      assert_within(t, want[name], want[name + "_err"], f"{name} {hints}")
  n = [1 + i % 3 for i in range(1500)]
  n[7], n[700], n[1499] = 5000, 2000, 900
  one, ko = list(range(len(n) + 1)), starts(n)
  q, k, v, _ = make(dev, len(n), ko[-1], 2, 1, 128, seed=7)
  want = attention(q, k, v, one, ko)
  out = ops.flash_attention_packed(q, k, v, ints(dev, one), ints(dev, ko), max_q=1, max_k=5000)
  assert_within(out, want["out"], want["out_err"], "tokens")
