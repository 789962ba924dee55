"""Packed attention on offsets that are not what a program should give: the work ends, and stays inside the tensors."""
import ctypes

import pytest
import torch

from maxdiffusion_amd import _lib, ops
from test_gpu_packed import BF16, ints, make

pytestmark = pytest.mark.gpu


def test_offsets_that_go_back_and_forth(dev):
  """Every second sequence names all rows: 250,000 of them would make a list longer than 31 bits count, of which a call walks no more than offsets
  that rise could make.  The rows around the tensors are left alone."""
  rows, sequences = 80000, 250000
  o = ints(dev, [0, rows] * (sequences // 2) + [0])
  q, k, v, _ = make(dev, rows, rows, 8, 1, 8, seed=1)
  for hints in (dict(max_q=1, max_k=1), dict(max_q=1, max_k=600)):
    print(hints, flush=True)
    out, lse = ops.flash_attention_packed(q, k, v, o, max_q=hints["max_q"], max_k=hints["max_k"], causal=False, return_lse=True)
    torch.cuda.synchronize()
    assert out.shape == q.shape and lse.shape == (8, rows)


@pytest.mark.parametrize("hints", [{}, dict(max_q=1, max_k=1), dict(max_q=1, max_k=700)])
def test_what_lies_around_the_output_stays(dev, lib, hints):
  """Offsets that go back, through the C interface into the middle of a larger buffer."""
  rows, h, d = 1000, 4, 64
  q, k, v, _ = make(dev, rows, rows, h, 1, d, seed=2)
  room = torch.full((rows + 64, h, d), 7.0, dtype=BF16, device=dev)
  lse = torch.full((h * rows + 64,), 7.0, device=dev)
  for o in ([0, 1000] * 40 + [0], [500, 0, 1000, 3, 900, 2], [1000, 0], [2**31 - 1, -5, 700]):
    offsets = ints(dev, o)
    p = _lib.Packed(offsets.data_ptr(), offsets.data_ptr(), None, len(o) - 1, rows, rows, h, 1, d, 1, hints.get("max_q", 0), hints.get("max_k", 0))
    n = lib.mdattn_fwd_bf16_packed_workspace_floats(ctypes.byref(p))
    ws = torch.full((n + 64,), 7.0, device=dev)
    at = lambda t, i=0: ctypes.c_void_p(t.data_ptr() + i)
    st = lambda heads: ctypes.byref(_lib.Strides(0, heads * d, d))
    rc = lib.mdattn_fwd_bf16_packed(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), ctypes.byref(p), at(q), at(k), at(v), at(room, 32 * h * d * 2), None,
                                    at(lse, 32 * 4), st(h), st(1), st(1), st(h), 0.125, at(ws, 0), n)
    assert rc == _lib.E_OK
    torch.cuda.synchronize()
    assert bool((room[:32] == 7).all()) and bool((room[-32:] == 7).all()) and bool((lse[:32] == 7).all()) and bool((lse[-32:] == 7).all())
    assert bool((ws[n:] == 7).all())
