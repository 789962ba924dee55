"""Attention over packed sequences without a GPU: the header, and what is refused before anything is launched."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

from maxdiffusion_amd import _lib, attention_op, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mdpacked.h")
P = ctypes.c_void_p
FAKE, ODD = P(0x1000), P(0x1008)  # never dereferenced


def test_header_and_binding_agree(lib):
  text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
  declared = sorted(set(re.findall(r"\b(mdattn_[a-z0-9_]+)\s*\(", text)))
  assert declared == sorted(_lib.PACKED_SIGNATURES)
  fields = re.search(r"typedef struct \{(.*?)\} mdattn_packed;", text, re.S).group(1)
  names = re.findall(r"(\w+)\s*(?=[,;])", fields)
  assert names == [n for n, _ in _lib.Packed._fields_]
  gcc = shutil.which("gcc")
  if gcc:
    for std in ("-std=c99", "-xc++"):
      subprocess.run([gcc, std, "-Wall", "-Wextra", "-pedantic", "-Werror", "-fsyntax-only", "-I" + os.path.dirname(HEADER), "-include", HEADER, "-x",
                      "c" if std == "-std=c99" else "c++", "/dev/null"], check=True)


def packed(**kw):
  d = dict(q_offsets=0x1000, k_offsets=0x1000, k_lengths=None, sequences=2, q_rows=300, k_rows=300, heads=8, kv_heads=2, head_dim=128, causal=1, max_q=0, max_k=0)
  d.update(kw)
  return _lib.Packed(**d)


def strides(seq=1024, head=128):
  return ctypes.byref(_lib.Strides(0, seq, head))


def fwd(lib, p=None, q=FAKE, out=FAKE, rest=None, st=None, scale=0.1, ws=None, nws=0):
  s = st or strides()
  return lib.mdattn_fwd_bf16_packed(None, ctypes.byref(p or packed()), q, FAKE, FAKE, out, rest, None, s, strides(), strides(), strides(), scale, ws, nws)


def bwd(lib, p=None, rest=None, lse=FAKE, dq=FAKE, st=None, scale=0.1, ws=FAKE, nws=1 << 40):
  s = strides()
  return lib.mdattn_bwd_bf16_packed(None, ctypes.byref(p or packed()), FAKE, FAKE, FAKE, FAKE, rest, FAKE, lse, dq, FAKE, FAKE, st or s, s, s, s, s, s, s, scale, ws, nws)


@pytest.mark.parametrize("call", [fwd, bwd])
def test_bad_arguments_are_rejected_on_the_host(lib, call):
  assert call(lib, packed(q_offsets=None)) == _lib.E_BADARG
  assert call(lib, packed(k_offsets=None)) == _lib.E_BADARG
  assert call(lib, packed(sequences=-1)) == _lib.E_BADARG
  assert call(lib, packed(q_rows=-1)) == _lib.E_BADARG
  assert call(lib, packed(heads=7)) == _lib.E_BADARG
  assert call(lib, packed(kv_heads=0)) == _lib.E_BADARG
  assert call(lib, packed(head_dim=0)) == _lib.E_BADARG
  assert call(lib, packed(head_dim=100)) == _lib.E_UNSUPPORTED
  assert call(lib, packed(head_dim=136)) == _lib.E_UNSUPPORTED
  assert call(lib, packed(q_rows=1 << 28)) == _lib.E_UNSUPPORTED  # rows of all heads are counted in 31 bits
  assert call(lib, packed(heads=4096)) == _lib.E_UNSUPPORTED
  assert call(lib, packed(q_offsets=0x1002)) == _lib.E_ALIGN
  assert call(lib, scale=0.0) == call(lib, scale=float("nan")) == call(lib, scale=float("inf")) == _lib.E_BADARG
  assert call(lib, st=strides(1025)) == call(lib, st=strides(1 << 23)) == call(lib, st=strides(-1024)) == call(lib, st=strides(1024, 4)) == _lib.E_ALIGN


def test_the_forms_own_refusals(lib):
  assert fwd(lib, q=None) == fwd(lib, out=None) == _lib.E_BADARG
  assert fwd(lib, q=ODD) == fwd(lib, rest=ODD) == bwd(lib, rest=ODD) == _lib.E_ALIGN
  assert fwd(lib, packed(q_rows=0), q=None, out=None) == _lib.E_OK  # nothing to be done
  assert bwd(lib, packed(k_lengths=0x1000)) == _lib.E_BADARG
  assert bwd(lib, dq=None) == bwd(lib, lse=None) == bwd(lib, ws=None) == bwd(lib, nws=3) == _lib.E_BADARG
  assert bwd(lib, dq=ODD) == bwd(lib, lse=P(0x1002)) == bwd(lib, st=strides(1024, 1 << 28)) == _lib.E_ALIGN
  assert bwd(lib, packed(q_rows=0, k_rows=0)) == _lib.E_OK


def test_workspaces_are_bounded_by_the_call(lib):
  """Whatever the hints say: pieces of at least 256 keys, 64 of them at most, and of at least 512 rows."""
  for hints in ((0, 0), (1, 1 << 30), (1 << 30, 1), (-5, -5), (1, 100000), (2**31 - 1, 2**31 - 1)):
    for sizes in (dict(q_rows=16, k_rows=100000, sequences=16), dict(q_rows=1, k_rows=1, sequences=1), dict(q_rows=5000, k_rows=5000, sequences=3)):
      p = packed(max_q=hints[0], max_k=hints[1], **sizes)
      n = lib.mdattn_fwd_bf16_packed_workspace_floats(ctypes.byref(p))
      assert 0 <= n <= 64 * p.q_rows * p.heads * (p.head_dim + 2)
      n = lib.mdattn_bwd_bf16_packed_workspace_floats(ctypes.byref(p))
      least = 2 * p.q_rows * p.heads
      assert least <= n <= least + 4 + (p.q_rows * 4 / 512 + 1) * 2 * p.k_rows * p.kv_heads * p.head_dim
  assert lib.mdattn_fwd_bf16_packed_workspace_floats(None) == lib.mdattn_bwd_bf16_packed_workspace_floats(None) == 0
  assert lib.mdattn_fwd_bf16_packed_workspace_floats(ctypes.byref(packed(head_dim=100))) == 0


def test_tensors_outside_the_device_are_refused(lib):
  q, o = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
  with pytest.raises(ValueError, match="device memory"):
    attention_op.hip_flash_packed(q, q, q, o)
  with pytest.raises(ValueError, match="device memory"):
    ops.flash_attention_packed(q, q, q, o)


def test_no_hint_makes_a_workspace_large(lib):
  """Pieces' rows of 256 MiB and sums of a GiB at most, whatever the hints say; with less than two pieces none."""
  for sizes in (dict(sequences=1, q_rows=1, k_rows=1 << 20), dict(sequences=512, q_rows=512, k_rows=1 << 21, heads=32, kv_heads=8),
                dict(sequences=3, q_rows=100000, k_rows=100000, heads=32, kv_heads=8), dict(sequences=1, q_rows=1 << 20, k_rows=1 << 20, heads=64, kv_heads=1),
                dict(sequences=1, q_rows=1 << 20, k_rows=1, heads=1024, kv_heads=1)):
    for max_q in (0, 1, 33, 1 << 30):
      for max_k in (0, 1, 700, 1 << 30):
        p = packed(**sizes, max_q=max_q, max_k=max_k)
        rows = p.q_rows * p.heads
        assert 0 <= lib.mdattn_fwd_bf16_packed_workspace_floats(ctypes.byref(p)) <= 1 << 26
        sums = lib.mdattn_bwd_bf16_packed_workspace_floats(ctypes.byref(p)) - (2 * rows + 3) // 4 * 4
        assert sums == 0 or 4 * p.k_rows * p.kv_heads * p.head_dim <= sums <= max(1 << 28, 4 * p.k_rows * p.kv_heads * p.head_dim)
