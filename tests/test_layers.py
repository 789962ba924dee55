"""include/mdlayers.h without a GPU: every declared symbol is exported and bound, the header is plain C, and malformed requests are
refused on the host before anything is launched."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

from maxdiffusion_amd import _lib, layer_op, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "mdlayers.h")
P = ctypes.c_void_p
FAKE, ODD = P(0x1000), P(0x1001)  # never dereferenced: every call below must fail validation first


def test_every_declared_symbol_is_exported_and_bound(lib):
  text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
  declared = sorted(set(re.findall(r"\b(mdattn_[a-z0-9_]+)\s*\(", text)))
  assert declared == sorted(_lib.LAYER_SIGNATURES)
  for name in declared:
    assert hasattr(lib, name), name


def test_header_is_plain_c(tmp_path):
  gcc, gxx = shutil.which("gcc"), shutil.which("g++")
  if not gcc or not gxx:
    pytest.skip("no host C / C++ compiler")
  inc = os.path.dirname(HEADER)
  for exe, std, name in ((gcc, "c99", "h.c"), (gxx, "c++11", "h.cc")):
    src = tmp_path / name
    src.write_text('#include "mdlayers.h"\nint main(void) { return 0; }\n')
    subprocess.run([exe, f"-std={std}", "-Wall", "-Wextra", "-pedantic", "-Werror", "-fsyntax-only", f"-I{inc}", str(src)], check=True)


def test_layer_norm_refuses(lib):
  f = lambda x=FAKE, y=FAKE, w=FAKE, b=FAKE, xf=0, yf=0, wf=1, g=1, r=8, c=64, eps=1e-6, off=0.0: lib.mdattn_layer_norm(
      None, x, xf, y, yf, w, b, wf, g, r, c, r * c, c, r * c, c, 0, eps, off)
  assert f(x=None) == _lib.E_BADARG and f(y=None) == _lib.E_BADARG
  assert f(g=0) == f(r=0) == f(c=0) == f(c=-8) == _lib.E_BADARG
  assert f(eps=-1.0) == f(eps=float("nan")) == f(off=float("nan")) == _lib.E_BADARG
  assert f(c=16385) == _lib.E_UNSUPPORTED
  assert f(x=ODD) == f(y=ODD) == f(w=ODD) == f(b=P(0x1002)) == f(x=P(0x1002), xf=1) == _lib.E_ALIGN
  q = lambda q=FAKE, s=FAKE, c=64: lib.mdattn_layer_norm_e4m3(None, FAKE, 0, q, s, FAKE, FAKE, 1, 1, 8, c, 8 * c, c, 0, 1e-6, 0.0)
  assert q(q=None) == q(s=None) == _lib.E_BADARG and q(c=16385) == _lib.E_UNSUPPORTED and q(q=P(0x1008)) == _lib.E_ALIGN


def test_layer_norm_backward_refuses(lib):
  n = lib.mdattn_layer_norm_bwd_workspace_floats(2, 100, 64)
  assert n > 0 and n % (2 * 64) == 0
  assert lib.mdattn_layer_norm_bwd_workspace_floats(0, 100, 64) == lib.mdattn_layer_norm_bwd_workspace_floats(1, 1, 16385) == 0
  f = lambda x=FAKE, g=FAKE, dx=FAKE, w=FAKE, dw=FAKE, db=FAKE, ws=FAKE, nws=n, c=64: lib.mdattn_layer_norm_bwd(
      None, x, 0, g, dx, w, dw, db, 1, 2, 100, c, 6400, c, 6400, c, 6400, c, 0, 1e-6, 0.0, ws, nws)
  assert f(x=None) == f(g=None) == f(dx=None) == _lib.E_BADARG
  assert f(w=None) == _lib.E_BADARG  # a weight's gradient without the weight
  assert f(ws=None) == f(nws=n - 1) == _lib.E_BADARG
  assert f(c=20000) == _lib.E_UNSUPPORTED and f(dx=ODD) == f(dw=P(0x1002)) == _lib.E_ALIGN


def test_quant_refuses(lib):
  f = lambda x=FAKE, r=8, c=8, br=1, q=FAKE, s=FAKE, qt=None, st=None, cs=None: lib.mdattn_quant_block_e4m3(None, x, 0, r, c, c, br, q, s, qt, st, cs)
  assert f(x=None) == f(r=0) == f(c=0) == _lib.E_BADARG
  assert f(q=None) == f(s=None) == f(qt=FAKE) == f(st=FAKE) == f(q=None, s=None) == _lib.E_BADARG
  assert f(br=64) == _lib.E_UNSUPPORTED
  assert f(x=ODD) == f(q=P(0x1008)) == f(s=P(0x1002)) == f(cs=P(0x1002)) == _lib.E_ALIGN
  assert lib.mdattn_sum_rows(None, None, 4, 4, FAKE, 1) == lib.mdattn_sum_rows(None, FAKE, 0, 4, FAKE, 1) == _lib.E_BADARG
  assert lib.mdattn_sum_rows(None, FAKE, 4, 4, P(0x1002), 1) == _lib.E_ALIGN


def test_matmul_refuses(lib):
  f = lambda a=FAKE, sa=FAKE, b=FAKE, sb=FAKE, br=128, bias=None, bf=0, c=FAKE, cs=64, m=8, n=64, k=128, ws=None: lib.mdattn_matmul_fp8_block(
      None, a, sa, b, sb, br, bias, bf, c, cs, m, n, k, ws, 0)
  assert f(a=None) == f(sa=None) == f(b=None) == f(sb=None) == f(c=None) == _lib.E_BADARG
  assert f(m=0) == f(n=0) == f(k=0) == f(cs=63) == _lib.E_BADARG
  assert f(br=32) == f(k=(1 << 23) + 1) == f(m=1 << 31) == _lib.E_UNSUPPORTED
  assert f(a=P(0x1008)) == f(b=P(0x1008)) == f(sa=P(0x1002)) == f(c=ODD) == f(bias=ODD) == f(bias=P(0x1002), bf=1) == f(ws=P(0x1004)) == _lib.E_ALIGN


def test_python_refuses_before_it_looks_for_a_gpu():
  x = torch.zeros(2, 8)
  with pytest.raises(ValueError, match="device memory"):
    ops.layer_norm(x)
  with pytest.raises(ValueError, match="device memory"):
    layer_op.hip_layer_norm(x)
  with pytest.raises(ValueError, match="device memory"):
    ops.quant_block_e4m3(x)
  u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
  q = ops.BlockQuant(u8(3, 256), u8(3, 4), 3, 200, 1)
  assert torch.equal(q.dequantize(), torch.zeros(3, 200))
  w = ops.BlockQuant(u8(130, 128), u8(2, 4), 130, 100, 128)
  for bad in ((u8(3, 200), u8(3, 4), 3, 200, 1), (u8(3, 256), u8(3, 2), 3, 200, 1), (u8(3, 256), u8(3, 4), 3, 200, 64),
              (u8(3, 256).to(torch.int8), u8(3, 4), 3, 200, 1), (u8(256, 3).t(), u8(3, 4), 3, 200, 1)):
    with pytest.raises(ValueError, match="BlockQuant"):
      ops.BlockQuant(*bad)
  with pytest.raises(ValueError, match="device memory"):
    ops.matmul_fp8_block(q, w)
  # gradients that do not exist are refused, not dropped
  xg = torch.zeros(2, 100, dtype=torch.bfloat16, requires_grad=True)
  with pytest.raises(NotImplementedError, match="quantised weight"):
    layer_op.hip_linear_fp8(xg, w)
  with pytest.raises(NotImplementedError, match="no backward"):
    layer_op.hip_layer_norm_linear_fp8(xg, None, None, w)
  with pytest.raises(ValueError, match="must be bf16"):
    layer_op.hip_linear_fp8(xg, torch.zeros(4, 100))
  with pytest.raises(ValueError, match="weight must be"):
    layer_op.hip_linear_fp8(xg, torch.zeros(4, 99, dtype=torch.bfloat16))
