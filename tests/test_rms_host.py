"""RMS norm without a GPU: what its entry points refuse on the host."""
import ctypes

import pytest
import torch

from maxdiffusion_amd import _lib, layer_op, ops

P = ctypes.c_void_p
FAKE, ODD = P(0x1000), P(0x1001)  # never dereferenced: every call below must be refused before it launches anything


def test_forward_refuses(lib):
  f = lambda x=FAKE, xf=0, r=FAKE, rf=0, y=FAKE, s=FAKE, w=FAKE, b=FAKE, wf=1, g=1, n=8, c=64, eps=1e-6, off=0.0: lib.mdattn_rms_norm(
      None, x, xf, r, rf, y, s, w, b, wf, g, n, c, n * c, c, n * c, c, n * c, c, n * c, c, 0, eps, off)
  assert f(x=None) == f(y=None) == f(s=None) == f(r=None) == _lib.E_BADARG  # a sum without a residual, and the other way round
  assert f(g=0) == f(n=0) == f(c=0) == f(c=-8) == f(eps=-1.0) == f(eps=float("nan")) == f(off=float("nan")) == _lib.E_BADARG
  assert f(c=16385) == f(xf=1, rf=0) == _lib.E_UNSUPPORTED
  assert f(x=ODD) == f(y=ODD) == f(s=ODD) == f(r=ODD) == f(w=ODD) == f(b=P(0x1002)) == f(s=P(0x1002), rf=1) == f(x=P(0x1002), xf=1, rf=1) == _lib.E_ALIGN
  q = lambda q=FAKE, sc=FAKE, s=FAKE, c=64: lib.mdattn_rms_norm_e4m3(None, FAKE, 0, FAKE, 0, q, sc, s, FAKE, FAKE, 1, 1, 8, c, 8 * c, c, 8 * c, c, 8 * c, c, 0, 1e-6, 0.0)
  assert q(q=None) == q(sc=None) == q(s=None) == _lib.E_BADARG and q(c=16385) == _lib.E_UNSUPPORTED and q(q=P(0x1008)) == _lib.E_ALIGN


def test_backward_refuses(lib):
  n = lib.mdattn_rms_norm_bwd_workspace_floats(2, 100, 64)
  assert n > 0 and n % (2 * 64) == 0
  assert lib.mdattn_rms_norm_bwd_workspace_floats(0, 100, 64) == lib.mdattn_rms_norm_bwd_workspace_floats(1, 1, 16385) == 0
  f = lambda s=FAKE, sf=0, g=FAKE, gf=0, gs=FAKE, ds=FAKE, dx=None, w=FAKE, dw=FAKE, db=FAKE, ws=FAKE, nws=n, c=64, eps=1e-6, res=None: lib.mdattn_rms_norm_bwd(
      None, s, sf, res, g, gf, gs, ds, dx, w, dw, db, 1, 2, 100, c, 6400, c, 6400, c, 6400, c, 6400, c, 0, eps, 0.0, ws, nws)
  assert f(s=None) == f(g=None) == f(ds=None) == f(eps=-1.0) == _lib.E_BADARG
  assert f(w=None) == _lib.E_BADARG  # a weight's gradient without the weight
  assert f(ws=None) == f(nws=n - 1) == _lib.E_BADARG
  assert f(c=20000) == f(gf=1) == f(sf=1, gf=1, dx=FAKE) == f(sf=1, res=FAKE) == _lib.E_UNSUPPORTED
  assert f(s=ODD) == f(g=ODD) == f(gs=ODD) == f(ds=ODD) == f(sf=1, dx=ODD) == f(dw=P(0x1002)) == f(ws=P(0x1002)) == f(res=P(0x1001)) == _lib.E_ALIGN


def test_grids_past_2_32_threads_are_refused_before_a_launch(lib):
  norm = lambda groups, c: lib.mdattn_rms_norm(None, FAKE, 1, None, 0, FAKE, None, FAKE, None, 1, groups, 1, c, c, c, 0, 0, c, c, c, c, c, 1e-6, 0.0)
  assert norm(2**32 // 64, 1) == norm(2**32 // 1024, 16384) == _lib.E_UNSUPPORTED

  def backward(groups, c, vectors):
    nws = lib.mdattn_rms_norm_bwd_workspace_floats(groups, 1, c)
    d = FAKE if vectors else None
    return lib.mdattn_rms_norm_bwd(None, FAKE, 1, None, FAKE, 1, None, FAKE, None, FAKE, d, d, 1, groups, 1, c, c, c, c, c, c, c, c, c, c, 1e-6, 0.0, FAKE, nws)

  assert backward(2**32 // 1024, 64, True) == backward(2**32 // 256, 1, False) == _lib.E_UNSUPPORTED


def test_python_refuses_before_it_looks_for_a_gpu(lib):
  x = torch.zeros(2, 8)
  for call in (ops.rms_norm, ops.rms_norm_quant, layer_op.hip_rms_norm, lambda x: ops.rms_norm_backward(x, None, None, x)):
    with pytest.raises(ValueError, match="device memory"):
      call(x)
  w8 = ops.BlockQuant(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.uint8), 4, 8, 128)
  with pytest.raises(NotImplementedError, match="no backward"):
    layer_op.hip_rms_norm_linear_fp8(x.requires_grad_(True), None, None, w8)
