"""Packed attention on the GPU: calls that its documentation allows and the forms' own tests do not make, and refusals."""
import pytest
import torch

from maxdiffusion_amd import attention_op as A
from maxdiffusion_amd import ops
from test_gpu_packed import ints, make

pytestmark = pytest.mark.gpu


def test_an_empty_head_dim_is_refused(dev):
  q, k, v, _ = (t[..., :0] for t in make(dev, 64, 64, 4, 2, 64))
  for grad in (False, True):
    for call in (A.hip_flash_packed, ops.flash_attention_packed):
      with pytest.raises(ValueError, match="head_dim=0"):
        call(q.detach().requires_grad_(grad), k, v, ints(dev, [0, 64]))
