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


def test_a_scale_that_the_backward_pass_refuses_is_refused_by_the_forward(dev):
  q, k, v, g = make(dev, 64, 64, 4, 2, 64)
  o = ints(dev, [0, 64])
  leaf = q.clone().requires_grad_(True)
  for t in (leaf, torch.cat((leaf, leaf), 2)[..., :64].transpose(0, 1).contiguous().transpose(0, 1)):
    with pytest.raises(ValueError, match="scale"):
      A.hip_flash_packed(t, k, v, o, scale=1e-31)
  with torch.no_grad():
    A.hip_flash_packed(leaf, k, v, o, scale=1e-31)
  y = A.hip_flash_packed(leaf, k, v, o, scale=1e-30)
  assert bool(torch.isfinite(torch.autograd.grad(y, leaf, g)[0]).all())


def test_second_derivatives_are_refused(dev):
  """By name, and where the loss has another way to the input as well: a gradient cut off would leave that one alone."""
  q, k, v, g = make(dev, 64, 64, 4, 2, 64, seed=1)
  o = ints(dev, [0, 64])
  for odd in (False, True):
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    args = [torch.cat((t, t[..., :4]), 2)[..., :64] for t in leaves] if odd else leaves  # (strides that the native node leaves to the Python one)
    y = A.hip_flash_packed(*args, o)
    for i, (leaf, grad) in enumerate(zip(leaves, torch.autograd.grad(y, leaves, g, create_graph=True))):
      with pytest.raises(NotImplementedError, match="second derivatives"):
        torch.autograd.grad(grad.float().sum() + leaf.float().square().sum(), leaf, retain_graph=True)
