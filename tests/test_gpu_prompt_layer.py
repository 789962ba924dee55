"""A prompt encoder's layer as the operators make it up -- norm with the residual, dense layer, attention over packed prompts with grouped heads, dense layer,
norm with the residual -- trained, and answering token by token from a cache, its prologue in e4m3, in a replayed graph.  Each operator is held to
its own bound at the inputs and gradients that it met there."""
import pytest
import torch
from torch.nn import functional as F

from maxdiffusion_amd import attention_op as A
from maxdiffusion_amd import layer_op as L
from packed_reference import assert_within, attention, starts
from test_gpu_layers import BF16, F32, U, close, half_ulp, rand
from test_gpu_rms import rms64

pytestmark = pytest.mark.gpu


def check_norm(x, w, res, y, s):
  """Values and gradients of one norm, f32 stream and bf16 branch, from the tensors' own .grad (bounds: test_gpu_rms.py)."""
  want, ws, h, r, m, size = rms64(x.detach(), res.detach(), w.detach(), None, 1e-6, 0.0)
  close(y.detach(), want, half_ulp(want, BF16) + 16 * U * size, "y")
  assert torch.equal(s.detach(), x.detach().float() + res.detach())
  g, up = y.grad.double(), s.grad.double()
  a = g * m
  mean, size = (a * h).mean(-1, keepdim=True), (a * h).abs().mean(-1, keepdim=True)
  want = r * (a - h * mean) + up
  err = 32 * U * (r * (a.abs() + h.abs() * size) + up.abs()) + U * (r * (a - h * mean)).abs() + 1.02 * r * h.abs() * 2 * U * (mean.abs() + size)
  close(res.grad, want, half_ulp(want, F32) + err, "residual's gradient")
  close(x.grad, want, half_ulp(want, BF16) + err, "x's gradient")
  gh = g * h
  close(w.grad, gh.sum(0), half_ulp(gh.sum(0), w.dtype) + (2.04 * U + (2 * len(g)**0.5 + 32) * U) * gh.abs().sum(0), "w's gradient")


@pytest.mark.parametrize("h,hkv,d,c,wt", [(8, 2, 128, 512, BF16), (4, 4, 64, 200, F32), (6, 2, 40, 1000, F32)])
def test_training(dev, h, hkv, d, c, wt):
  lengths = [77, 1, 130, 0, 33]
  o = starts(lengths)
  offsets, t = torch.tensor(o, dtype=torch.int32, device=dev), o[-1]
  x, stream = rand(dev, t, c, seed=1, dtype=BF16), rand(dev, t, c, seed=2, dtype=F32, std=3.0)
  w1, w2 = (rand(dev, c, seed=i, dtype=wt, mean=1.0, std=0.2) for i in (3, 4))
  qkv_w, out_w = rand(dev, (h + 2 * hkv) * d, c, seed=5, dtype=BF16, std=c**-0.5), rand(dev, c, h * d, seed=6, dtype=BF16, std=(h * d)**-0.5)
  leaves = [z.requires_grad_(True) for z in (x, stream, w1, w2, qkv_w, out_w)]
  y1, s1 = L.hip_rms_norm(x, w1, residual=stream)
  q, k, v = F.linear(y1, qkv_w).unflatten(1, (h + 2 * hkv, d)).split((h, hkv, hkv), 1)  # views of one buffer
  att = A.hip_flash_packed(q, k, v, offsets)
  branch = F.linear(att.flatten(1), out_w)
  y2, s2 = L.hip_rms_norm(branch, w2, residual=s1)
  for z in (y1, s1, q, k, v, att, branch, y2, s2):
    z.retain_grad()
  torch.autograd.backward((y2, s2), (rand(dev, t, c, seed=7, dtype=BF16), rand(dev, t, c, seed=8, dtype=F32)))
  assert all(z.grad is not None and z.grad.dtype == z.dtype and bool(torch.isfinite(z.grad).all()) for z in leaves)
  check_norm(x, w1, stream, y1, s1)
  check_norm(branch, w2, s1, y2, s2)
  want = attention(q, k, v, o, o, dout=att.grad)
  assert_within(att, want["out"], want["out_err"], "attention")
  for name, z in (("dq", q), ("dk", k), ("dv", v)):
    assert_within(z.grad, want[name], want[name + "_err"], name)


def test_answering_from_a_cache(dev):
  """Prompts of several lengths in one call fill the cache's slots; then token by token, each step a replay of one graph, the cache's lengths on the
  device.  What the graph leaves is what the calls give outside it, and the attention at every step is the formula's over all keys so far."""
  h, hkv, d, c, room = 8, 2, 128, 640, 160
  lengths, steps = [40, 1, 97, 128], 5
  n, o = len(lengths), starts(lengths)
  w = rand(dev, c, seed=1, dtype=BF16, mean=1.0, std=0.2)
  w8 = L.quantize_weight(rand(dev, (h + 2 * hkv) * d, c, seed=2, dtype=BF16, std=c**-0.5))
  cache_k, cache_v = (torch.full((n * room, hkv, d), float("nan"), device=dev, dtype=BF16) for _ in range(2))
  slots = torch.arange(n + 1, dtype=torch.int32, device=dev) * room
  one = torch.arange(n + 1, dtype=torch.int32, device=dev)
  filled = torch.tensor(lengths, dtype=torch.int32, device=dev)

  def layer(x, stream):
    y, s = L.hip_rms_norm_linear_fp8(x, w, None, w8, residual=stream)
    return (*y.unflatten(1, (h + 2 * hkv, d)).split((h, hkv, hkv), 1), s)

  with torch.no_grad():
    x, stream = rand(dev, o[-1], c, seed=3, dtype=BF16), rand(dev, o[-1], c, seed=4, dtype=BF16)
    q, k, v, _ = layer(x, stream)
    at = torch.tensor([i * room + j for i, m in enumerate(lengths) for j in range(m)], device=dev)
    cache_k[at], cache_v[at] = k, v
    prompt = A.hip_flash_packed(q, k, v, torch.tensor(o, dtype=torch.int32, device=dev))
    # the same from the cache, whose slots hold more than the prompts
    cached = A.hip_flash_packed(q, cache_k, cache_v, torch.tensor(o, dtype=torch.int32, device=dev), slots, k_lengths=filled, max_k=room)
    want = attention(q, k, v, o, o)
    assert_within(prompt, want["out"], want["out_err"], "prompts")
    assert_within(cached, want["out"], want["out_err"], "prompts from the cache")

    x, stream = torch.empty(n, c, device=dev, dtype=BF16), torch.empty(n, c, device=dev, dtype=BF16)
    x.copy_(rand(dev, n, c, seed=10, dtype=BF16))
    stream.copy_(rand(dev, n, c, seed=20, dtype=BF16))

    def step():
      q, k, v, s = layer(x, stream)
      at = (slots[:-1] + filled).long()
      cache_k.index_copy_(0, at, k)
      cache_v.index_copy_(0, at, v)
      filled.add_(1)
      return q, A.hip_flash_packed(q, cache_k, cache_v, one, slots, k_lengths=filled, max_q=1, max_k=room), s

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      step()
    torch.cuda.current_stream().wait_stream(side)
    filled.sub_(1)  # (the step's keys are written again)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      got = step()
    for i in range(steps):
      x.copy_(rand(dev, n, c, seed=10 + i, dtype=BF16))
      stream.copy_(rand(dev, n, c, seed=20 + i, dtype=BF16))
      graph.replay()
      torch.cuda.synchronize()
      now = [m + i + 1 for m in lengths]
      assert filled.tolist() == now
      want = attention(got[0], cache_k, cache_v, list(range(n + 1)), slots.tolist(), now)
      assert_within(got[1], want["out"], want["out_err"], f"token {i}")
      filled.sub_(1)
      for a, b in zip(got, step()):
        assert torch.equal(a, b)
