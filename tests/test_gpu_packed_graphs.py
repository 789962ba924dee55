"""Packed attention and RMS norm in graphs that torch captures beside older autograd graphs of the same leaves, and from several threads."""
import threading

import pytest
import torch

from maxdiffusion_amd import attention_op as A
from maxdiffusion_amd import layer_op as L
from test_gpu_packed import BF16, ints, make

pytestmark = pytest.mark.gpu


class Layer(torch.nn.Module):

  def __init__(self, offsets, h=8, hkv=2, d=64, c=256):
    super().__init__()
    self.offsets, self.heads, self.d = offsets, (h, hkv, hkv), d
    gen = torch.Generator(device=offsets.device).manual_seed(1)
    r = lambda *s: torch.randn(s, generator=gen, device=offsets.device)
    self.norm = torch.nn.Parameter(1 + 0.1 * r(c))
    self.qkv = torch.nn.Parameter((r((h + 2 * hkv) * d, c) * c**-0.5).to(BF16))

  def forward(self, x, stream):
    y, s = L.hip_rms_norm(x, self.norm, residual=stream)
    q, k, v = torch.nn.functional.linear(y, self.qkv).unflatten(1, (sum(self.heads), self.d)).split(self.heads, 1)
    return A.hip_flash_packed(q, k, v, self.offsets).flatten(1), s


def test_graphed_callables(dev):
  """Torch's own warm-up leaves a graph of the parameters on the stream that it ran on."""
  offsets = ints(dev, [0, 60, 61, 200])
  layer, eager = Layer(offsets), Layer(offsets)
  inputs = lambda seed: [torch.randn(200, 256, generator=torch.Generator(device=dev).manual_seed(seed + i), device=dev).to(BF16).requires_grad_(True) for i in range(2)]
  graphed = torch.cuda.make_graphed_callables(layer, tuple(inputs(0)))
  for rep in range(3):
    got, want = [], []
    for call, module, to in ((graphed, layer, got), (eager, eager, want)):
      a = inputs(10 * rep)
      out, s = call(*a)
      torch.autograd.backward((out, s), (torch.ones_like(out), torch.full_like(s, 0.5)))
      torch.cuda.synchronize()
      to += [out.detach().clone(), s.detach().clone(), *(t.grad for t in a), *(p.grad.clone() for p in module.parameters())]
      for p in module.parameters():
        p.grad = None
    for x, y in zip(got, want):
      assert torch.equal(x, y) and bool(x.any())


def test_a_capture_beside_an_older_graph_of_a_stream_of_its_own(dev):
  q, k, v, g = make(dev, 64, 64, 4, 2, 64, seed=3)
  o = ints(dev, [0, 64])
  x, w = torch.randn(8, 256, device=dev), torch.ones(256, device=dev)
  for tensors, call, grad in (([q, k, v], lambda t: A.hip_flash_packed(*t, o), g), ([x, w], lambda t: L.hip_rms_norm(t[0], t[1]), torch.randn(8, 256, device=dev))):
    leaves = [t.clone().requires_grad_(True) for t in tensors]
    step = lambda: torch.autograd.grad(call(leaves), leaves, grad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      want = step()
      older = call(leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      got = step()
    for _ in range(3):
      for t in got:
        t.fill_(0.5)
      graph.replay()
      torch.cuda.synchronize()
      for a, b in zip(got, want):
        assert torch.equal(a, b)
    for a, b in zip(torch.autograd.grad(older, leaves, grad), want):  # the older graph is still whole
      assert torch.equal(a, b)


def test_threads(dev):
  """Training steps from four threads at once, each on a stream of its own."""
  offsets = ints(dev, [0, 100, 300])
  layer = Layer(offsets)
  x, s = (torch.randn(300, 256, generator=torch.Generator(device=dev).manual_seed(i), device=dev).to(BF16) for i in range(2))

  def step():
    leaves = [t.clone().requires_grad_(True) for t in (x, s)]
    out, total = layer(*leaves)
    return torch.autograd.grad((out, total), leaves, (torch.ones_like(out), torch.ones_like(total)))

  want = step()
  torch.cuda.synchronize()
  results = [[] for _ in range(4)]

  def run(i):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
      for _ in range(20):
        results[i].append(step())
      stream.synchronize()

  threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
  for t in threads:
    t.start()
  for t in threads:
    t.join()
  for r in results:
    assert len(r) == 20 and all(torch.equal(a, b) for got in r for a, b in zip(got, want))
