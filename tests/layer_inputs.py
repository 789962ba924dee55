"""Operands of products whose results are known exactly: whole numbers and powers of two, which blocks of e4m3 hold as they are."""
import torch


def _sparse(gen, device, rows, k, nonzero, values):
  """[rows, k]: `nonzero` of the entries drawn from `values`, the others zero."""
  pick = torch.tensor(values, device=device)[torch.randint(0, len(values), (rows, k), generator=gen, device=device)]
  return pick * (torch.rand((rows, k), generator=gen, device=device) < nonzero)


def scaled(m, n, k, device, seed=0):
  """a [m, k], b [n, k] and a b^T, all f32: small whole numbers times 2^(of the row + of the block of 128 columns) in a and 2^(of the row - of the
  block) in b, so that scale bytes differ between rows and between blocks and the sums stay exact: below 256 times a power of two."""
  gen = torch.Generator(device=device).manual_seed(seed)
  a, b = (_sparse(gen, device, r, k, 3.0 * k**-0.5, (-2.0, -1.0, 1.0, 2.0)) for r in (m, n))
  want = a @ b.t()
  assert want.abs().max() < 256
  ra, rb = (torch.randint(-1, 2, (r, 1), generator=gen, device=device) for r in (m, n))
  blocks = torch.randint(-6, 7, (1, -(-k // 128)), generator=gen, device=device).repeat_interleave(128, 1)[:, :k]
  return torch.ldexp(a, ra + blocks), torch.ldexp(b, rb - blocks), torch.ldexp(want, ra + rb.t())


def cancelling(m, n, k, device, seed=0):
  """The same without powers of two, but with sums that climb to 16 K / 2 and more before they come back below 256: every partial sum needs
  the 16 to 19 bits that f32 has and bf16 or fp16 have not."""
  gen = torch.Generator(device=device).manual_seed(seed)
  half = k // 2
  a, b = torch.zeros(m, k, device=device), torch.zeros(n, k, device=device)
  lift = _sparse(gen, device, m, half, 0.1, (-2.0, -1.0, 1.0, 2.0)) + 1.0
  a[:, :half] = a[:, half : 2 * half] = lift
  b[:, :half], b[:, half : 2 * half] = 16.0, -16.0
  b += _sparse(gen, device, n, k, 2.0 * k**-0.5, (-2.0, 2.0)) * (b != 0)
  want = a @ b.t()
  assert want.abs().max() < 256 and (want != 0).any()
  return a, b, want
