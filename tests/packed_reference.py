"""Attention over packed sequences in 64 bits, sequence by sequence and head by head, with what bf16 roundings can make of it: the
reference of the tests, and the bounds that they hold the kernels to."""
import math

import torch

U = 2.0**-8  # bf16: half a step, relative to the value


def spans(offsets, rows):
  return [(a, b) for a, b in zip(offsets, offsets[1:])]


def attention(q, k, v, q_off, k_off, k_len=None, causal=True, scale=None, dout=None, rest=True):
  """q [Tq,H,D], k, v [Tk,Hkv,D] (any type), offsets as lists -> dict of results in 64 bits and of the errors that the kernels' roundings may make:
  P and dS rounded to bf16 in front of their products, outputs rounded to bf16, everything else in f32; delta from out and, with `rest`, what
  out's rounding left (rounded in its turn: U squared)."""
  q, k, v = (t.detach().double() for t in (q, k, v))
  tq, h, d = q.shape
  hkv = k.shape[1]
  scale = d**-0.5 if scale is None else scale
  r = dict(out=torch.zeros_like(q), lse=torch.full((h, tq), -math.inf, dtype=torch.float64, device=q.device), out_err=torch.zeros_like(q))
  if dout is not None:
    g = dout.double()
    for n, like in (("dq", q), ("dk", k), ("dv", v)):
      r[n], r[n + "_err"] = torch.zeros_like(like), torch.zeros_like(like)
  for i, ((a, b), (c, e)) in enumerate(zip(spans(q_off, tq), spans(k_off, k.shape[0]))):
    if k_len is not None:
      e = min(e, c + k_len[i])
    m, n = b - a, e - c
    if not m or not n:
      continue
    hide = (torch.arange(n, device=q.device)[None] > torch.arange(m, device=q.device)[:, None] + (n - m)) if causal else None
    for j in range(h):
      kv = j // (h // hkv)
      Q, K, V = q[a:b, j], k[c:e, kv], v[c:e, kv]
      s = scale * Q @ K.T
      if hide is not None:
        s = s.masked_fill(hide, -math.inf)
      lse = torch.logsumexp(s, 1, keepdim=True)
      p = torch.where(lse == -math.inf, torch.zeros_like(s), torch.exp(s - lse))
      o = p @ V
      r["out"][a:b, j], r["lse"][j, a:b] = o, lse[:, 0]
      o_err = U * (p @ V.abs() + o.abs())
      r["out_err"][a:b, j] = o_err
      if dout is None:
        continue
      G = g[a:b, j]
      ds = p * (G @ V.T - (G * o).sum(1, keepdim=True))
      # dS is rounded, and delta comes from an out made with rounded P, itself rounded
      ds_err = U * ds.abs() + p * (G.abs() * (U * (p @ V.abs()) + U * (U if rest else 1) * o.abs())).sum(1, keepdim=True)
      r["dv"][c:e, kv] += p.T @ G
      r["dv_err"][c:e, kv] += U * (p.T @ G.abs())
      r["dq"][a:b, j] = scale * ds @ K
      r["dq_err"][a:b, j] = scale * ds_err @ K.abs()
      r["dk"][c:e, kv] += scale * ds.T @ Q
      r["dk_err"][c:e, kv] += scale * ds_err.T @ Q.abs()
  if dout is not None:
    for n in ("dq", "dk", "dv"):
      r[n + "_err"] += U * r[n].abs()
  return r


def assert_within(got, want, err, name):
  """The bound, with a part in fifty for the terms of second order, and 2^-17 of the largest value for the f32 arithmetic (logits of some 128
  products, an exponential of two units in the last place)."""
  got = got.detach().double()
  assert bool(torch.isfinite(got).all()), name
  room = 1.02 * err + 2.0**-17 * want.abs().max()
  over = (got - want).abs() - room
  worst = int(over.argmax())
  assert float(over.max()) <= 0, f"{name}: {float(got.flatten()[worst])} for {float(want.flatten()[worst])}, room {float(room.flatten()[worst]):.3g}"


def starts(lengths, front=0):
  at = [front]
  for n in lengths:
    at.append(at[-1] + n)
  return at
