"""Plain implementations in 64 bits of the operators along the node order of an octree level, with the sizes of the
sums that their tolerances are made of.  One sequence after another, dense score matrices, no blocking."""
import math

import numpy as np
import torch


def half_step(dtype):
  return torch.finfo(dtype).eps / 2


def spans(offsets):
  o = [int(x) for x in offsets]
  return list(zip(o[:-1], o[1:]))


def rotary(x, pos, freq, pairs, interleaved, inverse):
  """(result, |x| + |y| of each pair) in 64 bits"""
  x = x.double().cpu()
  out, size = x.clone(), x.abs()
  n, p = sum(pairs), 0
  freq = freq.double().cpu()
  for axis, count in enumerate(pairs):
    for _ in range(count):
      # the angle in extended precision: positions in the millions must keep their phase
      t = (np.asarray(pos[:, axis].double().cpu(), dtype=np.longdouble) * np.longdouble(float(freq[p])))
      if inverse:
        t = -t
      c, s = (torch.from_numpy(np.asarray(f(t), dtype=np.float64))[:, None] for f in (np.cos, np.sin))
      i, j = (2 * p, 2 * p + 1) if interleaved else (p, n + p)
      a, b = x[..., i], x[..., j]
      out[..., i], out[..., j] = a * c - b * s, a * s + b * c
      size[..., i] = size[..., j] = a.abs() + b.abs()
      p += 1
  return out, size


def visible(lq, lk, left, right, sinks):
  p = torch.arange(lq)[:, None] + lk - lq
  j = torch.arange(lk)[None]
  ok = torch.ones(lq, lk, dtype=torch.bool)
  if right >= 0:
    ok &= j <= p + right
  if left >= 0:
    ok &= (j >= p - left) | (j < sinks)
  return ok


def attention(q, k, v, q_offsets, k_offsets, k_lengths=None, left=-1, right=-1, sinks=0, scale=None, key_mask=None,
              grad=None, dtype=None):
  """dict of out, lse (and dq, dk, dv), each with the bound `<name>_tol` on what 32-bit arithmetic and the
  roundings of the kernel's operands to `dtype` may change.

  Counted roundings.  u = half a step of `dtype` (2^-24 for fp32).  A score is a sum of dim products in 32
  bits: off by ds <= dim 2^-24 scale sum|q||k| (plus 2^-22 |s| of the exponent's argument); every probability is
  then off by the factor 2 ds and by 2^-20 of the 32-bit exponential, sum and division.
    out: sum p |v| (2 ds + 2^-20 + u for the probability as an operand) + u |out| for the result
    dv : the same sums over the queries, with dO for v
    dS = P (dP - D): dP is off by dim 2^-24 sum|dO||v|, D by u sum|dO||out| (the stored output is rounded), P as
         above, and dS is rounded as an operand (u); dq, dk sum these with |k|, |q|.
  For fp32 operands are not rounded: u counts the sums' own roundings instead, which 2^-20 covers many times over."""
  q, k, v = (t.double().cpu() for t in (q, k, v))
  heads, kvh, dim = q.size(1), k.size(1), q.size(2)
  scale = dim ** -0.5 if scale is None else scale
  u = half_step(dtype) if dtype is not None else 0.0
  r = {"out": torch.zeros_like(q), "out_tol": torch.zeros_like(q),
       "lse": torch.full(q.shape[:2], -math.inf, dtype=torch.float64), "lse_tol": torch.zeros(q.shape[:2], dtype=torch.float64)}
  if grad is not None:
    grad = grad.double().cpu()
    for n, t in (("dq", q), ("dk", k), ("dv", v)):
      r[n], r[n + "_tol"] = torch.zeros_like(t), torch.zeros_like(t)
  group = heads // kvh
  for b, ((qa, qb), (ka, kb)) in enumerate(zip(spans(q_offsets), spans(k_offsets))):
    lq, lk = qb - qa, kb - ka
    if k_lengths is not None:
      lk = min(max(int(k_lengths[b]), 0), lk)
    if not lq or not lk:
      continue
    ok = visible(lq, lk, left, right, sinks)
    if key_mask is not None:
      ok &= key_mask[ka:ka + lk].cpu()[None]
    some = ok.any(1)
    for h in range(heads):
      g = h // group
      qh, kh, vh = q[qa:qb, h], k[ka:ka + lk, g], v[ka:ka + lk, g]
      # (what a key or value that no query sees holds has no influence)
      seen = ok.any(0)[:, None]
      kh, vh = torch.where(seen, kh, 0.0), torch.where(seen, vh, 0.0)
      s = (qh @ kh.t()) * scale
      s = torch.where(ok, s, -math.inf)
      ds = (qh.abs() @ kh.abs().t()) * (abs(scale) * dim * 2.0 ** -24) + torch.where(ok, s.abs(), 0.0) * 2.0 ** -22
      ds = torch.where(ok, ds, 0.0).amax(1, keepdim=True)
      top = torch.where(some, s.amax(1), 0.0)
      lse = torch.where(some, top + torch.log(torch.exp(s - top[:, None]).sum(1)), -math.inf)
      p = torch.where(ok, torch.exp(s - torch.where(some, lse, 0.0)[:, None]), 0.0)
      out = p @ vh
      rel = 2 * ds + 2.0 ** -20 + u
      r["out"][qa:qb, h], r["lse"][qa:qb, h] = out, lse
      r["out_tol"][qa:qb, h] = (p @ vh.abs()) * rel + u * out.abs()
      r["lse_tol"][qa:qb, h] = torch.where(some, ds[:, 0] + 2.0 ** -20 * (1 + lse.abs()), 0.0)
      if grad is None:
        continue
      go = grad[qa:qb, h]
      dp, delta = go @ vh.t(), (go * out).sum(1, keepdim=True)
      dscore = p * (dp - delta)
      size = p * ((dp - delta).abs() * rel + dim * 2.0 ** -24 * (go.abs() @ vh.abs().t())
                  + (u + 2.0 ** -20) * (go.abs() * out.abs()).sum(1, keepdim=True)
                  + (go.abs() * r["out_tol"][qa:qb, h]).sum(1, keepdim=True))
      r["dq"][qa:qb, h] = dscore @ kh * scale
      r["dq_tol"][qa:qb, h] = (size + 2.0 ** -20 * dscore.abs()) @ kh.abs() * abs(scale)
      r["dk"][ka:ka + lk, g] += dscore.t() @ qh * scale
      r["dk_tol"][ka:ka + lk, g] += (size + 2.0 ** -20 * dscore.abs()).t() @ qh.abs() * abs(scale)
      r["dv"][ka:ka + lk, g] += p.t() @ go
      r["dv_tol"][ka:ka + lk, g] += (p * rel).t() @ go.abs()
  if grad is not None:
    for n in ("dq", "dk", "dv"):
      r[n + "_tol"] += u * r[n].abs()
  return r


def recurrence(gate, data, offsets, state=None, reverse=False, grad=None, grad_last=None):
  """dict of out, last (and dgate, ddata, dstate), row by row in 64 bits"""
  g, x = gate.double().cpu(), data.double().cpu()
  n, c = x.shape
  seqs = spans(offsets)
  a, b = torch.sigmoid(g), torch.sigmoid(-g)
  h0 = torch.zeros(len(seqs), c, dtype=torch.float64) if state is None else state.double().cpu()
  r = {"out": torch.zeros_like(x), "last": h0.clone()}
  if grad is not None:
    r |= {"dgate": torch.zeros_like(x), "ddata": torch.zeros_like(x), "dstate": torch.zeros_like(h0)}
    grad = grad.double().cpu()
  for i, (begin, end) in enumerate(seqs):
    rows = list(range(begin, end))
    if reverse:
      rows.reverse()
    h, before = h0[i], {}
    for t in rows:
      before[t] = h
      h = a[t] * h + b[t] * x[t]
      r["out"][t] = h
    r["last"][i] = h
    if grad is None:
      continue
    m = torch.zeros(c, dtype=torch.float64) if grad_last is None else grad_last[i].double().cpu()
    for t in reversed(rows):
      lam = grad[t] + m
      r["ddata"][t] = b[t] * lam
      r["dgate"][t] = a[t] * b[t] * lam * (before[t] - x[t])
      m = a[t] * lam
    r["dstate"][i] = m
  return r


def recurrence_tolerance(gate, data, state, dtype, longest):
  """Bound on |h|'s 32-bit error: a step adds at most 2^-20 of the largest value around (two roundings of the
  update and the gates' 2^-22), and a step keeps a part a of what was there: over a sequence the sum is at most
  min(its length, 1 / (1 - a_max)) such steps."""
  big = float(data.double().abs().max()) if data.numel() else 0.0
  if state is not None and state.numel():
    big = max(big, float(state.double().abs().max()))
  b_min = float(torch.sigmoid(-gate.double()).min()) if gate.numel() else 1.0
  return big * 2.0 ** -20 * (1 + min(longest, 1 / max(b_min, 1e-300)))
