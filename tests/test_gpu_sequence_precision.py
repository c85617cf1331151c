"""How exact the operators along the node order of an octree level are where a looser bound would hide a missing term: rows
that see few keys, gradients over long sequences.  References in 64 bits, bounds from the roundings that are counted beside
each."""
import pytest
import torch

import sequence_reference as ref
from test_gpu_sequence import BF16, attention_inputs, offs, within

pytestmark = pytest.mark.gpu


# ---- rows that see few keys -----------------------------------------------------------------------------
def few_rows_reference(q, k, v, go, lengths, left, right, sinks, mask):
  """Gradients in 64 bits and their bounds where rowsum(P dP) comes from the scores and not from the output in bf16.

  e_s, e_p: the sums of dim products q k and dO v in 32 bits.  P is off by the factor r = 2 e_s + 2^-19 (1 + |lse|) (scores,
  lse, exponential), D = rowsum(P dP) by e_D = sum P (r |dP| + e_p + 2^-20 |dP|), dS = P (dP - D) by |dS| (r + 2^-17)
  + P (e_p + e_D) -- 2^-17: held as two bf16 -- and dq, dk sum that with |k|, |q| in 32 bits (2^-20 of the terms) and are
  rounded once.  dO is taken as zero for rows that see more than 32 keys, which are not meant here."""
  heads, kvh, dim = q.size(1), k.size(1), q.size(2)
  scale, u = dim ** -0.5, ref.half_step(BF16)
  r = {n: torch.zeros(t.shape, dtype=torch.float64) for n, t in (("dq", q), ("dq_tol", q), ("dk", k), ("dk_tol", k))}
  few_rows = torch.zeros(q.size(0), dtype=torch.bool)
  for a, b in ref.spans(offs(lengths)):
    if a == b:
      continue
    ok = ref.visible(b - a, b - a, left, right, sinks)
    if mask is not None:
      ok &= mask[a:b][None]
    few_rows[a:b] = ok.sum(1) <= 32
    few = few_rows[a:b, None]
    go[a:b] *= few[:, :, None]
    for h in range(heads):
      g = h // (heads // kvh)
      qh, gh = q[a:b, h].double(), go[a:b, h].double()
      kh, vh = k[a:b, g].double(), v[a:b, g].double()
      s = torch.where(ok, qh @ kh.t() * scale, -float("inf"))
      some = ok.any(1, keepdim=True)
      lse = torch.where(some, torch.logsumexp(s, 1, keepdim=True), 0.0)
      p = torch.where(ok, torch.exp(s - lse), 0.0)
      e_s = (qh.abs() @ kh.abs().t()) * (scale * dim * 2.0 ** -24)
      e_p = (gh.abs() @ vh.abs().t()) * (dim * 2.0 ** -24)
      rel = 2 * torch.where(ok, e_s, 0.0).amax(1, keepdim=True) + 2.0 ** -19 * (1 + lse.abs())
      dp = gh @ vh.t()
      big_d = (p * dp).sum(1, keepdim=True)
      e_d = (p * (dp.abs() * (rel + 2.0 ** -20) + e_p)).sum(1, keepdim=True)
      ds = p * (dp - big_d)
      e_ds = ds.abs() * (rel + 2.0 ** -17 + 2.0 ** -20) + p * (e_p + e_d)
      r["dq"][a:b, h] = ds @ kh * scale
      r["dq_tol"][a:b, h] = e_ds @ kh.abs() * scale
      r["dk"][a:b, g] += ds.t() @ qh * scale
      r["dk_tol"][a:b, g] += e_ds.t() @ qh.abs() * scale
  for n in ("dq", "dk"):
    r[n + "_tol"] += u * r[n].abs()
  return r, few_rows


FEW = [
    # lengths, heads, kv heads, dim, left, right, sinks, every how many keys the mask keeps
    ([200], 2, 1, 64, -1, 0, 0, 0), ([1500, 90, 40, 0, 1], 4, 4, 32, 511, 0, 0, 0), ([300, 70], 2, 2, 96, 40, 0, 4, 0),
    ([150, 33], 4, 1, 128, 0, -1, 0, 0), ([400, 100], 2, 1, 64, 200, 200, 3, 20), ([700], 3, 3, 64, -1, -1, 0, 23),
    ([260], 2, 2, 40, 60, 10, 2, 3),
]


@pytest.mark.parametrize("empty", [0, 330], ids=["few-workgroups", "many"])
@pytest.mark.parametrize("case", FEW, ids=lambda c: "%s-%dx%dx%d-%d-%d-%d-%d" % (("+".join(map(str, c[0])),) + c[1:]))
def test_gradient_of_rows_that_see_few_keys(oc, case, empty):
  """the output in bf16 would leave their dq twice as far off as its own rounding (2 keys), and the dk of the keys they see;
  empty sequences behind, which the rules count as work, take the larger workgroups"""
  lengths, heads, kvh, dim, left, right, sinks, every = case
  q, k, v, go = attention_inputs(lengths, lengths, heads, kvh, dim, BF16, 51)
  mask = torch.arange(sum(lengths)) % every == 0 if every else None
  want, few = few_rows_reference(q, k, v, go, lengths, left, right, sinks, mask)
  assert 8 <= int(few.sum())
  q, k, v, go, o = (t.cuda() for t in (q, k, v, go, offs(lengths + [0] * empty)))
  kw = dict(left=left, right=right, sinks=sinks, key_mask=mask.cuda() if every else None)
  out, lse = oc.nn.octree_attention(q, k, v, o, return_lse=True, **kw)
  dq, dk, _ = oc.nn.octree_attention_grad(go, q, k, v, out, lse, o, **kw)
  within(dq[few.cuda()], want["dq"][few], want["dq_tol"][few], "dq")
  within(dk, want["dk"], want["dk_tol"], "dk")
