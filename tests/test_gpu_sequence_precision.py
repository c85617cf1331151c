"""How exact the operators along the node order of an octree level are where a looser bound would hide a missing term: rows
that see few keys, gradients over long sequences.  References in 64 bits, bounds from the roundings that are counted beside
each."""
import pytest
import torch

import sequence_reference as ref
from test_gpu_sequence import BF16, attention_inputs, offs, recurrence_inputs, within

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


# ---- the recurrence, row by row ---------------------------------------------------------------------------
def recurrence_bounds(gate, data, offsets, state=None, reverse=False, grad=None, grad_last=None):
  """ref.recurrence's results and a bound for each element.

  h_t is a sum of terms b_s x_s a_{s+1} .. a_t.  The kernels form a and b to the relative errors ra = 2^-22 (1 + b |g|) and
  rb = 2^-22 (1 + a |g|) (the argument of the exponential is rounded), and multiply and add in 32 bits in whatever order the
  chunks give.  So each factor of a term costs ra + 2^-23, and each term passes at most 48 sums of partial results beside the
  steps of the recurrence: with H_t = a H_{t-1} + b |x| the sum of the terms' sizes,
    E_t = a (E_{t-1} + (ra + 2^-23) H_{t-1}) + b (rb + 2^-23) |x|,  |error of h_t| <= E_t + 48 2^-23 H_t,
  which follows the local a_t.  The gradient's sum L_t = dh_t + a_{t+1} L_{t+1} is bounded in the same way;
    dx = b L, dg = a b L (h_{t-1} - x)
  carry the bounds of their factors, ra + rb for a and b and 2^-22 for the products and the difference."""
  g, x = gate.double().cpu(), data.double().cpu()
  a, b = torch.sigmoid(g), torch.sigmoid(-g)
  ra, rb = 2.0 ** -22 * (1 + b * g.abs()) + 2.0 ** -23, 2.0 ** -22 * (1 + a * g.abs()) + 2.0 ** -23
  seqs, c = ref.spans(offsets), x.size(1)
  h0 = torch.zeros(len(seqs), c, dtype=torch.float64) if state is None else state.double().cpu()
  r = {"out": torch.zeros_like(x), "last": h0.clone()}
  if grad is not None:
    r |= {"dgate": torch.zeros_like(x), "ddata": torch.zeros_like(x), "dstate": torch.zeros_like(h0)}
    grad = grad.double().cpu()
  r |= {n + "_tol": torch.zeros_like(t) for n, t in r.items()}
  many = 48 * 2.0 ** -23
  for i, (begin, end) in enumerate(seqs):
    rows = range(end - 1, begin - 1, -1) if reverse else range(begin, end)
    h, size, e = h0[i], h0[i].abs(), torch.zeros(c, dtype=torch.float64)
    before, slack = torch.zeros(end - begin, c, dtype=torch.float64), torch.zeros(end - begin, c, dtype=torch.float64)
    for n, t in enumerate(rows):
      before[n], slack[n] = h, e + many * size
      e = a[t] * (e + ra[t] * size) + b[t] * rb[t] * x[t].abs()
      h, size = a[t] * h + b[t] * x[t], a[t] * size + b[t] * x[t].abs()
      r["out"][t], r["out_tol"][t] = h, e + many * size
    r["last"][i], r["last_tol"][i] = h, e + many * size
    if grad is None:
      continue
    m = torch.zeros(c, dtype=torch.float64) if grad_last is None else grad_last[i].double().cpu()
    size, e = m.abs(), torch.zeros(c, dtype=torch.float64)
    for n, t in reversed(list(enumerate(rows))):
      lam, lam_size, lam_e = grad[t] + m, grad[t].abs() + size, e + 2.0 ** -23 * (grad[t].abs() + size)
      lam_e = lam_e + many * lam_size
      gap, gap_e = (before[n] - x[t]).abs(), slack[n] + 2.0 ** -23 * (before[n].abs() + x[t].abs())
      r["ddata"][t], r["ddata_tol"][t] = b[t] * lam, b[t] * (lam_e + (rb[t] + 2.0 ** -22) * lam_size)
      r["dgate"][t] = a[t] * b[t] * lam * (before[n] - x[t])
      r["dgate_tol"][t] = a[t] * b[t] * (lam_e * (gap + gap_e) + lam.abs() * (gap_e + (ra[t] + rb[t] + 2.0 ** -22) * gap))
      e = a[t] * (e + (ra[t] + 2.0 ** -23) * lam_size)
      m, size = a[t] * lam, a[t] * lam_size
    r["dstate"][i], r["dstate_tol"][i] = m, e + many * size
  return r


def held(got, want, name, dtype):
  """within the bound (and the result's rounding), and the bound is one that a missing term cannot meet"""
  tol = want[name + "_tol"] + (ref.half_step(dtype) if name not in ("last", "dstate") else 2.0 ** -24) * want[name].abs()
  if want[name].numel():
    assert float(tol.max()) <= 2.0 ** -7 * float(want[name].abs().max()), (name, float(tol.max()), float(want[name].abs().max()))
  within(got, want[name], tol, name)


SKEWED = [
    # sequences of a few rows on average with long ones among them; channels; rows behind the last
    ([1] * 63 + [961], 64, 0), ([1] * 255 + [3800], 97, 0), ([3800] + [1] * 255, 8, 5), ([0] * 130 + [65, 64, 63, 1000, 0, 128], 20, 0),
    ([1] * 40, 33, 500), ([2] * 100 + [300, 0, 1, 700] + [3] * 200, 256, 65), ([5] * 3000 + [6000] + [0] * 1000, 130, 0),
]


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("case", SKEWED, ids=lambda c: "%d-rows-in-%d-x-%d+%d" % (sum(c[0]), len(c[0]), c[1], c[2]))
def test_recurrence_of_single_rows_and_a_long_sequence(oc, case, dtype, reverse):
  """a step of running sequences together with a new one, without carries: one launch, which must not walk the long one"""
  lengths, channels, extra = case
  gate, data, state, _, _ = recurrence_inputs(lengths, channels, dtype, 61, extra)
  o = offs(lengths)
  want = recurrence_bounds(gate, data, o, state, reverse)
  args = [t.cuda() for t in (gate, data, o, state)]
  out, last = oc.nn.octree_recurrence(*args, reverse)
  held(out, want, "out", dtype)
  held(last, want, "last", dtype)
  room = torch.full_like(out, 5.0)
  again, last2 = oc.nn.octree_recurrence(*args, reverse, out=room)
  assert torch.equal(again[:sum(lengths)], out[:sum(lengths)]) and torch.equal(last2, last)
  assert bool((room[sum(lengths):] == 5.0).all()) and bool((out[sum(lengths):] == 0).all())


@pytest.mark.parametrize("lengths, extra", [([1] * 255 + [3800], 0), ([1] * 2047 + [20000], 0), ([1] * 1000, 15000)],
                         ids=["3800-among-255", "20000-among-2047", "rows-of-none"])
def test_skewed_batches_do_not_wait_for_one_thread(oc, lengths, extra):
  """The call that keeps carries takes forms that are bounded by the rows; the one without took 20 times as long and more, a
  thread a channel walking the longest sequence.  (Eight times is far from both.)"""
  gate, data, state, _, _ = (t.cuda() for t in recurrence_inputs(lengths, 64, BF16, 62, extra))
  o = offs(lengths).cuda()

  def time(carries):
    best = float("inf")
    for _ in range(8):
      begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
      begin.record()
      oc.nn.octree_recurrence(gate, data, o, state, return_carries=carries)
      end.record()
      torch.cuda.synchronize()
      best = min(best, begin.elapsed_time(end))
    return best
  bounded = time(True)
  assert time(False) < 8 * max(bounded, 0.02)


LONG = [
    # lengths, channels: a workgroup a sequence; chunks whose list is scanned in one launch, in two; chunks of 64 rows
    ([1000, 3, 0, 777], 12), ([300] * 20, 33), ([5000], 12), ([20000], 24), ([9000, 0, 1, 7777, 300], 256), ([12000, 1, 0, 8003], 1680),
]


@pytest.mark.parametrize("dtype", [torch.float32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("case, reverse, ends", [
    pytest.param(c, r, e, id="%s-%d%s-%s" % ("+".join(map(str, c[0][:5])), c[1], "-reverse" if r else "", "state" if e else "zeros"))
    for c in LONG for r in (False, True) for e in (True, False) if c[1] < 1000 or r != e])
def test_gradient_of_the_recurrence_over_long_sequences(oc, case, dtype, reverse, ends):
  """every result within a bound that follows the local gates: of the forward call, and of the gradient with and without a
  state to begin with and a gradient of the last one"""
  lengths, channels = case
  gate, data, state, dy, dl = recurrence_inputs(lengths, channels, dtype, 63, extra=9)
  if not ends:
    state = dl = None
  o = offs(lengths)
  want = recurrence_bounds(gate, data, o, state, reverse, dy, dl)
  gate, data, state, dy, dl, o = (None if t is None else t.cuda() for t in (gate, data, state, dy, dl, o))
  out, last, carries = oc.nn.octree_recurrence(gate, data, o, state, reverse, return_carries=True)
  held(out, want, "out", dtype)
  held(last, want, "last", dtype)
  grads = oc.nn.octree_recurrence_grad(dy, gate, data, o, carries, state, dl, reverse)
  for name, g in zip(("dgate", "ddata", "dstate"), grads):
    held(g, want, name, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, BF16], ids=["float32", "bfloat16"])
def test_skewed_batches_repeat_in_graphs(oc, dtype):
  """the launch that walks short sequences and scans long ones, captured twice, replayed with new inputs and at once"""
  lengths = [2] * 100 + [300, 0, 1, 700] + [3] * 200
  gate, data, state, _, _ = (t.cuda() for t in recurrence_inputs(lengths, 72, dtype, 66, 90))
  o = offs(lengths).cuda()
  run = lambda: oc.nn.octree_recurrence(gate, data, o, state, True)   # noqa: E731
  run()
  torch.cuda.synchronize()
  graphs = []
  for _ in range(2):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      outs = run()
    graphs.append((g, outs))
  side = torch.cuda.Stream()
  for turn in range(4):
    data.copy_(torch.randn(data.shape, generator=torch.Generator().manual_seed(turn)).to(dtype))
    want = run()
    torch.cuda.synchronize()
    graphs[0][0].replay()
    with torch.cuda.stream(side):
      graphs[1][0].replay()
    torch.cuda.synchronize()
    for _, outs in graphs:
      assert all(torch.equal(a, b) for a, b in zip(outs, want)), turn


# ---- probabilities as operands ------------------------------------------------------------------------------
STEPS = [
    # query lengths, key lengths, heads, kv heads, dim, window: few rows a sequence
    ([1, 1, 1], [50, 1, 200], 8, 2, 64, dict(right=0)), ([1, 2, 0, 3], [300, 40, 9, 70], 4, 1, 128, dict(left=20, right=0, sinks=2)),
    ([7], [600], 3, 1, 48, dict(left=30)), ([2, 1], [2000, 900], 6, 2, 24, {}), ([9, 20, 4], [9, 20, 4], 2, 2, 96, dict(right=0)),
]


@pytest.mark.parametrize("case", STEPS, ids=lambda c: "%s-of-%s-%dx%dx%d" % (
    "+".join(map(str, c[0])), "+".join(map(str, c[1])), c[2], c[3], c[4]))
def test_probabilities_of_few_rows_are_not_rounded_once(oc, case):
  """The bound of ref.attention without the rounding of the probabilities, but for 2^-17 of each: two bf16.  (Products waiting
  for memory, the second one costs nothing.)"""
  qlen, klen, heads, kvh, dim, window = case
  q, k, v, _ = attention_inputs(qlen, klen, heads, kvh, dim, BF16, 71)
  qo, ko = offs(qlen), offs(klen)
  want = ref.attention(q, k, v, qo, ko, **window)
  size = ref.attention(q, k, v.abs(), qo, ko, **window)["out"]
  out = oc.nn.octree_attention(q.cuda(), k.cuda(), v.cuda(), qo.cuda(), ko.cuda(), **window)
  within(out, want["out"], want["out_tol"] + size * 2.0 ** -17 + ref.half_step(BF16) * want["out"].abs(), "out")


@pytest.mark.parametrize("empty", [0, 330], ids=["few-workgroups", "many"])
@pytest.mark.parametrize("lengths, heads, kvh, dim, window", [
    ([300], 2, 1, 64, dict(right=0)), ([90, 200, 1], 4, 2, 32, dict(left=20, right=20, sinks=3)), ([140], 2, 2, 128, {}),
    ([700], 2, 1, 96, dict(left=9, right=0, sinks=40))], ids=["300", "90+200+1", "140", "700"])
def test_gradient_of_the_values_is_not_rounded_twice(oc, lengths, heads, kvh, dim, window, empty):
  """dv = P^T dO with P off by 2 e_s + 2^-19 (1 + |lse|) (scores, lse, exponential) and 2^-17 (two bf16), rounded once"""
  q, k, v, go = attention_inputs(lengths, lengths, heads, kvh, dim, BF16, 72)
  o = offs(lengths)
  want = ref.attention(q, k, v, o, o, grad=go, **window)
  # sum over the rows of P |dO|, and the largest relative error of a probability: the scores' from their own largest size
  size = ref.attention(q, k, v, o, o, grad=go.abs(), **window)["dv"]
  e_s = dim ** 0.5 * 2.0 ** -24 * max(float((q[a:b, h].double().abs() @ k[a:b, h * kvh // heads].double().abs().t()).max())
                                      for a, b in ref.spans(o) for h in range(heads))
  rel = 2 * e_s + 2.0 ** -19 * (1 + float(want["lse"].abs().max())) + 2.0 ** -17
  assert rel < 2.0 ** -11                    # (far below a rounding to bf16)
  o = offs(lengths + [0] * empty).cuda()
  q, k, v, go = (t.cuda() for t in (q, k, v, go))
  out, lse = oc.nn.octree_attention(q, k, v, o, return_lse=True, **window)
  dv = oc.nn.octree_attention_grad(go, q, k, v, out, lse, o, **window)[2]
  within(dv, want["dv"], size * rel + ref.half_step(BF16) * want["dv"].abs(), "dv")
