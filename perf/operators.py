"""Timed cases of the sequence operators over octree levels: rotary positions with several axes,
attention with a sliding window and sinks, and the gated linear recurrence, each direction and type.

A level of a batched octree is one sequence per octree: its nodes lie in Morton order, octree after
octree, and `offsets` (int32 [batch + 1]) says where each begins.  Tensors are row-major, one row a
node: [rows, heads, dim] or [rows, channels].

  rotary      pair p of channels turns by the angle position[axis of p] * frequency[p]; the gradient
              is the turn back
  attention   key j of a sequence is visible to the query at position p when j <= p + right and
              (j >= p - left or j < sinks); -1 stands for no bound; the queries of a sequence are the last
              of its keys; a query that sees nothing gives zeros
  recurrence  h = a h + (1 - a) x with a = sigmoid(gate), from the first row of a sequence to its last
              (or back), starting from `state`
"""
import math

import torch

own = False

_ops = None


def _own():
  """The framework's operators (the package's name is no identifier, hence the import by name)."""
  global _ops
  if _ops is None:
    import importlib
    _ops = importlib.import_module("o-cnn_amd").nn
  return _ops


_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---- the cases ----------------------------------------------------------------------------------
def listed():
  return [
      # the new rows of eight sequences that grow by one row a step: latency, and positions far out
      {"name": "rotary_step", "op": "rotary", "rows": 8, "heads": 12, "dim": 64, "type": "bf16",
       "axes": "1", "pairs": "32", "reach": 1 << 20, "packed": False, "inverse": False, "interleaved": False},
      # queries and keys of a mid-size level at once, positions straight from the packed octree coordinates
      {"name": "rotary_level", "op": "rotary", "rows": 60001, "heads": 12, "dim": 48, "type": "bf16",
       "axes": "3", "pairs": "8,8,8", "reach": 128, "packed": True, "inverse": False, "interleaved": False},
      # the gradient on a depth-9 scene's level in fp32, with channels that carry no position
      {"name": "rotary_scene_grad", "op": "rotary", "rows": 213337, "heads": 8, "dim": 64, "type": "fp32",
       "axes": "3", "pairs": "10,10,10", "reach": 512, "packed": False, "inverse": True, "interleaved": True},
      # one new query for each of 32 sequences against all their keys: serving
      {"name": "attention_step", "op": "attention", "batch": 32, "rows": 2048, "queries": 1, "heads": 8, "kv_heads": 2,
       "dim": 64, "type": "bf16", "left": -1, "right": 0, "sinks": 0, "train": False},
      # one query against one very long sequence: few rows, a long axis
      {"name": "attention_step_long", "op": "attention", "batch": 1, "rows": 262147, "queries": 1, "heads": 16,
       "kv_heads": 2, "dim": 128, "type": "bf16", "left": -1, "right": 0, "sinks": 0, "train": False},
      # a scene's level, causal, with a window and four sinks: the large forward pass
      {"name": "attention_scene", "op": "attention", "batch": 4, "rows": 16384, "queries": 0, "heads": 8, "kv_heads": 8,
       "dim": 64, "type": "bf16", "left": 2047, "right": 0, "sinks": 4, "train": False},
      # training on a batch of 16 octrees, neighbours on both sides along the Morton order, shared key heads
      {"name": "attention_train", "op": "attention", "batch": 16, "rows": 1500, "queries": 0, "heads": 8, "kv_heads": 4,
       "dim": 64, "type": "bf16", "left": 255, "right": 256, "sinks": 4, "train": True},
      # training in the reference's precision, every node of an octree against every other
      {"name": "attention_train_fp32", "op": "attention", "batch": 8, "rows": 700, "queries": 0, "heads": 6, "kv_heads": 6,
       "dim": 32, "type": "fp32", "left": -1, "right": -1, "sinks": 0, "train": True},
      # one row a sequence from a kept state: serving
      {"name": "recurrence_step", "op": "recurrence", "batch": 64, "rows": 1, "channels": 256, "type": "bf16",
       "reverse": False, "train": False},
      # a batch of octrees at a mid level
      {"name": "recurrence_batch", "op": "recurrence", "batch": 16, "rows": 1500, "channels": 97, "type": "fp32",
       "reverse": False, "train": False},
      # a whole scene's level as one sequence
      {"name": "recurrence_scene", "op": "recurrence", "batch": 1, "rows": 262147, "channels": 256, "type": "bf16",
       "reverse": False, "train": False},
      # both directions of training, from the last node to the first
      {"name": "recurrence_train", "op": "recurrence", "batch": 8, "rows": 12000, "channels": 192, "type": "bf16",
       "reverse": True, "train": True},
  ]


def _spread(rng, lo, hi):
  """an integer between lo and hi, even over the logarithm"""
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  op = rng.choice(["rotary", "attention", "attention", "recurrence"])
  kind = rng.choice(["bf16", "bf16", "fp32"])
  if op == "rotary":
    dim = rng.choice([16, 24, 32, 40, 48, 64, 96, 128])
    axes = rng.randint(1, 3)
    packed = axes == 3 and rng.random() < 0.5
    pairs = [rng.randint(1, dim // 2 // axes) for _ in range(axes)]
    heads = rng.randint(1, 16)
    rows = _spread(rng, 1, 120000000 // (heads * dim * (4 if kind == "fp32" else 2)))
    return {"op": op, "rows": min(rows, 213337), "heads": heads, "dim": dim, "type": kind, "axes": str(axes),
            "pairs": ",".join(map(str, pairs)), "reach": 1 << rng.randint(4, 9 if packed else 20), "packed": packed,
            "inverse": rng.random() < 0.5, "interleaved": rng.random() < 0.5}
  if op == "recurrence":
    channels = _spread(rng, 8, 512)
    batch = _spread(rng, 1, 64)
    train = rng.random() < 0.5
    most = 18000000 if train else 60000000
    return {"op": op, "batch": batch, "rows": _spread(rng, 1, most // (channels * batch)), "channels": channels, "type": kind,
            "reverse": rng.random() < 0.5, "train": train}
  train = rng.random() < 0.5
  kv = rng.choice([1, 2, 3, 4])
  case = {"op": op, "heads": kv * rng.choice([1, 2, 3, 4]), "kv_heads": kv, "dim": rng.choice([16, 24, 32, 48, 64, 80, 96, 128]),
          "type": kind, "train": train, "sinks": rng.choice([0, 0, 1, 4, 16])}
  if not train and rng.random() < 0.4:            # a few new queries against many keys
    case |= {"batch": _spread(rng, 1, 48), "queries": rng.randint(1, 4), "left": rng.choice([-1, -1, _spread(rng, 16, 2048)]),
             "right": 0}
    case["rows"] = _spread(rng, 4, 120000 // case["batch"])
  else:
    two_sided = rng.random() < 0.5
    left = _spread(rng, 8, 512)
    case |= {"batch": _spread(rng, 1, 24), "queries": 0, "left": left, "right": rng.choice([left, left + 1]) if two_sided else 0}
    case["rows"] = _spread(rng, 16, (20000 if train else 40000) // case["batch"])
    if rng.random() < 0.25:
      case |= {"left": -1, "right": -1 if two_sided else 0, "sinks": 0, "rows": min(case["rows"], 900)}
  return case


# ---- lengths: one rule for every case, so that the work is known without the seed -------------------
def _lengths(case):
  """Rows of each sequence: about case["rows"] each, between a half and three halves of it; in a batch of
  three and more the second is empty and the third has one row (an octree with nothing at this level, a
  sequence just begun).  A step of single rows has one for each sequence."""
  n, rows = case["batch"], case["rows"]
  if n == 1 or rows == 1:
    return [rows] * n
  out = [max(1, int(rows * (0.5 + (b * 0.6180339887498949) % 1.0))) for b in range(n)]
  if n >= 3:
    out[1], out[2] = 0, 1
  return out


def _query_lengths(case):
  lengths = _lengths(case)
  return [min(case["queries"], k) for k in lengths] if case["queries"] else lengths


def _pairs_seen(case):
  """visible (query, key) pairs of one head"""
  total = 0
  left, right, sinks = case["left"], case["right"], case["sinks"]
  for lk, lq in zip(_lengths(case), _query_lengths(case)):
    if not lq:
      continue
    p = torch.arange(lk - lq, lk, dtype=torch.int64)
    end = torch.full_like(p, lk) if right < 0 else (p + right + 1).clamp(max=lk)
    begin = torch.zeros_like(p) if left < 0 else (p - left).clamp(min=0)
    total += int((end - begin).clamp(min=0).sum())
    total += int(torch.minimum(begin, end.clamp(max=sinks)).clamp(min=0, max=sinks).sum()) if sinks else 0
  return total


def work(case):
  e = 2 if case["type"] == "bf16" else 4
  if case["op"] == "rotary":
    n = case["rows"] * case["heads"]
    pairs = sum(map(int, case["pairs"].split(",")))
    positions = case["rows"] * (8 if case["packed"] else 4 * int(case["axes"]))
    return {"bytes": 2 * n * case["dim"] * e + positions + 8 * pairs, "flops": 6 * n * pairs}
  if case["op"] == "recurrence":
    n, state = sum(_lengths(case)) * case["channels"], 4 * case["batch"] * case["channels"]
    if case["train"]:
      return {"bytes": 6 * n * e + 4 * state, "flops": 20 * n}
    return {"bytes": 3 * n * e + 2 * state, "flops": 6 * n}
  nq, nk = sum(_query_lengths(case)) * case["heads"], sum(_lengths(case)) * case["kv_heads"]
  if case["queries"] and case["left"] >= 0:      # the rows of the cache that some query sees
    reach = case["left"] + case["queries"] + case["sinks"]
    nk = sum(min(k, reach) for k in _lengths(case)) * case["kv_heads"]
  size, flops = (2 * nq + 2 * nk) * case["dim"] * e, 4 * _pairs_seen(case) * case["heads"] * case["dim"]
  if case["train"]:
    return {"bytes": size + (2 * nq + 2 * nk) * case["dim"] * e, "flops": flops * 7 // 2}
  return {"bytes": size, "flops": flops}


# ---- inputs ---------------------------------------------------------------------------------------
def _offsets(lengths):
  return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32).cuda()


def prepare(case, seed):
  g = torch.Generator(device="cuda").manual_seed(seed)
  kind = _TYPES[case["type"]]

  def normal(*shape):
    return torch.randn(*shape, generator=g, device="cuda")

  state = {"case": case}
  if case["op"] == "rotary":
    rows, axes, reach = case["rows"], int(case["axes"]), case["reach"]
    pairs = [int(p) for p in case["pairs"].split(",")]
    state["data"] = normal(rows, case["heads"], case["dim"]).to(kind)
    pos = torch.randint(0, reach, (rows, 4 if case["packed"] else axes), generator=g, device="cuda", dtype=torch.int32)
    state["positions"] = pos.to(torch.int16).view(torch.int64).reshape(-1) if case["packed"] else pos
    state["pairs"] = pairs
    state["frequencies"] = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / n) for n in pairs]).cuda()
    return state
  lengths = _lengths(case)
  total = sum(lengths)
  state["offsets"], state["longest"] = _offsets(lengths), max(lengths)
  if case["op"] == "recurrence":
    c = case["channels"]
    # gates of a trained scan forget slowly: half-lives from a row to some hundreds of rows
    state["gate"] = (normal(total, c) * 1.5 + 2.5).to(kind)
    state["data"] = normal(total, c).to(kind)
    state["state"] = normal(case["batch"], c)
    if case["train"]:
      state["grad"] = normal(total, c).to(kind)
      state["grad_last"] = normal(case["batch"], c)
    return state
  qlen = _query_lengths(case)
  heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
  if case["queries"]:
    state["q"] = normal(sum(qlen), heads, dim).to(kind)
    state["k"], state["v"] = normal(total, kv, dim).to(kind), normal(total, kv, dim).to(kind)
    state["q_offsets"] = _offsets(qlen)
  else:                                           # slices of one projection's output
    joint = normal(total, heads + 2 * kv, dim).to(kind)
    state["q"], state["k"], state["v"] = joint[:, :heads], joint[:, heads:heads + kv], joint[:, heads + kv:]
    state["q_offsets"] = state["offsets"]
  state["q_longest"] = max(qlen)
  if case["train"]:
    state["grad"] = normal(sum(qlen), heads, dim).to(kind)
  return state


# ---- one pass ---------------------------------------------------------------------------------------
def run(state):
  return {"rotary": _rotary, "attention": _attention, "recurrence": _recurrence}[state["case"]["op"]](state)


def _rotary(s):
  case = s["case"]
  if own:
    return _own().octree_rotary(s["data"], s["positions"], s["frequencies"], s["pairs"], interleaved=case["interleaved"],
                                inverse=case["inverse"])
  pos = s["positions"]
  if case["packed"]:
    pos = pos.view(torch.int16).reshape(-1, 4)[:, :len(s["pairs"])]
  axis = torch.repeat_interleave(torch.arange(len(s["pairs"]), device=pos.device),
                                 torch.tensor(s["pairs"], device=pos.device), output_size=sum(s["pairs"]))
  angle = pos.double().index_select(1, axis) * s["frequencies"]
  if case["inverse"]:
    angle = -angle
  cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
  x, n = s["data"].float(), axis.numel()
  out = x.clone()
  if case["interleaved"]:
    a, b, to_a, to_b = x[..., 0:2 * n:2], x[..., 1:2 * n:2], out[..., 0:2 * n:2], out[..., 1:2 * n:2]
  else:
    a, b, to_a, to_b = x[..., :n], x[..., n:2 * n], out[..., :n], out[..., n:2 * n]
  to_a.copy_(a * cos - b * sin)
  to_b.copy_(a * sin + b * cos)
  return out.to(s["data"].dtype)


def _attention(s):
  case = s["case"]
  q, k, v = s["q"], s["k"], s["v"]
  if own:
    nn = _own()
    where = {"q_offsets": s["q_offsets"], "k_offsets": s["offsets"], "left": case["left"], "right": case["right"],
             "sinks": case["sinks"]}
    if not case["train"]:
      return nn.octree_attention(q, k, v, **where)
    out, lse = nn.octree_attention(q, k, v, return_lse=True, **where)
    return (out,) + tuple(nn.octree_attention_grad(s["grad"], q, k, v, out, lse, **where))
  if not case["train"]:
    return _plain_attention(s, q.float(), k.float(), v.float()).to(q.dtype)
  with torch.enable_grad():
    leaves = [t.detach().float().requires_grad_(True) for t in (q, k, v)]
    out = _plain_attention(s, *leaves)
  grads = torch.autograd.grad(out, leaves, s["grad"].float())
  return (out.detach().to(q.dtype),) + tuple(g.to(q.dtype) for g in grads)


def _plain_attention(s, q, k, v):
  case = s["case"]
  scale, share = 1.0 / math.sqrt(case["dim"]), case["heads"] // case["kv_heads"]
  if share > 1:
    k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
  if case["queries"] or case["left"] < 0:
    return _plain_padded(s, q * scale, k, v)
  return _plain_banded(s, q * scale, k, v)


def _seen(case, p, j):
  """whether key j is visible to the query at position p (tensors that broadcast)"""
  ok = torch.ones_like(p >= j) if case["right"] < 0 else j <= p + case["right"]
  return ok if case["left"] < 0 else ok & ((j >= p - case["left"]) | (j < case["sinks"]))


def _softmax(score, ok):
  score = score.masked_fill(~ok, -math.inf)
  top = score.amax(-1, keepdim=True)
  e = torch.exp(score - top.masked_fill(torch.isinf(top), 0.0))
  return e / e.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_padded(s, q, k, v):
  """every sequence padded to the longest: [batch, heads, queries, keys]"""
  case, dev = s["case"], q.device
  q0, k0 = s["q_offsets"].long(), s["offsets"].long()
  lq, lk = q0[1:] - q0[:-1], k0[1:] - k0[:-1]
  iq, ik = torch.arange(s["q_longest"], device=dev), torch.arange(s["longest"], device=dev)
  at_q, at_k = (q0[:-1, None] + iq).clamp(max=q.size(0) - 1), (k0[:-1, None] + ik).clamp(max=k.size(0) - 1)

  def batches(t, at):
    return t.index_select(0, at.reshape(-1)).reshape(*at.shape, *t.shape[1:]).transpose(1, 2).contiguous()

  p = iq + (lk - lq)[:, None]
  ok = _seen(case, p[:, :, None], ik[None, None]) & (ik < lk[:, None])[:, None]
  score = torch.matmul(batches(q, at_q), batches(k, at_k).transpose(2, 3).contiguous())
  out = torch.matmul(_softmax(score, ok[:, None]), batches(v, at_k)).transpose(1, 2)
  rows = torch.arange(q.size(0), device=dev)
  owner = (torch.searchsorted(q0, rows, right=True) - 1).clamp(max=q0.numel() - 2)
  return out.reshape(-1, *out.shape[2:]).index_select(0, owner * iq.numel() + rows - q0[owner])


def _plain_banded(s, q, k, v):
  """blocks of consecutive rows against the rows of the window around them, and every row against its sinks"""
  case, dev = s["case"], q.device
  n, left, right, sinks = q.size(0), case["left"], case["right"], case["sinks"]
  block = max(64, min(1024, left + right))
  blocks = (n + block - 1) // block
  offsets = s["offsets"].long()
  rows = torch.arange(blocks * block, device=dev)
  owner = (torch.searchsorted(offsets, rows, right=True) - 1).clamp(max=offsets.numel() - 2)
  first = offsets[owner]
  at_k = torch.arange(blocks, device=dev)[:, None] * block + torch.arange(-left, block + right, device=dev)
  inside = (at_k >= 0) & (at_k < n)
  at_k = at_k.clamp(0, n - 1)

  def blocks_of(t, at):
    return t.index_select(0, at.reshape(-1)).reshape(*at.shape, *t.shape[1:]).transpose(1, 2).contiguous()

  rows_b = rows.reshape(blocks, block)
  near = (owner.reshape(blocks, block)[:, :, None] == owner[at_k][:, None]) & inside[:, None]
  near = near & (at_k[:, None] <= rows_b[:, :, None] + right) & (at_k[:, None] >= rows_b[:, :, None] - left)
  q_b = blocks_of(q, rows_b.clamp(max=n - 1))
  score = torch.matmul(q_b, blocks_of(k, at_k).transpose(2, 3).contiguous())
  ok = near[:, None].expand_as(score)
  if sinks:
    at_s = (first[:, None] + torch.arange(sinks, device=dev))                # [rows, sinks]
    far = (at_s < (rows - left)[:, None]) & (at_s <= (rows + right)[:, None]) & (at_s < offsets[owner + 1][:, None])
    at_s = at_s.clamp(max=n - 1)
    k_s = k.index_select(0, at_s.reshape(-1)).reshape(blocks, block, sinks, *k.shape[1:]).permute(0, 3, 1, 2, 4)
    v_s = v.index_select(0, at_s.reshape(-1)).reshape(blocks, block, sinks, *v.shape[1:]).permute(0, 3, 1, 2, 4)
    score = torch.cat([score, (q_b[:, :, :, None] * k_s).sum(-1)], -1)
    ok = torch.cat([ok, far.reshape(blocks, 1, block, sinks).expand(-1, score.size(1), -1, -1)], -1)
  prob = _softmax(score, ok)
  out = torch.matmul(prob[..., :at_k.size(1)].contiguous(), blocks_of(v, at_k))
  if sinks:
    out = out + (prob[..., at_k.size(1):, None] * v_s).sum(3)
  return out.transpose(1, 2).reshape(blocks * block, *q.shape[1:])[:n]


def _recurrence(s):
  case = s["case"]
  gate, data, offsets, h0 = s["gate"], s["data"], s["offsets"], s["state"]
  if own:
    nn = _own()
    if not case["train"]:
      return nn.octree_recurrence(gate, data, offsets, state=h0, reverse=case["reverse"])
    out, last, carries = nn.octree_recurrence(gate, data, offsets, state=h0, reverse=case["reverse"], return_carries=True)
    return (out, last) + tuple(nn.octree_recurrence_grad(s["grad"], gate, data, offsets, carries, state=h0,
                                                         grad_last=s["grad_last"], reverse=case["reverse"]))
  n = data.size(0)
  at = offsets.long()
  if case["reverse"]:                                # the same from the other end
    at = (n - at).flip(0)
    gate, data, h0 = gate.flip(0), data.flip(0), h0.flip(0)
  first, end, some = at[:-1].clamp(max=max(n - 1, 0)), at[1:] - 1, (at[1:] > at[:-1])[:, None]
  a, b, x = torch.sigmoid(gate.float()), torch.sigmoid(-gate.float()), data.float()
  begins = torch.zeros(n, 1, device=x.device).index_add_(0, first, some.float()) > 0
  before = torch.zeros_like(x).index_add_(0, first, torch.where(some, h0, torch.zeros_like(h0)))
  h = _scan(a.masked_fill(begins, 0.0), b * x + a * before, s["longest"])
  last = torch.where(some, h.index_select(0, end.clamp(min=0)), h0)
  if not case["train"]:
    out = h.to(data.dtype)
    return (out.flip(0), last.flip(0)) if case["reverse"] else (out, last)
  dy, dlast = s["grad"].float(), s["grad_last"]
  if case["reverse"]:
    dy, dlast = dy.flip(0), dlast.flip(0)
  dy = dy.index_add(0, end.clamp(min=0), torch.where(some, dlast, torch.zeros_like(dlast)))
  after = torch.cat([a[1:].masked_fill(begins[1:], 0.0), torch.zeros_like(a[:1])])
  lam = _scan(after.flip(0), dy.flip(0), s["longest"]).flip(0)
  prev = torch.where(begins, before, torch.cat([torch.zeros_like(h[:1]), h[:-1]]))
  dgate, ddata = lam * (prev - x) * a * b, lam * b
  dstate = torch.where(some, (a * lam).index_select(0, first), dlast)
  outs = [h.to(data.dtype), last, dgate.to(data.dtype), ddata.to(data.dtype), dstate]
  return tuple(t.flip(0) for t in outs) if case["reverse"] else tuple(outs)


def _scan(a, b, longest):
  """h[t] = a[t] h[t - 1] + b[t] over the first axis, by doubling"""
  step = 1
  while step < longest:
    b = torch.cat([b[:step], b[step:] + a[step:] * b[:-step]])
    a = torch.cat([a[:step], a[step:] * a[:-step]])
    step *= 2
  return b


# ---- the definitions in 64 bits ---------------------------------------------------------------------
def exact(case, seed):
  s = prepare(case, seed)
  return {"rotary": _exact_rotary, "attention": _exact_attention, "recurrence": _exact_recurrence}[case["op"]](s)


def _exact_rotary(s):
  case, x = s["case"], s["data"].double()
  pos = s["positions"]
  if case["packed"]:
    pos = torch.stack([(pos >> (16 * i)) & 0xFFFF for i in range(3)], 1)
  n, p = sum(s["pairs"]), 0
  out = x.clone()
  for axis, count in enumerate(s["pairs"]):
    for _ in range(count):
      t = pos[:, axis, None].double() * s["frequencies"][p] * (-1.0 if case["inverse"] else 1.0)
      i, j = (2 * p, 2 * p + 1) if case["interleaved"] else (p, n + p)
      turned = torch.polar(torch.ones_like(t), t) * torch.complex(x[:, :, i], x[:, :, j])
      out[:, :, i], out[:, :, j] = turned.real, turned.imag
      p += 1
  return out


def _exact_attention(s):
  """sequence by sequence, some hundred queries at a time; the gradient by its formulas"""
  case = s["case"]
  q, k, v = (s[n].double() for n in "qkv")
  heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
  scale = dim ** -0.5
  out = torch.zeros_like(q)
  dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
  qo, ko = s["q_offsets"].tolist(), s["offsets"].tolist()
  group = torch.arange(heads, device=q.device) // (heads // kv)
  for b in range(case["batch"]):
    lq, lk = qo[b + 1] - qo[b], ko[b + 1] - ko[b]
    step = 512
    for i in range(0, lq, step):
      m = min(step, lq - i)
      p = torch.arange(i, i + m, device=q.device) + lk - lq
      hi = lk if case["right"] < 0 else min(lk, int(p[-1]) + 1 + case["right"])
      lo = 0 if case["left"] < 0 else max(0, int(p[0]) - case["left"])
      j = torch.arange(lo, hi, device=q.device)
      if lo and case["sinks"]:
        j = torch.cat([torch.arange(min(case["sinks"], lo, hi), device=q.device), j])
      if not j.numel():
        continue
      here = slice(qo[b] + i, qo[b] + i + m)
      qb = q[here].transpose(0, 1).contiguous()
      kb = k[ko[b] + j].transpose(0, 1)[group].contiguous()
      vb = v[ko[b] + j].transpose(0, 1)[group].contiguous()
      hidden = torch.zeros(m, j.numel(), dtype=torch.bool, device=q.device)
      if case["right"] >= 0:
        hidden |= j[None] > p[:, None] + case["right"]
      if case["left"] >= 0:
        hidden |= (j[None] < p[:, None] - case["left"]) & (j[None] >= case["sinks"])
      e = torch.bmm(qb, kb.transpose(1, 2).contiguous()) * scale
      e = torch.where(hidden, torch.full_like(e, -1e300), e)
      e = torch.exp(e - e.max(-1, keepdim=True)[0])
      e = torch.where(hidden, torch.zeros_like(e), e)
      norm = e.sum(-1, keepdim=True)
      prob = torch.where(norm > 0, e / norm, torch.zeros_like(e))
      ob = torch.bmm(prob, vb)
      out[here] = ob.transpose(0, 1)
      if case["train"]:
        go = s["grad"][here].double().transpose(0, 1).contiguous()
        ds = prob * (torch.bmm(go, vb.transpose(1, 2).contiguous()) - (go * ob).sum(-1, keepdim=True)) * scale
        dq[here] = torch.bmm(ds, kb).transpose(0, 1)
        dkb = torch.bmm(ds.transpose(1, 2).contiguous(), qb).reshape(kv, heads // kv, -1, dim).sum(1)
        dvb = torch.bmm(prob.transpose(1, 2).contiguous(), go).reshape(kv, heads // kv, -1, dim).sum(1)
        dk[ko[b] + j] += dkb.transpose(0, 1)
        dv[ko[b] + j] += dvb.transpose(0, 1)
  return (out, dq, dk, dv) if case["train"] else out


def _walk(a, b):
  """h[t] = a[t] h[t - 1] + b[t]: rows of a block one after another, all blocks at once, then the blocks in order"""
  n, c = a.shape
  size = max(1, min(512, int(n ** 0.5)))
  blocks = (n + size - 1) // size
  a = torch.cat([a, a.new_zeros(blocks * size - n, c)]).reshape(blocks, size, c)
  h = torch.cat([b, b.new_zeros(blocks * size - n, c)]).reshape(blocks, size, c).clone()
  grown = a.clone()
  for t in range(1, size):
    h[:, t] += a[:, t] * h[:, t - 1]
    grown[:, t] *= grown[:, t - 1]
  for i in range(1, blocks):
    h[i] += grown[i] * h[i - 1, -1]
  return h.reshape(-1, c)[:n]


def _exact_recurrence(s):
  case = s["case"]
  turn = (lambda t: t.flip(0)) if case["reverse"] else (lambda t: t)
  g, x, h0 = turn(s["gate"].double()), turn(s["data"].double()), turn(s["state"].double())
  n, ends = x.size(0), s["offsets"].tolist()
  lengths = [ends[i + 1] - ends[i] for i in range(len(ends) - 1)]
  if case["reverse"]:
    lengths = lengths[::-1]
  a, b = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
  seqs, at = [], 0
  for i, m in enumerate(lengths):
    if m:
      seqs.append((i, at, at + m - 1))
    at += m
  which, begin, end = (torch.tensor(t, device=x.device) for t in zip(*seqs))
  open_, drive = a.clone(), b * x
  open_[begin] = 0
  drive[begin] += a[begin] * h0[which]
  h = _walk(open_, drive)
  last = h0.clone()
  last[which] = h[end]
  if not case["train"]:
    return turn(h), turn(last)
  dlast = turn(s["grad_last"].double())
  dy = turn(s["grad"].double()).clone()
  dy[end] += dlast[which]
  later = torch.zeros_like(open_)
  later[:-1] = open_[1:]
  lam = _walk(later.flip(0), dy.flip(0)).flip(0)
  prev = torch.zeros_like(h)
  prev[1:] = h[:-1]
  prev[begin] = h0[which]
  dstate = dlast.clone()
  dstate[which] = (a * lam)[begin]
  return turn(h), turn(last), turn(a * b * lam * (prev - x)), turn(b * lam), turn(dstate)
