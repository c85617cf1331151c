"""Operators along the node order of an octree level (rotary positions, attention with a window and sinks, the gated
linear recurrence) against plain implementations in 64 bits (sequence_reference.py, where the tolerances are
derived), at the sizes, masks and layouts where they can go wrong."""
import numpy as np
import pytest
import torch

import sequence_reference as ref
from oracle.checker import OctreeBlob, make_points_blob

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
TYPES = [F32, BF16]


def ids(x):
  return str(x).split(".")[-1] if isinstance(x, torch.dtype) else None


def gen(seed):
  return torch.Generator().manual_seed(seed)


def offs(lengths):
  return torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int32)


def within(got, want, tol, what=""):
  got, want, tol = got.double().cpu(), want.double(), torch.as_tensor(tol, dtype=torch.float64).expand_as(want)
  assert got.shape == want.shape, what
  fine = torch.isfinite(want)
  assert torch.equal(torch.isnan(got), torch.isnan(want)), "%s: NaN elsewhere than in the reference" % what
  odd = ~fine & ~torch.isnan(want)
  assert torch.equal(got[odd], want[odd]), what
  err = (got - want).abs()[fine] - tol[fine] - 1e-30
  assert err.numel() == 0 or float(err.max()) <= 0, "%s: %g over the bound (error %g)" % (
      what, float(err.max()), float((got - want).abs()[fine].max()))


# ---- octree_offsets ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("nempty", [False, True])
def test_offsets_of_a_batch(oc, orc, synthetic, nempty):
  pbs = [make_points_blob(*synthetic.shape_cloud(n, 40 + i)[:2]) for i, n in enumerate((900, 30, 2500, 1))]
  host = orc.octree_batch([orc.points2octree(p, 6, 2) for p in pbs])
  blob, dev = OctreeBlob(host), torch.from_numpy(host).cuda()
  for depth in range(1, 7):
    key = blob.prop("key", depth).view(np.uint64).reshape(-1)
    child = blob.prop("child", depth).reshape(-1)
    owner = (key >> np.uint64(48)).astype(int)
    if nempty:
      owner = owner[child >= 0]
    want = np.searchsorted(owner, np.arange(5))
    got = oc.nn.octree_offsets(dev, depth, nempty)
    assert got.dtype == torch.int32 and got.tolist() == want.tolist(), depth
    assert got[-1] == (blob.nnum_nempty[depth] if nempty else blob.nnum[depth])
  with pytest.raises(oc.nn.OcnnError):
    oc.nn.octree_offsets(dev, 7)
  single = torch.from_numpy(orc.points2octree(pbs[0], 5, 2)).cuda()
  n = oc.nn.octree_info(single).nnum(5)
  assert oc.nn.octree_offsets(single, 5).tolist() == [0, n]


# ---- rotary positions ---------------------------------------------------------------------------------------
ROTARY = [
    # rows, heads, dim, pairs, reach
    (1, 1, 8, [4], 10), (7, 3, 16, [3, 2, 1], 100), (33, 12, 64, [32], 1 << 20), (130, 5, 48, [8, 8, 8], 512),
    (65, 2, 6, [1, 1], 50), (19, 1, 7, [3], 9), (40, 4, 128, [20, 20, 11, 13], 1 << 30), (9, 2, 30, [5, 0, 7], 300),
    (3, 130, 20, [10], 40), (517, 1, 24, [0], 5), (5, 2, 1024, [512], 1 << 16),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: "%dx%dx%d-%s" % (c[0], c[1], c[2], "+".join(map(str, c[3]))))
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_rotary(oc, dtype, case, interleaved):
  rows, heads, dim, pairs, reach = case
  g = gen(rows * dim)
  x = torch.randn(rows, heads, dim, generator=g).to(dtype)
  freq = oc.nn.rotary_frequencies(pairs, device="cpu")
  pos = torch.randint(-reach, reach, (rows, len(pairs)), generator=g, dtype=torch.int32)
  kinds = [("int32", pos, pos)]
  frac = pos.float() + 0.37
  kinds.append(("float32", frac, frac.double()))
  if len(pairs) <= 3 and reach <= 1 << 16:
    whole = torch.randint(0, min(2 * reach, 1 << 16), (rows, 4), generator=g)
    packed = sum(whole[:, i] << (16 * i) for i in range(3)) | ((whole[:, 3] % 7) << 48)
    kinds.append(("packed", packed, whole))
  for inverse in (False, True):
    for name, p, plain in kinds:
      want, size = ref.rotary(x, plain, freq, pairs, interleaved, inverse)
      got = oc.nn.octree_rotary(x.cuda(), p.cuda(), freq.cuda(), pairs, interleaved=interleaved, inverse=inverse)
      assert got.dtype == dtype
      # sine and cosine off by 2^-22 (the fraction of a turn is rounded to 32 bits: pi 2^-24, the functions to two
      # steps), the 64-bit angle by its own step, two products and a sum in 32 bits, and the result's rounding
      angle = 4.0 * float(plain.abs().max() if rows else 0) * 2.0 ** -52
      within(got, want, size * (2.0 ** -21 + angle) + ref.half_step(dtype) * want.abs(), "%s inverse=%s" % (name, inverse))
      n = 2 * sum(pairs)
      assert torch.equal(got[..., n:].cpu(), x[..., n:])


def test_rotary_layouts_and_in_place(oc):
  g = gen(3)
  joint = torch.randn(70, 9, 40, generator=g).to(BF16).cuda()
  pos = torch.randint(0, 300, (70, 5), generator=g, dtype=torch.int32).cuda()
  freq = oc.nn.rotary_frequencies([5, 6, 7])
  want = oc.nn.octree_rotary(joint[:, :6].contiguous(), pos[:, :3].contiguous(), freq, [5, 6, 7])
  assert torch.equal(oc.nn.octree_rotary(joint[:, :6], pos[:, :3], freq, [5, 6, 7]), want)
  # rows and heads that begin anywhere, a transposed view, every second head
  odd = torch.empty(70 * 6 * 41 + 1, dtype=BF16, device="cuda")[1:].view(70, 6, 41)[:, :, :40]
  odd.copy_(joint[:, :6])
  assert torch.equal(oc.nn.octree_rotary(odd, pos[:, :3], freq, [5, 6, 7]), want)
  turned = joint[:, :6].permute(1, 0, 2).contiguous().permute(1, 0, 2)
  assert torch.equal(oc.nn.octree_rotary(turned, pos[:, :3], freq, [5, 6, 7]), want)
  last = joint[:, :6].permute(0, 2, 1).contiguous().permute(0, 2, 1)
  assert torch.equal(oc.nn.octree_rotary(last, pos[:, :3], freq, [5, 6, 7]), want)
  assert torch.equal(oc.nn.octree_rotary(joint[:, :6:2], pos[:, :3], freq, [5, 6, 7]), want[:, ::2])
  # in place on a slice: the rest of the joint tensor stays
  keep = joint.clone()
  got = oc.nn.octree_rotary(joint[:, :6], pos[:, :3], freq, [5, 6, 7], out=joint[:, :6])
  assert torch.equal(got, want) and torch.equal(joint[:, :6], want) and torch.equal(joint[:, 6:], keep[:, 6:])
  # into rows of another tensor
  room = torch.full((70, 8, 48), 7.0, dtype=BF16, device="cuda")
  oc.nn.octree_rotary(keep[:, :6], pos[:, :3], freq, [5, 6, 7], out=room[:, 1:7, 4:44])
  assert torch.equal(room[:, 1:7, 4:44], want)
  room[:, 1:7, 4:44] = 7.0
  assert bool((room == 7.0).all())
  assert oc.nn.octree_rotary(joint[:0], pos[:0, :3], freq, [5, 6, 7]).shape == (0, 9, 40)


def test_rotary_turns_back(oc):
  """the inverse is the gradient: <R x, y> = <x, R^-1 y>, and R^-1 R x = x"""
  g = gen(4)
  x, y = (torch.randn(200, 4, 32, generator=g).cuda() for _ in range(2))
  pos = torch.randint(0, 1 << 20, (200, 2), generator=g, dtype=torch.int32).cuda()
  freq = oc.nn.rotary_frequencies([8, 8])
  for inter in (False, True):
    kw = dict(interleaved=inter)
    rx = oc.nn.octree_rotary(x, pos, freq, [8, 8], **kw)
    back = oc.nn.octree_rotary(rx, pos, freq, [8, 8], inverse=True, **kw)
    within(back, x.double().cpu(), 2.0 ** -19 * x.double().abs().amax().cpu())
    ry = oc.nn.octree_rotary(y, pos, freq, [8, 8], inverse=True, **kw)
    a, b = (rx.double() * y.double()).sum(), (x.double() * ry.double()).sum()
    assert abs(float(a - b)) < 2.0 ** -20 * float((x.double().abs() * y.double().abs()).sum() * 2)


# ---- recurrence ---------------------------------------------------------------------------------------------
RECURRENCE = [
    # lengths, channels
    ([1], 1), ([5, 0, 1, 17], 8), ([64, 64, 1], 24), ([129], 97), ([0, 0, 3], 5), ([16] * 40, 33), ([1] * 70, 64),
    ([1000, 3, 0, 777], 12), ([63, 65, 127, 128, 129], 7),
]


def recurrence_inputs(lengths, channels, dtype, seed, extra=0):
  g = gen(seed)
  n = sum(lengths) + extra
  gate = (torch.randn(n, channels, generator=g) * 2 + 2).to(dtype)
  data = torch.randn(n, channels, generator=g).to(dtype)
  state = torch.randn(len(lengths), channels, generator=g)
  return gate, data, state, torch.randn(n, channels, generator=g).to(dtype), torch.randn(len(lengths), channels, generator=g)


def check_recurrence(oc, dtype, lengths, channels, reverse, with_state, seed=5, extra=0):
  gate, data, state, dy, dl = recurrence_inputs(lengths, channels, dtype, seed, extra)
  if not with_state:
    state, dl = None, None
  o = offs(lengths)
  cuda = lambda t: None if t is None else t.cuda()   # noqa: E731
  want = ref.recurrence(gate, data, o, state, reverse, dy, dl)
  tol = ref.recurrence_tolerance(gate, data, state, dtype, max(lengths))
  u = ref.half_step(dtype)
  out, last = oc.nn.octree_recurrence(gate.cuda(), data.cuda(), o.cuda(), cuda(state), reverse)
  out2, last2, carries = oc.nn.octree_recurrence(gate.cuda(), data.cuda(), o.cuda(), cuda(state), reverse, return_carries=True)
  for y, e in ((out, last), (out2, last2)):
    within(y, want["out"], tol + u * want["out"].abs(), "out")
    within(e, want["last"], tol, "last")
  dg, dx, ds = oc.nn.octree_recurrence_grad(dy.cuda(), gate.cuda(), data.cuda(), o.cuda(), carries, cuda(state), cuda(dl), reverse)
  # the gradient runs the same recurrence backwards over dh: its error is bounded the same way, and h - x adds h's
  back = ref.recurrence_tolerance(gate, dy, dl, dtype, max(lengths))
  b_min = float(torch.sigmoid(-gate.double()).min())
  grow = back * min(max(lengths), 1 / b_min)          # (a dh is not scaled by 1 - a: the sum of up to 1 / (1 - a) of them)
  lam = float(want["ddata"].abs().max() / b_min) if dx.numel() else 0.0
  big = 2 * max(float(data.double().abs().max()), 1.0 if state is None else float(state.abs().max()))
  within(dx, want["ddata"], grow + u * want["ddata"].abs(), "ddata")
  within(dg, want["dgate"], grow * big + min(lam, 100.0) * tol + u * want["dgate"].abs(), "dgate")
  within(ds, want["dstate"], grow, "dstate")


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("case", RECURRENCE, ids=lambda c: "%s-%d" % ("+".join(map(str, c[0][:5])), c[1]))
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_recurrence(oc, dtype, case, reverse):
  check_recurrence(oc, dtype, case[0], case[1], reverse, True)
  check_recurrence(oc, dtype, case[0], case[1], reverse, False, seed=6, extra=11)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_recurrence_with_long_chunks(oc, dtype):
  """sizes that take several channels a thread, and lists of chunks in two launches"""
  check_recurrence(oc, dtype, [9000, 0, 1, 7777, 300], 256, False, True)
  check_recurrence(oc, dtype, [17003], 250, True, True)


def test_recurrence_rows_of_no_sequence(oc):
  gate, data, state, dy, _ = recurrence_inputs([30, 12], 20, BF16, 8, extra=25)
  o = offs([30, 12]).cuda()
  room = torch.full((67, 24), 3.0, dtype=BF16, device="cuda")
  for reverse in (False, True):
    for carries in (False, True):
      full = oc.nn.octree_recurrence(gate.cuda(), data.cuda(), o, state.cuda(), reverse, return_carries=carries)
      assert bool((full[0][42:] == 0).all())
      room.fill_(3.0)
      part = oc.nn.octree_recurrence(gate.cuda(), data.cuda(), o, state.cuda(), reverse, out=room[:, 2:22], return_carries=carries)
      assert torch.equal(room[:42, 2:22], full[0][:42]) and torch.equal(part[1], full[1])
      room[:42, 2:22] = 3.0
      assert bool((room == 3.0).all())
    grads = oc.nn.octree_recurrence_grad(dy.cuda(), gate.cuda(), data.cuda(), o, full[2], state.cuda(), None, reverse)
    assert bool((grads[0][42:] == 0).all()) and bool((grads[1][42:] == 0).all())


def test_recurrence_extreme_gates(oc):
  """gates that close, open, are infinite or far apart; a NaN stays in its sequence and channel"""
  g = torch.tensor([[-1e4, 1e4, 0.0, 80.0, -80.0, float("inf"), float("-inf"), 120.0]]).repeat(40, 1)
  x = torch.randn(40, 8, generator=gen(1))
  o = offs([25, 15])
  for dtype in TYPES:
    want = ref.recurrence(g.to(dtype), x.to(dtype), o)
    out, _ = oc.nn.octree_recurrence(g.to(dtype).cuda(), x.to(dtype).cuda(), o.cuda())
    within(out, want["out"], 2.0 ** -18 * 4 + ref.half_step(dtype) * want["out"].abs())
  x[10, 3] = float("nan")
  want = ref.recurrence(torch.zeros(40, 8), x, o)
  for kw in ({}, {"return_carries": True}):
    out = oc.nn.octree_recurrence(torch.zeros(40, 8).cuda(), x.cuda(), o.cuda(), **kw)[0]
    within(out, want["out"], 2.0 ** -18 * 4)


def test_recurrence_gradient_where_nothing_changes(oc):
  """constant data: h - x shrinks to nothing, and the gradient of the gate with it (a rounded h would leave 2^-9)"""
  x = torch.full((300, 4), 1.7).to(BF16)
  gate = torch.full((300, 4), 1.0).to(BF16)
  dy = torch.randn(300, 4, generator=gen(2)).to(BF16)
  o = offs([300])
  want = ref.recurrence(gate, x, o, None, False, dy)
  out, _, carries = oc.nn.octree_recurrence(gate.cuda(), x.cuda(), o.cuda(), return_carries=True)
  dg = oc.nn.octree_recurrence_grad(dy.cuda(), gate.cuda(), x.cuda(), o.cuda(), carries)[0]
  within(dg, want["dgate"], 2.0 ** -18 * float(dy.abs().max()) * 4 + ref.half_step(BF16) * want["dgate"].abs())


def test_recurrence_step_continues_a_sequence(oc):
  """a sequence in one call, in two, and row by row from the kept state"""
  gate, data, _, _, _ = recurrence_inputs([50, 50], 16, F32, 9)
  o = offs([50, 50]).cuda()
  whole, end = oc.nn.octree_recurrence(gate.cuda(), data.cuda(), o)
  g, x = gate.view(2, 50, 16).cuda(), data.view(2, 50, 16).cuda()
  rows, state, one = [], None, offs([1, 1]).cuda()
  for t in range(50):
    y, state = oc.nn.octree_recurrence(g[:, t].contiguous(), x[:, t].contiguous(), one, state)
    rows.append(y)
  got = torch.stack(rows, 1).reshape(100, 16)
  within(got, whole.double().cpu(), 2.0 ** -17)
  within(state, end.double().cpu(), 2.0 ** -17)


def test_recurrence_strided_inputs(oc):
  joint = torch.randn(90, 3, 20, generator=gen(6)).to(BF16).cuda()
  o = offs([40, 50]).cuda()
  a = oc.nn.octree_recurrence(joint[:, 0].contiguous(), joint[:, 2].contiguous(), o)
  b = oc.nn.octree_recurrence(joint[:, 0], joint[:, 2], o)
  assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
  odd = torch.empty(90 * 21 + 1, dtype=BF16, device="cuda")[1:].view(90, 21)[:, :20]
  odd.copy_(joint[:, 0])
  c = oc.nn.octree_recurrence(odd, joint[:, 2].t().contiguous().t(), o)
  assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


# ---- attention ------------------------------------------------------------------------------------------------
def attention_inputs(qlen, klen, heads, kvh, dim, dtype, seed, q_extra=0, k_extra=0):
  g = gen(seed)
  r = lambda n, h: torch.randn(n, h, dim, generator=g).to(dtype)   # noqa: E731
  return (r(sum(qlen) + q_extra, heads), r(sum(klen) + k_extra, kvh), r(sum(klen) + k_extra, kvh),
          r(sum(qlen) + q_extra, heads))


def check_attention(oc, dtype, q, k, v, go, qo, ko, backward=True, **kw):
  want = ref.attention(q, k, v, qo, ko, grad=go if backward else None, dtype=dtype, **kw)
  dev = {n: (x.cuda() if torch.is_tensor(x) else x) for n, x in kw.items()}
  out, lse = oc.nn.octree_attention(q.cuda(), k.cuda(), v.cuda(), qo.cuda(), ko.cuda(), return_lse=True, **dev)
  assert torch.equal(out, oc.nn.octree_attention(q.cuda(), k.cuda(), v.cuda(), qo.cuda(), ko.cuda(), **dev))
  within(out, want["out"], want["out_tol"], "out")
  within(lse, want["lse"], want["lse_tol"], "lse")
  if not backward:
    return out, lse
  grads = oc.nn.octree_attention_grad(go.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse, qo.cuda(), ko.cuda(), **dev)
  for n, g in zip(("dq", "dk", "dv"), grads):
    assert g.dtype == dtype
    within(g, want[n], want[n + "_tol"], n)
  return out, lse, grads


SELF = [
    # lengths, heads, kv heads, dim, window
    ([1], 1, 1, 8, {}),
    ([5, 0, 1, 33], 4, 2, 16, {}),
    ([70, 3], 2, 2, 24, dict(right=0)),
    ([64, 64, 64], 2, 1, 32, dict(left=10, right=10)),
    ([129, 1, 0, 260], 3, 3, 40, dict(left=31, right=0)),
    ([300], 6, 2, 64, dict(left=16, right=0, sinks=4)),
    ([257, 40], 4, 4, 64, dict(left=0, right=0)),
    ([400, 130], 2, 1, 72, dict(left=50, right=20, sinks=3)),
    ([150], 5, 1, 80, dict(left=-1, right=3)),
    ([90, 200], 3, 1, 96, dict(left=7, right=-1, sinks=64)),
    ([140], 2, 2, 128, dict(left=40, right=1, sinks=1)),
    ([700], 2, 1, 16, dict(left=5, right=5, sinks=17)),
]


@pytest.mark.parametrize("case", SELF, ids=lambda c: "%s-%dx%dx%d-%s" % (
    "+".join(map(str, c[0])), c[1], c[2], c[3], "".join("%s%d" % (n[0], x) for n, x in c[4].items())))
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_and_its_gradient(oc, dtype, case):
  lengths, heads, kvh, dim, window = case
  q, k, v, go = attention_inputs(lengths, lengths, heads, kvh, dim, dtype, 11)
  check_attention(oc, dtype, q, k, v, go, offs(lengths), offs(lengths), **window)


CROSS = [
    # query lengths, key lengths, heads, kv heads, dim, window: few queries, more queries than keys, none of either
    ([1, 1, 1], [50, 1, 200], 8, 2, 64, dict(right=0)),
    ([1, 2, 0, 3], [300, 40, 9, 0], 4, 1, 128, dict(left=20, right=0, sinks=2)),
    ([10, 4], [3, 4], 2, 2, 32, dict(right=0)),
    ([10, 4], [3, 4], 2, 2, 32, dict(left=2, right=1, sinks=1)),
    ([150, 7], [20, 400], 3, 1, 48, dict(left=30, right=-1)),
    ([33, 0], [0, 65], 2, 1, 16, {}),
    ([3], [2100], 12, 3, 96, dict(left=-1, right=0)),
    ([200], [3000], 2, 1, 64, dict(left=-1, right=0)),
    ([200], [3000], 2, 1, 64, dict(left=700, right=0, sinks=5)),
]


@pytest.mark.parametrize("case", CROSS, ids=lambda c: "%s-of-%s-%dx%dx%d" % (
    "+".join(map(str, c[0])), "+".join(map(str, c[1])), c[2], c[3], c[4]))
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_queries_at_the_end_of_their_keys(oc, dtype, case):
  qlen, klen, heads, kvh, dim, window = case
  q, k, v, go = attention_inputs(qlen, klen, heads, kvh, dim, dtype, 12)
  check_attention(oc, dtype, q, k, v, go, offs(qlen), offs(klen), **window)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_split_keys(oc, dtype):
  """long key axes that are dealt out over workgroups, for few rows and for a tile of them; ragged, some empty"""
  for qlen, klen, heads, kvh, dim, window in (
      ([1], [9000], 4, 2, 64, dict(right=0)),
      ([1, 1, 1], [6000, 0, 31], 4, 4, 128, dict(right=0)),
      ([2, 1], [5000, 2000], 6, 2, 24, dict(left=1500, right=0, sinks=7)),
      ([100], [6000], 2, 1, 32, dict(right=0))):
    q, k, v, go = attention_inputs(qlen, klen, heads, kvh, dim, dtype, 13, q_extra=2)
    out, lse = check_attention(oc, dtype, q, k, v, go, offs(qlen), offs(klen), backward=False, **window)
    assert bool((out[sum(qlen):] == 0).all()) and bool(torch.isinf(lse[sum(qlen):]).all())
    room = torch.full_like(out, 5.0)
    oc.nn.octree_attention(q.cuda(), k.cuda(), v.cuda(), offs(qlen).cuda(), offs(klen).cuda(), out=room, **window)
    assert torch.equal(room[:sum(qlen)], out[:sum(qlen)]) and bool((room[sum(qlen):] == 5.0).all())


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_key_mask(oc, dtype):
  """masked keys (whole sequences of them too) that hold infinities and NaN"""
  lengths = [90, 40, 130]
  q, k, v, go = attention_inputs(lengths, lengths, 4, 2, 48, dtype, 14)
  mask = torch.rand(260, generator=gen(1)) < 0.6
  mask[90:130] = False
  mask[130:140] = False
  k[~mask] = float("nan")
  v[~mask] = float("inf")
  for window in ({}, dict(left=9, right=0, sinks=12), dict(left=3, right=4)):
    out, lse, grads = check_attention(oc, dtype, q, k, v, go, offs(lengths), offs(lengths), key_mask=mask, **window)
    assert bool((out[90:130] == 0).all()) and bool(torch.isinf(lse[90:130]).all())
    assert bool((grads[1][~mask.cuda()] == 0).all()) and bool((grads[2][~mask.cuda()] == 0).all())


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_cache_with_room(oc, dtype):
  """key rows behind k_lengths hold NaN, the last sequence's end lies before the rows' end"""
  room, keys, qlen = [64, 200, 7, 130], [50, 200, 0, 101], [1, 3, 2, 1]
  q, k, v, go = attention_inputs(qlen, room, 6, 3, 64, dtype, 15, q_extra=4, k_extra=70)
  ko = offs(room)
  live = torch.zeros(k.size(0), dtype=torch.bool)
  for a, n in zip(ko.tolist(), keys):
    live[a:a + n] = True
  k[~live] = float("nan")
  v[~live] = float("nan")
  lens = torch.tensor(keys, dtype=torch.int32)
  for window in (dict(right=0), dict(left=30, right=0, sinks=2)):
    out, lse, grads = check_attention(oc, dtype, q, k, v, go, offs(qlen), ko, k_lengths=lens, **window)
    assert bool((out[7:] == 0).all()) and bool((grads[0][7:] == 0).all())
    assert bool((grads[1][~live.cuda()] == 0).all()) and bool((grads[2][~live.cuda()] == 0).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_bad_values_stay_with_the_rows_that_see_them(oc, dtype, bad):
  """one value row and one query row that are not finite: rows outside their window, in the same tiles, are right"""
  lengths = [200, 60]
  window = dict(left=12, right=3, sinks=2)
  for few in (False, True):
    qlen = [6, 4] if few else lengths
    q, k, v, go = attention_inputs(qlen, lengths, 2, 1, 32, dtype, 16)
    v[150] = bad
    k[20, 0, 3] = bad
    out, lse = oc.nn.octree_attention(q.cuda(), k.cuda(), v.cuda(), offs(qlen).cuda(), offs(lengths).cuda(), return_lse=True,
                                      **window)
    grads = oc.nn.octree_attention_grad(go.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse, offs(qlen).cuda(),
                                        offs(lengths).cuda(), **window)
    # the rows that see one of them
    hit_q = torch.zeros(q.size(0), dtype=torch.bool)
    hit_k = torch.zeros(k.size(0), dtype=torch.bool)
    for (qa, qb), (ka, kb) in zip(ref.spans(offs(qlen)), ref.spans(offs(lengths))):
      ok = ref.visible(qb - qa, kb - ka, **window)
      poor = torch.zeros(kb - ka, dtype=torch.bool)
      for row in (150, 20):
        if ka <= row < kb:
          poor[row - ka] = True
      hit = (ok & poor[None]).any(1)
      hit_q[qa:qb] = hit
      hit_k[ka:kb] = (ok & hit[:, None]).any(0)
    assert few or hit_q.any()
    assert not hit_q.all() and not hit_k.all()
    v[150], k[20] = 0, 0
    want = ref.attention(q, k, v, offs(qlen), offs(lengths), grad=go, dtype=dtype, **window)
    for n, g, hit in (("out", out, hit_q), ("lse", lse, hit_q), ("dq", grads[0], hit_q), ("dk", grads[1], hit_k),
                      ("dv", grads[2], hit_k)):
      within(g[~hit.cuda()], want[n][~hit], want[n + "_tol"][~hit], n)
    if not few and bad != bad:
      # (an infinite key gives a query with the other sign the score -inf: probability 0, a finite row)
      assert not torch.isfinite(out.float().sum((1, 2)))[hit_q.cuda()].any()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_large_scores(oc, dtype):
  """scores in the thousands and the lowest finite values: no overflow, the softmax is one-hot"""
  lengths = [100, 30]
  q, k, v, go = attention_inputs(lengths, lengths, 2, 2, 32, dtype, 17)
  q, k = q * 40, k * 40
  check_attention(oc, dtype, q, k, v, go, offs(lengths), offs(lengths), left=60, right=60)
  low = torch.finfo(dtype).min
  k2 = torch.zeros_like(k)
  k2[::2, :, 0] = low / 64
  q2 = torch.zeros_like(q)
  q2[..., 0] = 1.0
  check_attention(oc, dtype, q2, k2, v, go, offs(lengths), offs(lengths), backward=False, left=60, right=60, scale=1.0)
  # negative and zero scales
  check_attention(oc, dtype, q / 40, k / 40, v, go, offs(lengths), offs(lengths), right=0, scale=-0.3)
  check_attention(oc, dtype, q, k, v, go, offs(lengths), offs(lengths), right=0, scale=0.0)


def test_attention_layouts(oc):
  """slices of one projection, transposed heads, rows that begin off 16 bytes, an output inside a larger tensor"""
  lengths = [120, 77]
  o = offs(lengths).cuda()
  kw = dict(left=20, right=2, sinks=1)
  joint = torch.randn(197, 10, 40, generator=gen(18)).to(BF16).cuda()
  q, k, v = joint[:, :6], joint[:, 6:8], joint[:, 8:]
  want, lse = oc.nn.octree_attention(q.contiguous(), k.contiguous(), v.contiguous(), o, return_lse=True, **kw)
  go = torch.randn(197, 6, 40, generator=gen(19)).to(BF16).cuda()
  want_g = oc.nn.octree_attention_grad(go, q.contiguous(), k.contiguous(), v.contiguous(), want, lse, o, **kw)
  heads_first = [t.permute(1, 0, 2).contiguous().permute(1, 0, 2) for t in (q, k, v)]
  odd = torch.empty(197 * 6 * 41 + 1, dtype=BF16, device="cuda")[1:].view(197, 6, 41)[:, :, :40]
  odd.copy_(q)
  for a, b, c in ((q, k, v), heads_first, (odd, k, v)):
    assert torch.equal(oc.nn.octree_attention(a, b, c, o, **kw), want)
    got = oc.nn.octree_attention_grad(go.transpose(0, 1).contiguous().transpose(0, 1), a, b, c, want, lse, o, **kw)
    assert all(torch.equal(x, y) for x, y in zip(got, want_g))
  room = torch.full((197, 8, 48), 2.0, dtype=BF16, device="cuda")
  oc.nn.octree_attention(q, k, v, o, out=room[:, 1:7, 8:48], **kw)
  assert torch.equal(room[:, 1:7, 8:48], want)
  room[:, 1:7, 8:48] = 2.0
  assert bool((room == 2.0).all())
  with pytest.raises(oc.nn.OcnnError, match="overlaps an input"):
    oc.nn.octree_attention(q, k, v, o, out=q, **kw)
  with pytest.raises(oc.nn.OcnnError, match="16 bytes"):
    oc.nn.octree_attention(q, k, v, o, out=room[:, 1:7, 4:44], **kw)
  empty = oc.nn.octree_attention(q[:0], k[:0], v[:0], offs([0, 0]).cuda())
  assert empty.shape == (0, 6, 40)


def test_offsets_that_are_wrong_stay_inside_the_tensors(oc):
  """tables that run backwards, are negative or too large: any values, no access outside (the kernels clamp)"""
  x = torch.randn(100, 16, device="cuda")
  q = torch.randn(100, 2, 16, device="cuda")
  for table in ([0, 400, 50], [-5, 30, 100], [70, 20, 100], [2 ** 31 - 1, -2 ** 31, 7]):
    t = torch.tensor(table, dtype=torch.int32, device="cuda")
    y, _, carries = oc.nn.octree_recurrence(x, x, t, return_carries=True)
    oc.nn.octree_recurrence_grad(x, x, x, t, carries)
    out, lse = oc.nn.octree_attention(q, q, q, t, k_lengths=torch.tensor([2 ** 30, -4], dtype=torch.int32, device="cuda"),
                                      left=5, right=0, sinks=2, return_lse=True)
    oc.nn.octree_attention_grad(q, q, q, q, out, lse, t, left=5, right=0, sinks=2)
  torch.cuda.synchronize()
