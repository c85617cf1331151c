"""The operators along the node order of a level as they are used: through autograd, the modules and the U-Net trunk, on
several streams, captured in graphs, through the compiled module, on caches beyond 2^31 elements."""
import importlib

import pytest
import torch

import sequence_reference as ref
import test_gpu_sequence as S
from oracle.checker import make_points_blob
from test_gpu_sequence import TYPES, attention_inputs, check_attention, ids, offs, recurrence_inputs, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tree(oc, orc, synthetic):
  pbs = [make_points_blob(*synthetic.shape_cloud(n, 61 + i)[:2]) for i, n in enumerate((3000, 700))]
  return torch.from_numpy(orc.octree_batch([orc.points2octree(p, 6, 2) for p in pbs])).cuda()


# ---- positions, autograd, modules ---------------------------------------------------------------------
def test_positions_of_a_level(oc, tree):
  for depth in (3, 6):
    xyz = oc.nn.octree_property(tree, "xyz", depth)
    child = oc.nn.octree_property(tree, "child", depth)
    assert torch.equal(oc.nn.octree_positions(tree, depth), xyz)
    assert torch.equal(oc.nn.octree_positions(tree, depth, True), xyz[child >= 0])


def test_functions_are_the_operators_and_their_gradients(oc):
  A, nn = oc.autograd, oc.nn
  o = offs([40, 25]).cuda()
  for dtype in TYPES:
    q, k, v, go = (t.cuda() for t in attention_inputs([40, 25], [40, 25], 4, 2, 24, dtype, 3))
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    kw = (o, None, None, 9, 2, 1, 0.3, None)
    out = A.octree_attention(q, k, v, *kw)
    want, lse = nn.octree_attention(q, k, v, *kw, return_lse=True)
    assert torch.equal(out, want)
    got = torch.autograd.grad(out, (q, k, v), go)
    assert all(torch.equal(a, b) for a, b in zip(got, nn.octree_attention_grad(go, q, k, v, want, lse, *kw)))
    gate, data, state, dy, dl = (t.cuda() for t in recurrence_inputs([40, 25], 12, dtype, 4))
    leaves = [t.requires_grad_(True) for t in (gate, data, state)]
    h, last = A.octree_recurrence(*leaves[:2], o, leaves[2], True)
    full = nn.octree_recurrence(gate, data, o, state, True, return_carries=True)
    assert torch.equal(h, full[0]) and torch.equal(last, full[1])
    for grads in ((dy, dl), (dy, None), (None, dl)):
      outs, gs = zip(*[(t, g) for t, g in zip((h, last), grads) if g is not None])
      got = torch.autograd.grad(outs, leaves, gs, retain_graph=True)
      want = nn.octree_recurrence_grad(torch.zeros_like(dy) if grads[0] is None else dy, gate, data, o, full[2], state,
                                       grads[1], True)
      assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = torch.randn(30, 2, 16, device="cuda").to(dtype).requires_grad_(True)
    pos = torch.randint(0, 99, (30, 2), dtype=torch.int32, device="cuda")
    f = nn.rotary_frequencies([3, 4])
    y = A.octree_rotary(x, pos, f, [3, 4])
    g = torch.randn_like(y)
    assert torch.equal(torch.autograd.grad(y, x, g)[0], nn.octree_rotary(g, pos, f, [3, 4], inverse=True))
  with pytest.raises(oc.nn.OcnnError, match="take no gradient"):
    A.octree_rotary(x, pos, oc.nn.rotary_frequencies([3, 4]).requires_grad_(True), [3, 4])
  with pytest.raises(RuntimeError):                # (no second derivative: said, not computed wrongly)
    y = A.octree_attention(q, k, v, o)
    g, = torch.autograd.grad(y, q, torch.ones_like(y).requires_grad_(True), create_graph=True)
    g.sum().backward()


def test_gradients_against_differences(oc):
  """central differences of the fp32 operators: the step 2^-7 leaves 2^-13 of curvature and 2^-16 of rounding per
  unit of the loss, a sum of some hundred terms of about one"""
  o = offs([30, 9]).cuda()
  eps = 2.0 ** -7

  def check(f, leaves, seed):
    g = torch.Generator().manual_seed(seed)
    out = f(*leaves)
    w = torch.randn(out.shape, generator=g).cuda()
    grads = torch.autograd.grad(out, leaves, w)
    for t, dt in zip(leaves, grads):
      d = torch.randn(t.shape, generator=g).cuda()
      d /= d.norm()
      with torch.no_grad():
        up, down = ((f(*[x + s * eps * d if x is t else x for x in leaves]).double() * w.double()).sum() for s in (1, -1))
      slope, size = float((up - down) / (2 * eps)), float((dt.double() * d.double()).sum())
      assert abs(slope - size) < 2.0 ** -9 * (1 + float(dt.norm())), (slope, size)

  q, k, v, _ = (t.cuda().requires_grad_(True) for t in attention_inputs([30, 9], [30, 9], 4, 2, 16, torch.float32, 8))
  check(lambda a, b, c: oc.autograd.octree_attention(a, b, c, o, None, None, 12, 3, 2), [q, k, v], 1)
  gate, data, state, _, _ = (t.cuda().requires_grad_(True) for t in recurrence_inputs([30, 9], 6, torch.float32, 9))
  check(lambda a, b, c: oc.autograd.octree_recurrence(a, b, o, c)[0], [gate, data, state], 2)


@pytest.mark.parametrize("nempty", [False, True])
def test_modules_on_an_octree_level(oc, tree, nempty):
  """OctreeAttention and OctreeRecurrence against the same composition in 64 bits; gradients reach every parameter"""
  depth, c = 5, 64
  info = oc.nn.octree_info(tree)
  rows = info.nnum_nempty(depth) if nempty else info.nnum(depth)
  x = torch.randn(1, c, rows, 1, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_(True)
  xr = x.detach()[0, :, :, 0].t().double().cpu()
  o = oc.nn.octree_offsets(tree, depth, nempty).cpu()
  torch.manual_seed(0)
  for kv, window in ((2, dict(left=20, right=11, sinks=2)), (4, {})):
    m = oc.OctreeAttention(depth, c, 4, kv, nempty=nempty, **window).cuda()
    y = m(x, tree)
    assert y.shape == x.shape
    joint = (xr @ m.qkv.detach().double().cpu().t()).unflatten(1, (-1, 16))
    q, k, v = joint[:, :4], joint[:, 4:4 + kv], joint[:, 4 + kv:]
    pos = oc.nn.octree_positions(tree, depth, nempty).cpu()
    pos = torch.stack([(pos >> (16 * i)) & 0xffff for i in range(3)], 1)
    f = oc.nn.rotary_frequencies([2, 2, 2], device="cpu")
    q, k = (ref.rotary(t, pos, f, [2, 2, 2], False, False)[0] for t in (q, k))
    mixed = ref.attention(q, k, v, o, o, **window)["out"].flatten(1) @ m.out.detach().double().cpu().t()
    # (the convolutions are fp32 within 1e-4 of their largest value, as everywhere; the operators are finer)
    within(y.detach()[0, :, :, 0].t(), mixed, 3e-4 * float(mixed.abs().max()))
    y.square().sum().backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) and float(p.grad.abs().max()) > 0 for p in m.parameters())
  for both in (False, True):
    m = oc.OctreeRecurrence(depth, c, nempty=nempty, both=both).cuda()
    y = m(x, tree)
    joint = xr @ m.gate_value.detach().double().cpu().t()
    gate, value = joint[:, :c], joint[:, c:]
    cut = c // 2 if both else 0
    h = torch.cat([ref.recurrence(gate[:, :cut], value[:, :cut], o, None, True)["out"],
                   ref.recurrence(gate[:, cut:], value[:, cut:], o)["out"]], 1) @ m.out.detach().double().cpu().t()
    within(y.detach()[0, :, :, 0].t(), h, 3e-4 * float(h.abs().max()))
    y.square().sum().backward()
    assert all(p.grad is not None and float(p.grad.abs().max()) > 0 for p in m.parameters())
  assert bool(torch.isfinite(x.grad).all())
  with pytest.raises(oc.nn.OcnnError, match="multiples of 8"):
    oc.OctreeAttention(depth, c, 16, nempty=nempty).cuda()(x, tree)


def mixer_params(c, heads, kv, dtype, scan=True):
  g = torch.Generator().manual_seed(5)
  dim = c // heads

  def linear(rows, cols, scale=1.0):
    return ((torch.randn(rows, cols, generator=g) * scale / cols ** 0.5).cuda(), (torch.randn(rows, generator=g) * 0.1 * scale).cuda())
  mix = {"heads": heads, "kv_heads": kv, "pairs": [2, 2, 2], "left": 30, "right": 30, "sinks": 1,
         "qkv": linear((heads + 2 * kv) * dim, c), "out": linear(c, c)}
  if scan:
    mix |= {"scan": linear(2 * c, c), "scan_out": linear(c, c)}
  return mix


@pytest.mark.parametrize("nempty", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_node_mixer(oc, tree, dtype, nempty):
  """the sequence projection -> rotary -> attention -> projection -> scan -> projection against 64 bits"""
  depth, c, heads, kv = 4, 64, 4, 2
  info = oc.nn.octree_info(tree)
  rows = info.nnum_nempty(depth) if nempty else info.nnum(depth)
  x = torch.randn(1, c, rows, 1, generator=torch.Generator().manual_seed(2)).to(dtype)
  mix = mixer_params(c, heads, kv, dtype)
  got = oc.stacks.node_mixer(x.cuda(), tree, depth, mix, nempty)
  assert got.dtype == dtype and got.shape == x.shape
  o = oc.nn.octree_offsets(tree, depth, nempty).cpu()
  pos = oc.nn.octree_positions(tree, depth, nempty).cpu()
  pos = torch.stack([(pos >> (16 * i)) & 0xffff for i in range(3)], 1)
  w = {n: (mix[n][0].to(dtype).double().cpu(), mix[n][1].double().cpu()) for n in ("qkv", "out", "scan", "scan_out")}
  xr = x[0, :, :, 0].t().double()
  joint = (xr @ w["qkv"][0].t() + w["qkv"][1]).unflatten(1, (-1, 16))
  f = oc.nn.rotary_frequencies([2, 2, 2], device="cpu")
  q, k = (ref.rotary(t, pos, f, [2, 2, 2], False, False)[0] for t in (joint[:, :heads], joint[:, heads:heads + kv]))
  mixed = ref.attention(q, k, joint[:, heads + kv:], o, o, left=30, right=30, sinks=1)["out"].flatten(1)
  xr = xr + mixed @ w["out"][0].t() + w["out"][1]
  gv = xr @ w["scan"][0].t() + w["scan"][1]
  xr = xr + ref.recurrence(gv[:, :c], gv[:, c:], o)["out"] @ w["scan_out"][0].t() + w["scan_out"][1]
  # fp32: the framework's 1e-4 for convolutions, four in a row; bf16: its 2e-2
  err = float((got[0, :, :, 0].t().double().cpu() - xr).abs().max() / xr.abs().max())
  assert err < (4e-4 if dtype == torch.float32 else 2e-2), err


@pytest.mark.parametrize("nempty", [False, True])
def test_unet_trunk_with_a_mixer(oc, tree, nempty):
  """("mix", d) runs between encoder and decoder; without it, and with projections of zeros, the trunk is what it was"""
  g = torch.Generator().manual_seed(7)
  ch = {6: 16, 5: 32, 4: 64}
  params = {}

  def mk(key, shape, fan):
    n = shape[1] // 8 if key[0] == "up" else shape[0]
    params[key] = ((torch.randn(shape, generator=g) / fan ** 0.5).cuda(), (torch.randn(n, generator=g) * 0.1).cuda())
  mk(("conv", 6), (16, 81), 81)
  for d in (6, 5):
    mk(("down", d), (ch[d - 1], ch[d] * 8), ch[d] * 8)
    mk(("conv", d - 1), (ch[d - 1], ch[d - 1] * 27), ch[d - 1] * 27)
  for d in (4, 5):
    mk(("up", d), (ch[d], ch[d + 1] * 8), ch[d])
    mk(("dec", d + 1), (ch[d + 1], 2 * ch[d + 1] * 27), 2 * ch[d + 1] * 27)
  stacks = oc.stacks
  plain = stacks.unet_trunk(tree, 6, params, stages=2, nempty=nempty)
  mix = mixer_params(64, 4, 2, torch.float32)
  mixed = stacks.unet_trunk(tree, 6, params | {("mix", 4): mix}, stages=2, nempty=nempty)
  assert mixed.shape == plain.shape and bool(torch.isfinite(mixed).all()) and not torch.equal(mixed, plain)
  nothing = mix | {n: tuple(torch.zeros_like(t) for t in mix[n]) for n in ("out", "scan_out")}
  assert torch.equal(stacks.unet_trunk(tree, 6, params | {("mix", 4): nothing}, stages=2, nempty=nempty), plain)
  narrow = {key: (w.bfloat16(), b) for key, (w, b) in params.items()}
  rows = stacks.unet_trunk_rows(tree, 6, narrow, stages=2, nempty=nempty)
  assert torch.equal(stacks.unet_trunk_rows(tree, 6, narrow | {("mix", 4): nothing}, stages=2, nempty=nempty), rows)
  rows_mixed = stacks.unet_trunk_rows(tree, 6, narrow | {("mix", 4): mix}, stages=2, nempty=nempty)
  err = float((rows_mixed.float() - mixed).abs().max() / mixed.abs().max())
  assert err < 0.1, err          # (bf16 between some twenty operators, none of them checked here: that it is the same network)


# ---- many sequences at once: the shapes that a filled chip takes --------------------------------------------
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_of_many_sequences(oc, dtype, dim):
  """as many workgroups as fill the chip, most of them of short sequences, one sequence with rows that see its sinks only"""
  lengths = [(7 * i) % 23 for i in range(200)]
  lengths[50], lengths[120] = 300, 150
  q, k, v, go = attention_inputs(lengths, lengths, 4, 2, dim, dtype, 17)
  o = offs(lengths)
  for kw in (dict(left=40, right=0, sinks=2), dict(left=9, right=5), {}):
    check_attention(oc, dtype, q, k, v, go, o, o, **kw)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_among_many_empty_sequences(oc, dtype, monkeypatch):
  """the cases of the few-workgroup shapes again with 330 empty sequences behind, which the rules count as work"""
  plain = S.offs
  monkeypatch.setattr(S, "offs", lambda lengths: plain(list(lengths) + [0] * 330))
  for case in S.SELF:
    S.test_attention_and_its_gradient(oc, dtype, case)
  for bad in (float("nan"), float("inf")):
    S.test_attention_bad_values_stay_with_the_rows_that_see_them(oc, dtype, bad)
  S.test_attention_key_mask(oc, dtype)
  S.test_attention_large_scores(oc, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_split_keys_with_large_scores(oc, dtype):
  """many rows whose keys are dealt out over workgroups: weights beyond the base's reach, and a bad value"""
  lengths = [4096]
  q, k, v, go = attention_inputs(lengths, lengths, 2, 2, 32, dtype, 23)
  check_attention(oc, dtype, q * 40, k * 40, v, go, offs(lengths), offs(lengths), backward=False)
  v[3000] = float("nan")
  out = oc.nn.octree_attention(q.cuda(), k.cuda(), v.cuda(), offs(lengths).cuda(), right=0)
  v[3000] = 0.0
  want = ref.attention(q, k, v, offs(lengths), offs(lengths), right=0, dtype=dtype)
  within(out[:3000], want["out"][:3000], want["out_tol"][:3000])
  assert bool(torch.isnan(out[3000:]).all())


@pytest.mark.parametrize("lengths, channels", [
    ([5000], 12), ([3000, 2500], 33),                          # chunks, their list in one launch
    ([20000], 24),                                             # chunks, their list in two launches
    ([2000, 1, 1900, 0, 15, 17], 7),                           # a workgroup a sequence, 4 channels
    ([1500, 0, 1, 2100, 1024, 1025] * 5, 20), ([700] * 9, 64),  # 8 channels, one and more loads of rows
], ids=lambda x: "+".join(map(str, x[:6])) if isinstance(x, list) else str(x))
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_recurrence_in_each_of_its_shapes(oc, dtype, reverse, lengths, channels):
  S.check_recurrence(oc, dtype, lengths, channels, reverse, True, seed=41, extra=37)
  S.check_recurrence(oc, dtype, lengths, channels, reverse, False, seed=42)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_share_of_nan_keys(oc, dtype):
  """one query whose keys are dealt out: shares in which no visible score is a number must not be lost in the join"""
  for keys in (512, 2048, 4096):
    q, k, v, go = (t.cuda() for t in attention_inputs([1], [keys], 1, 1, 64, dtype, 43))
    for first in range(0, keys, 128):
      bad = k.clone()
      bad[first:first + 128] = float("nan")
      out, lse = oc.nn.octree_attention(q, bad, v, offs([1]).cuda(), offs([keys]).cuda(), return_lse=True)
      assert bool(torch.isnan(out).all()) and bool(torch.isnan(lse).all()), (keys, first)


def test_attention_of_nothing_but_nan_ends_soon(oc):
  """a diverged model: every row is taken again, and ends at its first NaN (30000 rows; a full second pass takes seconds)"""
  q, k, v, go = (torch.full((30000, 2, 64), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(4))
  o = offs([30000]).cuda()
  out, lse = oc.nn.octree_attention(q, k, v, o, return_lse=True)
  grads = oc.nn.octree_attention_grad(go, q, k, v, out, lse, o)
  assert all(bool(torch.isnan(t).all()) for t in (out, lse, *grads))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("lengths", [[50, 70, 1, 0, 90], [3000, 900, 2000, 0, 1, 2500] * 2, [3000, 900, 5000, 0, 1, 4000]],
                         ids=["short", "many", "long"])
def test_recurrence_bad_values_stay_in_their_sequence(oc, dtype, reverse, lengths):
  gate, data, state, dy, dl = recurrence_inputs(lengths, 20, dtype, 24)
  o = offs(lengths)
  a, b = int(o[1]), int(o[2])
  bad = [x.clone() for x in (gate, data, state, dy, dl)]
  bad[0][a + 3], bad[1][a + 5], bad[1][b - 2], bad[2][1], bad[3][a], bad[4][1] = (
      float("nan"), float("inf"), float("nan"), float("inf"), float("nan"), float("inf"))

  def run(gate, data, state, dy, dl):
    gate, data, state, dy, dl = (x.cuda() for x in (gate, data, state, dy, dl))
    h, last, carries = oc.nn.octree_recurrence(gate, data, o.cuda(), state, reverse, return_carries=True)
    grads = oc.nn.octree_recurrence_grad(dy, gate, data, o.cuda(), carries, state, dl, reverse)
    return (h, *grads[:2]), (last, grads[2])
  rows, states = run(gate, data, state, dy, dl)
  bad_rows, bad_states = run(*bad)
  keep = torch.ones(rows[0].size(0), dtype=torch.bool, device="cuda")
  keep[a:b] = False
  assert all(torch.equal(x[keep], y[keep]) for x, y in zip(rows, bad_rows))
  keep = torch.arange(len(lengths), device="cuda") != 1
  assert all(torch.equal(x[keep], y[keep]) for x, y in zip(states, bad_states))
  assert not bool(torch.isfinite(bad_rows[0][a:b]).all())


def test_attention_axes_of_one_and_the_lse_beside_an_output(oc):
  """axes of one with strides of their own; the lse of rows of no sequence where `out` is given"""
  o = offs([60, 20]).cuda()
  q, k, v, go = (t.cuda() for t in attention_inputs([60, 20], [60, 20], 1, 1, 16, torch.float32, 25))
  want, lse = oc.nn.octree_attention(q, k, v, o, return_lse=True)
  far = [t.as_strided(t.shape, (t.stride(0), (1 << 23) + 3, 1)) for t in (q, k, v)]
  assert torch.equal(oc.nn.octree_attention(*far, o), want)
  out = torch.empty_like(q).as_strided(q.shape, (q.stride(0), 7, 1))
  assert torch.equal(oc.nn.octree_attention(*far, o, out=out), want)
  grads = oc.nn.octree_attention_grad(go, q, k, v, want, lse, o)
  assert all(torch.equal(a, b) for a, b in zip(oc.nn.octree_attention_grad(go, *far, want, lse, o), grads))
  one = [t[:1].as_strided((1, 1, 16), (7, 5, 1)) for t in (q, k, v)]
  assert torch.equal(oc.nn.octree_attention(*one, offs([1]).cuda()), v[:1])
  rest = torch.full((90, 1, 16), 3.0, device="cuda")
  more = [torch.cat([t, torch.full_like(t[:10], float("nan"))]) for t in (q, k, v)]
  got, lse90 = oc.nn.octree_attention(*more, o, out=rest, return_lse=True)
  assert torch.equal(got[:80], want) and bool((got[80:] == 3.0).all())
  assert torch.equal(lse90[:80], lse) and bool((lse90[80:] == -float("inf")).all())


# ---- streams, graphs, repeats ------------------------------------------------------------------------------
def every_call(oc, dtype, seed=21):
  """calls that between them reach every kernel, and the inputs they read"""
  nn = oc.nn
  lengths, few, long = [300, 0, 1, 170], [2, 1], [9000, 700]
  q, k, v, go = (t.cuda() for t in attention_inputs(lengths, lengths, 4, 2, 64, dtype, seed))
  q1, k1, v1, _ = (t.cuda() for t in attention_inputs(few, long, 8, 2, 64, dtype, seed + 1))
  gate, data, state, dy, dl = (t.cuda() for t in recurrence_inputs([700, 3, 900], 40, dtype, seed + 2))
  step = [t.cuda() for t in recurrence_inputs([1] * 9, 40, dtype, seed + 3)]
  gate2, data2, state2, dy2, dl2 = (t.cuda() for t in recurrence_inputs([20000], 12, dtype, seed + 4))
  o, fo, lo, ro, so = (offs(x).cuda() for x in (lengths, few, long, [700, 3, 900], [1] * 9))
  full, short, whole = (offs(x).cuda() for x in (lengths + [0] * 330, [5000], [20000]))
  pos = torch.randint(0, 500, (q.size(0), 3), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).cuda()
  f = nn.rotary_frequencies([8, 8, 8])
  w = dict(left=40, right=20, sinks=3)

  def run():
    out, lse = nn.octree_attention(q, k, v, o, return_lse=True, **w)
    h, last, carries = nn.octree_recurrence(gate, data, ro, state, return_carries=True)
    out2, lse2 = nn.octree_attention(q, k, v, full, return_lse=True, **w)
    more = [out2, lse2, *nn.octree_attention_grad(go, q, k, v, out2, lse2, full, **w)]
    for offsets, n in ((short, 5000), (whole, 20000)):
      h2, last2, carries2 = nn.octree_recurrence(gate2[:n], data2[:n], offsets, state2, return_carries=True)
      more += [h2, last2, *nn.octree_recurrence_grad(dy2[:n], gate2[:n], data2[:n], offsets, carries2, state2, dl2)]
    return more + [nn.octree_rotary(q, pos, f, [8, 8, 8]), nn.octree_rotary(q, pos, f, [8, 8, 8], True, True), out, lse,
            *nn.octree_attention_grad(go, q, k, v, out, lse, o, **w), nn.octree_attention(q1, k1, v1, fo, lo, right=0),
            h, last, *nn.octree_recurrence_grad(dy, gate, data, ro, carries, state, dl),
            *nn.octree_recurrence(step[0], step[1], so, step[2])]
  return run, [q, k, v, go, q1, k1, v1, gate, data, state, dy, dl, gate2, data2, state2, dy2, dl2] + step[:3]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_calls_repeat_and_run_on_streams(oc, dtype):
  """no result depends on timing: three runs, and two streams at once, give the same bits"""
  run, _ = every_call(oc, dtype)
  other, _ = every_call(oc, dtype, 31)
  want, want2 = run(), other()
  torch.cuda.synchronize()
  for _ in range(2):
    assert all(torch.equal(a, b) for a, b in zip(run(), want))
  sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
  got = []
  for _ in range(4):
    for s, f in ((sa, run), (sb, other)):
      with torch.cuda.stream(s):
        got.append((f(), want if f is run else want2))
  torch.cuda.synchronize()
  for a, b in got:
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_calls_in_graphs(oc, dtype):
  """two graphs over the same inputs, replayed in turn and at once, with new inputs and eager calls between"""
  run, inputs = every_call(oc, dtype)
  run()
  torch.cuda.synchronize()
  graphs = []
  for _ in range(2):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      outs = run()
    graphs.append((g, outs))
  side = torch.cuda.Stream()
  gen = torch.Generator().manual_seed(1)
  for turn in range(4):
    for t in inputs:
      t.copy_(torch.randn(t.shape, generator=gen).to(t.dtype))
    want = run()
    torch.cuda.synchronize()
    graphs[0][0].replay()
    with torch.cuda.stream(side):
      graphs[1][0].replay()
    torch.cuda.synchronize()
    for _, outs in graphs:
      assert all(torch.equal(a, b) for a, b in zip(outs, want)), turn


def test_training_step_in_a_graph(oc):
  """forward and backward through autograd, captured, against the same eager step"""
  A = oc.autograd
  o = offs([90, 38]).cuda()
  x, w = (torch.randn(128, 96, generator=torch.Generator().manual_seed(i)).cuda() for i in (1, 2))
  pos = torch.arange(128, dtype=torch.int32, device="cuda")[:, None].contiguous()
  f = oc.nn.rotary_frequencies([8])

  def step():
    leaf = x.detach().requires_grad_(True)
    q, k, v = leaf.view(128, 6, 16).split([2, 2, 2], 1)
    y = A.octree_attention(A.octree_rotary(q, pos, f, [8]), A.octree_rotary(k, pos, f, [8]), v, o, None, None, 20, 0)
    h, last = A.octree_recurrence(leaf[:, :32], y.flatten(1), o)
    return torch.autograd.grad(h.mul(w[:, :32]).sum() + last.square().sum(), leaf)[0]

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step()
  torch.cuda.current_stream().wait_stream(side)
  g = torch.cuda.CUDAGraph()
  with torch.cuda.graph(g):
    got = step()
  for i in range(4):
    x.normal_(generator=torch.Generator("cuda").manual_seed(i))
    want = step()
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want), i


# ---- the two host paths, far rows -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_compiled_module_and_ctypes_are_one(oc, tree, dtype, monkeypatch):
  run, _ = every_call(oc, dtype)
  fast = run()
  sequence = importlib.import_module("o-cnn_amd.sequence")
  assert sequence._compiled()
  monkeypatch.setattr(sequence, "_fast", False)
  assert all(torch.equal(a, b) for a, b in zip(run(), fast))
  aten = oc.lib.aten()
  assert torch.equal(aten.octree_offsets(tree, 5), oc.nn.octree_offsets(tree, 5))
  assert torch.equal(aten.octree_offsets(tree, 5, True), oc.nn.octree_offsets(tree, 5, True))
  q, k, v, go = (t.cuda() for t in attention_inputs([50, 9], [50, 9], 4, 2, 32, dtype, 2))
  o = offs([50, 9]).cuda()
  out, lse = aten.octree_attention(q, k, v, o, left=7, right=0, sinks=1, return_lse=True)
  want = oc.nn.octree_attention(q, k, v, o, left=7, right=0, sinks=1, return_lse=True)
  assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
  assert len(aten.octree_attention(q, k, v, o)) == 1
  got = aten.octree_attention_grad(go, q, k, v, out, lse, o, left=7, right=0, sinks=1)
  assert all(torch.equal(a, b) for a, b in zip(got, oc.nn.octree_attention_grad(go, q, k, v, out, lse, o, left=7, right=0, sinks=1)))
  gate, data, state, dy, dl = (t.cuda() for t in recurrence_inputs([50, 9], 24, dtype, 3))
  h, last, carries = aten.octree_recurrence(gate, data, o, state, return_carries=True)
  want = oc.nn.octree_recurrence(gate, data, o, state, return_carries=True)
  assert torch.equal(h, want[0]) and torch.equal(last, want[1])
  got = aten.octree_recurrence_grad(dy, gate, data, o, carries, state, dl)
  assert all(torch.equal(a, b) for a, b in zip(got, oc.nn.octree_recurrence_grad(dy, gate, data, o, carries, state, dl)))
  pos, f = torch.randint(0, 9, (59, 1), dtype=torch.int32, device="cuda"), oc.nn.rotary_frequencies([9])
  assert torch.equal(aten.octree_rotary(q, pos, f, [9]), oc.nn.octree_rotary(q, pos, f, [9]))
  for bad in (lambda: aten.octree_rotary(q, pos, f, [8]), lambda: aten.octree_attention(q.half(), k, v, o),
              lambda: aten.octree_recurrence(gate, data[:-1], o)):
    with pytest.raises(RuntimeError, match="must be on the current GPU"):
      bad()


def test_cache_beyond_32_bit_offsets(oc):
  """keys whose element offset passes 2^31: a window at the far end, against the same rows by themselves"""
  rows, kv, dim = 1100000, 16, 128                   # 2.25e9 elements a tensor
  k = torch.empty(rows, kv, dim, dtype=torch.bfloat16, device="cuda")
  v = torch.empty_like(k)
  tail = 600
  for t in (k, v):
    t[-tail:] = torch.randn(tail, kv, dim, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    t[:64] = torch.randn(64, kv, dim, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
  for queries in (1, 200):
    q = torch.randn(queries, 32, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    qo = offs([queries]).cuda()
    got, lse = oc.nn.octree_attention(q, k, v, qo, offs([rows]).cuda(), left=300, right=0, sinks=5, return_lse=True)
    # the same sequence without its middle: the sinks, then the last rows
    k2, v2 = (torch.cat([t[:64], t[-tail:]]) for t in (k, v))
    want, lse2 = oc.nn.octree_attention(q, k2, v2, qo, offs([64 + tail]).cuda(), left=300, right=0, sinks=5, return_lse=True)
    # (tiles begin at other keys, so sums are in another order: two bf16 roundings of the weights and of the result)
    within(got, want.double().cpu(), 2.0 ** -8 * 2 * float(v2.abs().max()) + 2.0 ** -7 * want.double().abs().cpu())
    within(lse, lse2.double().cpu(), 2.0 ** -18 * float(lse2.abs().max()))
  del k, v
  torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("reverse", [False, True])
def test_long_chunks_of_the_recurrence(oc, dtype, reverse):
  """2^25 elements and more go in chunks of 64 rows and past the caches; each sequence by itself goes in chunks of 16"""
  lengths, channels = [60001, 1, 0, 63, 74000], 264
  gate, data, state, dy, dl = (t.cuda() for t in recurrence_inputs(lengths, channels, dtype, 12))
  o = offs(lengths).cuda()
  h, last, carries = oc.nn.octree_recurrence(gate, data, o, state, reverse, return_carries=True)
  grads = oc.nn.octree_recurrence_grad(dy, gate, data, o, carries, state, dl, reverse)
  at = offs(lengths).tolist()
  # the same sums cut elsewhere: a few hundred rows weigh in a state, 2^-24 each of a partial sum: 2^-18 of the largest at most.
  # bf16: and a step more where that tips a rounding
  step = 0.0 if dtype == torch.float32 else 2.0 ** -7

  def near(a, b):
    b = b.double().cpu()
    within(a, b, 2.0 ** -18 * max(float(b.abs().max()), 1.0) + step * b.abs())
  for i, n in enumerate(lengths):
    if n == 0:
      continue
    r, own = slice(at[i], at[i + 1]), offs([n]).cuda()
    one = oc.nn.octree_recurrence(gate[r], data[r], own, state[i:i + 1], reverse, return_carries=True)
    near(h[r], one[0])
    near(last[i:i + 1], one[1])
    g = oc.nn.octree_recurrence_grad(dy[r], gate[r], data[r], own, one[2], state[i:i + 1], dl[i:i + 1], reverse)
    near(grads[0][r], g[0])
    near(grads[1][r], g[1])
    near(grads[2][i:i + 1], g[2])


def test_rotary_and_recurrence_beyond_32_bit_offsets(oc):
  rows, channels = 4400000, 512                      # 2.25e9 elements
  x = torch.zeros(rows, 8, 64, dtype=torch.bfloat16, device="cuda")
  x[-50:] = torch.randn(50, 8, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
  pos = torch.arange(rows, dtype=torch.int32, device="cuda")[:, None].contiguous()
  f = oc.nn.rotary_frequencies([32])
  y = oc.nn.octree_rotary(x, pos, f, [32])
  assert torch.equal(y[-50:], oc.nn.octree_rotary(x[-50:].contiguous(), pos[-50:].contiguous(), f, [32]))
  del y
  x = x.view(rows, channels)
  o = offs([rows - 40, 40]).cuda()
  h, last = oc.nn.octree_recurrence(x, x, o)
  alone, end = oc.nn.octree_recurrence(x[-40:].contiguous(), x[-40:].contiguous(), offs([40]).cuda())
  within(h[-40:], alone.double().cpu(), 2.0 ** -16 + 2.0 ** -7 * alone.double().abs().cpu())
  within(last[1:], end.double().cpu(), 2.0 ** -16)
  del x, h
  torch.cuda.empty_cache()
