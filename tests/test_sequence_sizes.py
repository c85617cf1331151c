"""Sizes and scales that the operators along the node order of a level cannot take: said, not cut to 32 bits.  Tensors of one
row stand for many (stride 0), so nothing here needs memory."""
import ctypes as C
import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def pkg():
  pkg = importlib.import_module("o-cnn_amd")
  pkg.lib.get()
  return pkg


def offs(*n):
  return torch.tensor(n, dtype=torch.int32)


MANY = [2 ** 31, 2 ** 32 + 4]     # (the second is 4 in 32 bits)


def calls(pkg, rows, device="cpu"):
  """every operator on `rows` rows"""
  nn = pkg.nn
  x3 = torch.zeros(1, 1, 16, device=device).expand(rows, 1, 16)
  x2 = torch.zeros(1, 8, device=device).expand(rows, 8)
  few = torch.zeros(4, 1, 16, device=device)
  o, lse = offs(0, 4).to(device), torch.zeros(1, 1, device=device).expand(rows, 1)
  pos, packed = torch.zeros(1, 1, dtype=torch.int32, device=device), torch.zeros(1, dtype=torch.int64, device=device)
  f = torch.zeros(8, dtype=torch.float64, device=device)
  return {
      "rotary": lambda: nn.octree_rotary(x3, pos.expand(rows, 1), f, [8]),
      "rotary of packed": lambda: nn.octree_rotary(x3, packed.expand(rows), f, [8]),
      "attention": lambda: nn.octree_attention(x3, x3, x3, o),
      "attention of queries": lambda: nn.octree_attention(x3, few, few, o, o),
      "attention of keys": lambda: nn.octree_attention(few, x3, x3, o, o),
      "attention gradient": lambda: nn.octree_attention_grad(x3, x3, x3, x3, x3, lse, o),
      "recurrence": lambda: nn.octree_recurrence(x2, x2, o),
      "recurrence gradient": lambda: nn.octree_recurrence_grad(x2, x2, x2, o, x2),
  }


@pytest.mark.parametrize("rows", MANY)
@pytest.mark.parametrize("name", ["rotary", "rotary of packed", "attention", "attention of queries", "attention of keys",
                                  "attention gradient", "recurrence", "recurrence gradient"])
def test_rows_beyond_32_bits_are_refused(pkg, name, rows):
  with pytest.raises(pkg.nn.OcnnError, match="2147483647"):
    calls(pkg, rows)[name]()


@pytest.mark.parametrize("shape", [(4, 2 ** 32 + 1, 16), (4, 1, 2 ** 32 + 16)])
def test_other_axes_beyond_32_bits_are_refused(pkg, shape):
  x = torch.zeros(1, 1, 1).expand(shape)
  with pytest.raises(pkg.nn.OcnnError, match="2147483647"):
    pkg.nn.octree_attention(x, x, x, offs(0, 4))


def test_tables_beyond_32_bits_are_refused(pkg):
  o = offs(0).expand(2 ** 32 + 2)
  x = torch.zeros(4, 1, 16)
  with pytest.raises(pkg.nn.OcnnError, match="2147483647"):
    pkg.nn.octree_attention(x, x, x, o)
  with pytest.raises(pkg.nn.OcnnError, match="2147483647"):
    pkg.nn.octree_recurrence(x[:, 0], x[:, 0], o)


@pytest.mark.parametrize("scale", [1e300, -1e39, 3e38])
def test_scales_beyond_32_bits_are_refused(pkg, scale):
  """(infinite or NaN in the kernels, where every score of zero would become NaN)"""
  x = torch.zeros(4, 1, 16)
  with pytest.raises(pkg.nn.OcnnError, match="scale"):
    pkg.nn.octree_attention(x, x, x, offs(0, 4), scale=scale)
  with pytest.raises(RuntimeError, match="no CPU path"):
    pkg.nn.octree_attention(x, x, x, offs(0, 4), scale=2e38)


def test_c_entry_points_refuse_scales_that_are_not_finite(pkg):
  for scale in (float("nan"), float("inf"), -float("inf")):
    p = pkg.lib.AttentionParams(16, 16, 16, 64, 16, 32, 16, 32, 16, 16, 16, 0, 0, 1, 4, 8, 4, 2, 16, -1, -1, 0, 0, scale)
    assert pkg.lib.get().ocnn_attention_workspace_bytes(C.byref(p), None, None) == -1
    assert b"scale" in pkg.lib.get().ocnn_last_error()


@pytest.mark.gpu
def test_rows_beyond_32_bits_are_refused_on_a_gpu(oc):
  """the compiled path, which takes tensors on a GPU as they are"""
  for rows in MANY:
    for name, call in calls(oc, rows, "cuda").items():
      with pytest.raises(oc.nn.OcnnError, match="2147483647"):
        call()
  aten = oc.lib.aten()
  x = torch.zeros(1, 8, device="cuda").expand(2 ** 32 + 4, 8)
  with pytest.raises(RuntimeError, match="documented shapes"):
    aten.octree_recurrence(x, x, offs(0, 4).cuda())


@pytest.mark.gpu
def test_scales_beyond_32_bits_are_refused_on_a_gpu(oc):
  x, o = torch.zeros(4, 1, 16, device="cuda"), offs(0, 4).cuda()
  for scale in (1e300, 3e38):
    with pytest.raises(oc.nn.OcnnError, match="scale"):
      oc.nn.octree_attention(x, x, x, o, scale=scale)
  assert bool((oc.nn.octree_attention(x, x, x, o, scale=2e38) == 0).all())


# ---- states in place ------------------------------------------------------------------------------------------
def recurrence_entry(pkg, rows, channels, n_seq, state, last, ws=(None, 0), tensors=(16, 16, 16, 16), dtype=0):
  """the C entry point with addresses: out, gate, data, offsets"""
  i64, p = C.c_int64, C.c_void_p
  out, gate, data, offsets = (p(t) for t in tensors)
  return pkg.lib.get().ocnn_octree_recurrence(out, i64(channels), p(last), None, gate, i64(channels), data, i64(channels), p(state),
                                              offsets, n_seq, rows, channels, 0, 0, dtype, p(ws[0]), C.c_size_t(ws[1]), None)


def test_states_that_overlap_are_refused(pkg):
  """chunks of a sequence read the state after others may have written the last one"""
  L, i64, p = pkg.lib.get(), C.c_int64, C.c_void_p
  base = 1 << 20
  for last in (base, base + 4, base + 4 * 8 - 4, base - 4):
    assert recurrence_entry(pkg, 5000, 8, 1, base, last, (4096, 1 << 30)) == -1
    assert b"overlaps" in L.ocnn_last_error()
  for last in (base + 4, base - 4):           # (a step: the state itself only)
    assert recurrence_entry(pkg, 4, 8, 4, base, last) == -1 and b"overlaps" in L.ocnn_last_error()

  def grad(rows, state, grad_last, grad_state):
    a = p(4096)
    return L.ocnn_octree_recurrence_grad(a, i64(8), a, i64(8), p(grad_state), a, i64(8), p(grad_last), a, i64(8), a, i64(8),
                                         p(state), a, a, 1, rows, 8, 0, 0, a, C.c_size_t(1 << 30), None)
  assert grad(5000, None, base, base) == -1 and b"overlaps" in L.ocnn_last_error()
  assert grad(5000, base, None, base + 4) == -1 and b"overlaps" in L.ocnn_last_error()
  assert grad(20, base, None, base) == -1 and b"overlaps" in L.ocnn_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[1] * 9, [1] * 80 + [400], [300, 0, 200]], ids=["walked", "walked-and-long", "a-workgroup-each"])
def test_a_step_in_place(oc, lengths):
  """the last state written over the one it began with"""
  g = torch.Generator().manual_seed(1)
  n, c = sum(lengths), 20
  gate, data, state = (torch.randn(r, c, generator=g).cuda() for r in (n, n, len(lengths)))
  o = offs(0, *torch.tensor(lengths).cumsum(0).tolist()).cuda()
  want, last = oc.nn.octree_recurrence(gate, data, o, state)
  out = torch.empty_like(want)
  torch.cuda.synchronize()
  assert recurrence_entry(oc, n, c, len(lengths), state.data_ptr(), state.data_ptr(),
                          tensors=[t.data_ptr() for t in (out, gate, data, o)]) == 0
  torch.cuda.synchronize()
  assert torch.equal(out, want) and torch.equal(state, last)
