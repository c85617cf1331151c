"""What the operators along the node order of a level refuse, without a GPU: the Python checks come before any device
work, and the C entry points check their arguments before they launch anything."""
import ctypes as C
import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def pkg():
  lib = importlib.import_module("o-cnn_amd.lib")
  lib.get()
  return importlib.import_module("o-cnn_amd")


def offs(*n):
  return torch.tensor(n, dtype=torch.int32)


# ---- rotary ---------------------------------------------------------------------------------------------
def rotary_case(**change):
  c = dict(data=torch.zeros(4, 2, 16), positions=torch.zeros(4, 3, dtype=torch.int32),
           frequencies=torch.zeros(6, dtype=torch.float64), pairs=[2, 2, 2], out=None)
  c.update(change)
  return c


@pytest.mark.parametrize("change, message", [
    (dict(data=torch.zeros(4, 16)), "3 axes"),
    (dict(pairs=[]), "1 to 4 axes"),
    (dict(pairs=[1] * 5, frequencies=torch.zeros(5, dtype=torch.float64)), "1 to 4 axes"),
    (dict(pairs=[3, 3, 3], frequencies=torch.zeros(9, dtype=torch.float64)), "18 channels"),
    (dict(pairs=[-1, 4, 3]), "pairs"),
    (dict(frequencies=torch.zeros(6)), "float64"),
    (dict(frequencies=torch.zeros(5, dtype=torch.float64)), "expected 6"),
    (dict(positions=torch.zeros(4, 2, dtype=torch.int32)), r"\[4, 3\]"),
    (dict(positions=torch.zeros(3, 3, dtype=torch.int32)), r"\[4, 3\]"),
    (dict(positions=torch.zeros(4, 3, dtype=torch.int16)), "int32, float32 or packed int64"),
    (dict(positions=torch.zeros(5, dtype=torch.int64)), "packed"),
    (dict(positions=torch.zeros(4, dtype=torch.int64), pairs=[1, 1, 1, 1], frequencies=torch.zeros(4, dtype=torch.float64)),
     "at most 3 axes"),
    (dict(out=torch.zeros(4, 2, 8)), "out must be"),
    (dict(out=torch.zeros(4, 2, 16, dtype=torch.bfloat16)), "out must be"),
    (dict(out=torch.zeros(1, 1, 16).expand(4, 2, 16)), "overlaps itself"),
])
def test_rotary_refuses(pkg, change, message):
  c = rotary_case(**change)
  with pytest.raises(pkg.nn.OcnnError, match=message):
    pkg.nn.octree_rotary(c["data"], c["positions"], c["frequencies"], c["pairs"], out=c["out"])


def test_rotary_refuses_an_output_on_part_of_the_input(pkg):
  joint = torch.zeros(4, 4, 16)
  c = rotary_case(data=joint[:, :2])
  with pytest.raises(pkg.nn.OcnnError, match="overlaps an input"):
    pkg.nn.octree_rotary(c["data"], c["positions"], c["frequencies"], c["pairs"], out=joint[:, 1:3])


def test_other_types_and_cpu_tensors(pkg):
  c = rotary_case(data=torch.zeros(4, 2, 16, dtype=torch.float16))
  with pytest.raises(TypeError, match="float32 or bfloat16"):
    pkg.nn.octree_rotary(c["data"], c["positions"], c["frequencies"], c["pairs"])
  c = rotary_case()
  with pytest.raises(RuntimeError, match="no CPU path"):
    pkg.nn.octree_rotary(c["data"], c["positions"], c["frequencies"], c["pairs"])
  with pytest.raises(RuntimeError, match="no CPU path"):
    pkg.nn.octree_recurrence(torch.zeros(4, 8), torch.zeros(4, 8), offs(0, 4))
  q = torch.zeros(4, 2, 16)
  with pytest.raises(RuntimeError, match="no CPU path"):
    pkg.nn.octree_attention(q, q, q, offs(0, 4))


# ---- attention ------------------------------------------------------------------------------------------
def attention_case(**change):
  c = dict(q=torch.zeros(6, 4, 16), k=torch.zeros(8, 2, 16), v=torch.zeros(8, 2, 16), q_offsets=offs(0, 2, 6),
           k_offsets=offs(0, 3, 8))
  c.update(change)
  return c


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros(6, 64)), "3 axes"),
    (dict(k=torch.zeros(8, 3, 16), v=torch.zeros(8, 3, 16)), "4 query heads over 3 key heads"),
    (dict(v=torch.zeros(8, 2, 24)), "v is"),
    (dict(k=torch.zeros(8, 2, 24), v=torch.zeros(8, 2, 24)), "channels a head"),
    (dict(k=torch.zeros(8, 2, 16, dtype=torch.bfloat16)), "expected torch.float32"),
    (dict(q=torch.zeros(6, 4, 12), k=torch.zeros(8, 2, 12), v=torch.zeros(8, 2, 12)), "multiples of 8"),
    (dict(q=torch.zeros(6, 4, 136), k=torch.zeros(8, 2, 136), v=torch.zeros(8, 2, 136)), "up to 128"),
    (dict(k_offsets=None), "need k_offsets"),
    (dict(k_offsets=offs(0, 8)), "expected 3"),
    (dict(q_offsets=torch.tensor([0, 2, 6])), "int32"),
    (dict(q_offsets=offs(0)), "one more"),
    (dict(k_lengths=offs(1, 2, 3)), "expected 2"),
    (dict(key_mask=torch.ones(8)), "bool"),
    (dict(key_mask=torch.ones(7, dtype=torch.bool)), "bool"),
    (dict(left=-2), "window"),
    (dict(right=-7), "window"),
    (dict(left=2 ** 31), "window"),
    (dict(sinks=65), "at most 64"),
    (dict(sinks=-1), "sinks"),
    (dict(scale=float("nan")), "scale"),
    (dict(q=torch.zeros(6, 65, 16), k=torch.zeros(8, 1, 16), v=torch.zeros(8, 1, 16)), "65 query heads a key head"),
])
def test_attention_refuses(pkg, change, message):
  with pytest.raises(pkg.nn.OcnnError, match=message):
    pkg.nn.octree_attention(**attention_case(**change))


@pytest.mark.parametrize("change, message", [
    (dict(grad_out=torch.zeros(6, 4, 8)), "grad_out"),
    (dict(out=torch.zeros(5, 4, 16)), "out is"),
    (dict(lse=torch.zeros(4, 6)), "lse"),
    (dict(lse=torch.zeros(6, 4, dtype=torch.float64)), "lse"),
])
def test_attention_grad_refuses(pkg, change, message, monkeypatch):
  # (shapes are checked behind the check for a GPU, which is taken as passed here: nothing is launched)
  monkeypatch.setattr(importlib.import_module("o-cnn_amd.sequence"), "_on_gpu", lambda t: None)
  c = attention_case(grad_out=torch.zeros(6, 4, 16), out=torch.zeros(6, 4, 16), lse=torch.zeros(6, 4))
  c.update(change)
  with pytest.raises(pkg.nn.OcnnError, match=message):
    pkg.nn.octree_attention_grad(c.pop("grad_out"), c.pop("q"), c.pop("k"), c.pop("v"), c.pop("out"), c.pop("lse"), **c)


# ---- recurrence -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("change, message", [
    (dict(gate=torch.zeros(4, 7)), "gate is"),
    (dict(gate=torch.zeros(4, 8, dtype=torch.bfloat16)), "expected torch.float32"),
    (dict(data=torch.zeros(4, 2, 4)), "2 axes"),
    (dict(gate=torch.zeros(4, 0), data=torch.zeros(4, 0)), "no channels"),
    (dict(offsets=offs(0)), "one more"),
    (dict(offsets=torch.tensor([0, 4])), "int32"),
    (dict(state=torch.zeros(2, 8)), "state"),
    (dict(state=torch.zeros(1, 8, dtype=torch.bfloat16)), "state"),
])
def test_recurrence_refuses(pkg, change, message):
  c = dict(gate=torch.zeros(4, 8), data=torch.zeros(4, 8), offsets=offs(0, 4))
  c.update(change)
  with pytest.raises(pkg.nn.OcnnError, match=message):
    pkg.nn.octree_recurrence(**c)


def test_recurrence_grad_refuses(pkg, monkeypatch):
  monkeypatch.setattr(importlib.import_module("o-cnn_amd.sequence"), "_on_gpu", lambda t: None)
  x, o = torch.zeros(4, 8), offs(0, 4)
  with pytest.raises(pkg.nn.OcnnError, match="return_carries"):
    pkg.nn.octree_recurrence_grad(x, x, x, o, None)
  with pytest.raises(pkg.nn.OcnnError, match="carries"):
    pkg.nn.octree_recurrence_grad(x, x, x, o, torch.zeros(1, 8))
  with pytest.raises(pkg.nn.OcnnError, match="grad_out"):
    pkg.nn.octree_recurrence_grad(x[:3], x, x, o, torch.zeros(2, 8))


# ---- the C entry points -------------------------------------------------------------------------------------
def test_c_entry_points_return_codes(pkg):
  """null pointers, bad enums, misaligned rows, small workspaces: a code and a message, no launch"""
  lib = pkg.lib
  L, null, one = lib.get(), C.c_void_p(0), C.c_void_p(16)
  i64 = C.c_int64
  pairs = (C.c_int * 4)(2, 2, 0, 0)

  def rotary(rows=1, dim=16, dtype=0, kind=0, axes=2, data=one):
    return L.ocnn_octree_rotary(one, i64(16), i64(16), data, i64(16), i64(16), rows, 1, dim, one, kind, i64(2), one, pairs,
                                axes, 0, 0, dtype, null)
  assert rotary(rows=0) == 0
  assert rotary(data=null) == -1 and rotary(dtype=5) == -1 and rotary(kind=3) == -1 and rotary(axes=0) == -1
  assert rotary(axes=4, kind=2) == -1
  assert rotary(dim=6) == -3 and b"channels" in L.ocnn_last_error()
  assert rotary(dim=2048) == -2

  def attention(ws=null, ws_bytes=0, q=16, q_row=64, entry="fwd", **kw):
    p = lib.AttentionParams(q, 16, 16, q_row, 16, 32, 16, 32, 16, 16, 16, 0, 0, 1, 4, 8, 4, 2, 16, -1, -1, 0, 0, 0.25)
    for n, x in kw.items():
      setattr(p, n, x)
    if entry == "fwd":
      return L.ocnn_octree_attention(one, i64(64), i64(16), null, C.byref(p), 0, ws, C.c_size_t(ws_bytes), null)
    return L.ocnn_octree_attention_grad(one, i64(64), i64(16), one, i64(32), i64(16), one, i64(32), i64(16), one, i64(64), i64(16),
                                        one, i64(64), i64(16), one, C.byref(p), ws, C.c_size_t(ws_bytes), null)
  assert attention(rows_q=0) == 0
  assert attention(q=0) == -1 and attention(dtype=9) == -1 and attention(n_seq=0) == -1 and attention(left=-2) == -1
  assert attention(heads=3) == -3 and attention(dim=20) == -2 and attention(sinks=65) == -2
  assert attention(q=8) == -1 and b"16 bytes" in L.ocnn_last_error()
  assert attention(q_row=66) == -1
  assert attention(rows_k=1 << 20) == -4 and b"bytes" in L.ocnn_last_error()     # few rows, many keys: split, needs a workspace
  assert attention(entry="grad") == -4
  assert attention(entry="grad", q_offsets=0) == -1
  need, grad = C.c_size_t(), C.c_size_t()
  assert L.ocnn_attention_workspace_bytes(null, C.byref(need), C.byref(grad)) == -1

  shape = (C.c_int64(), C.c_size_t(), C.c_size_t())
  assert L.ocnn_recurrence_shape(-1, 8, 1, 0, *map(C.byref, shape)) == -1
  assert L.ocnn_recurrence_shape(8, 8, 0, 0, *map(C.byref, shape)) == -1
  assert L.ocnn_recurrence_shape(1000, 8, 1, 1, *map(C.byref, shape)) == 0 and shape[0].value >= 1000 // 64

  def recurrence(rows=5000, channels=8, dtype=0, data=one, offsets=one, ws=null, ws_bytes=0):
    return L.ocnn_octree_recurrence(one, i64(8), null, null, one, i64(8), data, i64(8), null, offsets, 1, rows, channels, 0, 0,
                                    dtype, ws, C.c_size_t(ws_bytes), null)
  assert recurrence() == -4 and recurrence(ws=one, ws_bytes=64) == -4
  assert recurrence(data=null) == -1 and recurrence(offsets=null) == -1 and recurrence(dtype=2) == -1
  assert recurrence(channels=0) == -1
  assert L.ocnn_octree_recurrence_grad(one, i64(8), one, i64(8), null, one, i64(8), null, one, i64(8), one, i64(8), null, null, one,
                                       1, 10, 8, 0, 0, one, C.c_size_t(1 << 20), null) == -1    # no carries
  assert L.ocnn_octree_offsets(null, one, one, 1, 0, null) == -1


def test_reference_gradients_agree_with_differences():
  """The formulas the GPU results are tested against, against central differences in 64 bits"""
  import sequence_reference as ref
  g = torch.Generator().manual_seed(2)
  r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)   # noqa: E731
  qo, ko = [0, 3, 3, 9], [0, 5, 6, 12]
  q, k, v, go = r(9, 4, 8), r(12, 2, 8), r(12, 2, 8), r(9, 4, 8)
  kw = dict(left=2, right=1, sinks=1, key_mask=torch.tensor([1, 1, 0, 1, 1, 1, 1, 1, 1, 0, 1, 1], dtype=torch.bool))
  full = ref.attention(q, k, v, qo, ko, grad=go, **kw)
  f = lambda a, b, c: float((ref.attention(a, b, c, qo, ko, **kw)["out"] * go).sum())   # noqa: E731
  eps = 1e-5
  for name, which in (("dq", 0), ("dk", 1), ("dv", 2)):
    for _ in range(6):
      args = [q, k, v]
      at = tuple(int(torch.randint(0, n, (1,), generator=g)) for n in args[which].shape)
      ends = []
      for sign in (1, -1):
        moved = [t.clone() for t in args]
        moved[which][at] += sign * eps
        ends.append(f(*moved))
      assert abs((ends[0] - ends[1]) / (2 * eps) - float(full[name][at])) < 1e-7, (name, at)
  gate, x, h0, dy, dl, o = r(9, 3), r(9, 3), r(3, 3), r(9, 3), r(3, 3), [0, 4, 4, 9]
  for reverse in (False, True):
    full = ref.recurrence(gate, x, o, h0, reverse, dy, dl)

    def value(a, b, c):
      s = ref.recurrence(a, b, o, c, reverse)
      return float((s["out"] * dy).sum() + (s["last"] * dl).sum())
    for name, which in (("dgate", 0), ("ddata", 1), ("dstate", 2)):
      for _ in range(5):
        args = [gate, x, h0]
        at = tuple(int(torch.randint(0, n, (1,), generator=g)) for n in args[which].shape)
        ends = []
        for sign in (1, -1):
          moved = [t.clone() for t in args]
          moved[which][at] += sign * eps
          ends.append(value(*moved))
        assert abs((ends[0] - ends[1]) / (2 * eps) - float(full[name][at])) < 1e-7, (name, at, reverse)
