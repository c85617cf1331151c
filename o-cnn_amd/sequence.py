"""Operators along the node order of an octree level, re-exported by `nn`.

A level of a batched octree is one sequence per octree: its nodes lie in Morton order, octree after
octree.  `octree_offsets` says where each begins.  The reference has no counterpart: its feature
operators mix a node with its 27 neighbours only (octree/octree/octree_nn.cu:110-253).

Tensors are row-major, a row a node: [rows, heads, dim] or [rows, channels] (rows of a `to_rows` tensor
without its last one, or slices of one projection's output).  Tensors whose innermost axis is not
contiguous, or whose rows do not begin at the multiples of 16 bytes that attention reads, are copied.
All tensors of a call live on one GPU, which need not be the current one; work is queued on that GPU's
current stream.  A call takes at most 65535 sequences, and at most 2^31 - 1 entries on an axis.  The
forward and the gradient functions here launch kernels only and can be captured in a HIP graph; workspaces
are allocated per call, so captured graphs share none.
"""
import ctypes as C
import math

import torch

from . import lib as _lib
from .lib import OcnnError, AttentionParams
from .nn import _dtype_code, _ptr, _stream, _to_dev, octree_info, octree_property

__all__ = ["octree_offsets", "octree_positions", "rotary_frequencies", "octree_rotary", "octree_attention", "octree_attention_grad",
           "octree_recurrence", "octree_recurrence_grad"]

_POS_INT32, _POS_F32, _POS_XYZ = 0, 1, 2


# ---- checks -----------------------------------------------------------------------------------------
def _require(ok, message):
  if not ok:
    raise OcnnError(-1, message)


def _rows(t, name, ndim, like=None):
  """`t` with `ndim` axes, the innermost contiguous; of the type of `like` and on its device"""
  _require(torch.is_tensor(t) and t.dim() == ndim, "%s must be a tensor of %d axes" % (name, ndim))
  _require(max(t.shape) <= 2 ** 31 - 1, "%s is %s: an axis has at most 2147483647 entries" % (name, tuple(t.shape)))   # (C ints)
  _dtype_code(t)
  if like is not None:
    _require(t.dtype == like.dtype, "%s is %s, expected %s" % (name, t.dtype, like.dtype))
    _require(t.device == like.device, "%s is on %s, expected %s" % (name, t.device, like.device))
  if t.size(-1) > 1 and t.stride(-1) != 1:
    t = t.contiguous()
  return t


def _aligned(t):
  """rows and heads at multiples of 16 bytes and not too far apart for the kernels' offsets, copied where they are not"""
  e = 16 // t.element_size()
  if t.size(0) == 1 or t.size(1) == 1:       # (the stride of an axis of one is anything)
    t = t.as_strided(t.shape, [s if n > 1 else 0 for n, s in zip(t.shape, t.stride())][:2] + [1])
  if t.stride(0) >= 1 << 22 or t.stride(1) >= 1 << 22 or t.data_ptr() % 16 or t.stride(0) % e or t.stride(1) % e or (t.size(-1) > 1 and t.stride(-1) != 1):
    t = t.contiguous()
    if t.data_ptr() % 16:
      t = t.clone()
  return t


def _table(t, name, dtype, like, numel=None):
  _require(torch.is_tensor(t) and t.dim() == 1 and t.dtype == dtype, "%s must be a 1-D %s tensor" % (name, dtype))
  _require(t.device == like.device, "%s is on %s, expected %s" % (name, t.device, like.device))
  _require(numel is None or t.numel() == numel, "%s has %d entries, expected %s" % (name, t.numel(), numel))
  _require(t.numel() <= 2 ** 31 - 1, "%s has %d entries: at most 2147483647" % (name, t.numel()))
  return t.contiguous()


def _state(t, name, shape, like):
  if t is None:
    return None
  _require(torch.is_tensor(t) and t.dtype == torch.float32 and tuple(t.shape) == shape,
           "%s must be a float32 %s tensor" % (name, shape))
  _require(t.device == like.device, "%s is on %s, expected %s" % (name, t.device, like.device))
  return t.contiguous()


def _on_gpu(t):
  if not t.is_cuda:
    raise RuntimeError("o-cnn_amd needs a GPU: there is no CPU path (the tensors are on %s)" % t.device)


def _span(t):
  """first and last byte a tensor can touch"""
  if t.numel() == 0:
    return 0, 0
  far = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
  return t.data_ptr(), t.data_ptr() + (far + 1) * t.element_size()


def _apart(out, inputs, name):
  a, b = _span(out)
  for t in inputs:
    if t is None:
      continue
    c, d = _span(t)
    _require(b <= c or d <= a, "%s overlaps an input" % name)


def _own_rows(t, name):
  """a caller's output: its rows must not lie on each other"""
  _require(t.size(-1) <= 1 or t.stride(-1) == 1, "%s: the innermost axis must be contiguous" % name)
  need = 1
  for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda x: x[1]):
    _require(s >= need, "%s overlaps itself" % name)
    need = s * n


def _call(device, fn, *args):
  if device.index == torch.cuda.current_device():
    _lib.call(fn, *args, _stream())
  else:
    with torch.cuda.device(device):
      _lib.call(fn, *args, _stream())


def _i64(n):
  return C.c_int64(int(n))


_fast = None


def _compiled():
  """The compiled module's try_* functions (binding/ocnn_aten.cpp): the same calls of the same library where all
  tensors are ready as they are, for a third of the host time; None where the module is not built."""
  global _fast
  if _fast is None:
    import os
    _fast = _lib.aten() if os.path.exists(_lib.ATEN_PATH) else False
  return _fast


# ---- octree_offsets ---------------------------------------------------------------------------------
def octree_offsets(octree, depth, nempty=False):
  """Where the nodes (nempty: the non-empty nodes) of each octree of a batch begin at `depth`: int32
  [batch_size + 1] on the GPU, the last entry is their number.  Computed on the device, no wait."""
  octree = _to_dev(octree)
  info = octree_info(octree)
  out = torch.empty(info.batch_size + 1, dtype=torch.int32, device=octree.device)
  _call(octree.device, "ocnn_octree_offsets", _ptr(out), _ptr(octree), info.p, int(depth), int(bool(nempty)))
  return out


def octree_positions(octree, depth, nempty=False):
  """Packed coordinates (int64, 16 bits an axis) of the nodes (nempty: the non-empty nodes) of a level, in node
  order: what octree_rotary takes as positions."""
  octree = _to_dev(octree)
  xyz = octree_property(octree, "xyz", depth)
  if not nempty:
    return xyz
  count = octree_info(octree).nnum_nempty(depth)
  child = octree_property(octree, "child", depth).long()
  out = torch.empty(count + 1, dtype=xyz.dtype, device=xyz.device)     # (the last entry takes the empty nodes)
  out[torch.where(child >= 0, child, count)] = xyz
  return out[:count]


# ---- rotary positions -----------------------------------------------------------------------------
def rotary_frequencies(pairs, base=10000.0, device=None):
  """Radians a unit of position for each pair of channels, float64: an axis with n pairs gets
  base ** (-i / n), i = 0 .. n - 1."""
  _require(base > 0, "base %r" % (base,))
  rows = [[float(base) ** (-i / n) for i in range(n)] for n in map(int, pairs)]
  return torch.tensor([f for row in rows for f in row], dtype=torch.float64, device=device or "cuda")


def octree_rotary(data, positions, frequencies, pairs, interleaved=False, inverse=False, out=None):
  """Rotary positions with several axes: data [rows, heads, dim], `pairs[i]` pairs of channels for axis i.
  Pair p (the pairs of axis 0 first) turns by positions[row, axis] * frequencies[p]:
    (x, y) -> (x cos t - y sin t, x sin t + y cos t),
  channels (p, P + p) with P pairs in all, or (2 p, 2 p + 1) with interleaved=True.  Channels from 2 P on
  are copied.  inverse=True turns back: the gradient of the operator.
  positions: int32 or float32 [rows, axes] (at most 4 axes), or the packed coordinates that
  octree_property(octree, "xyz", depth) returns (int64 [rows], at most 3 axes).  The angle is formed in 64
  bits (frequencies: float64), so positions in the millions keep their phase.
  `out`: where the result goes; `data` itself, or a tensor that does not overlap it."""
  if out is None and _compiled():
    try:
      done = _fast.try_rotary(data, positions, frequencies, pairs, interleaved, inverse)
      if done is not None:
        return done
    except TypeError:        # an argument of another kind: named below
      pass
  data = _rows(data, "data", 3)
  rows, heads, dim = data.shape
  pairs = [int(n) for n in pairs]
  _require(1 <= len(pairs) <= 4, "pairs: 1 to 4 axes, got %d" % len(pairs))
  _require(min(pairs) >= 0 and 2 * sum(pairs) <= dim, "%s pairs need %d channels, a head has %d"
           % (pairs, 2 * sum(pairs), dim))
  frequencies = _table(frequencies, "frequencies", torch.float64, data, sum(pairs))
  _require(torch.is_tensor(positions) and positions.device == data.device, "positions must be a tensor on %s" % data.device)
  if positions.dtype == torch.int64:
    kind = _POS_XYZ
    _require(positions.dim() == 1 and positions.size(0) == rows and len(pairs) <= 3,
             "packed positions: int64 [%d], at most 3 axes" % rows)
    positions = positions.contiguous()
    stride = 1
  else:
    _require(positions.dtype in (torch.int32, torch.float32), "positions are int32, float32 or packed int64, got %s"
             % positions.dtype)
    kind = _POS_INT32 if positions.dtype == torch.int32 else _POS_F32
    _require(positions.dim() == 2 and positions.size(0) == rows and positions.size(1) >= len(pairs),
             "positions must be [%d, %d]" % (rows, len(pairs)))
    if positions.size(1) > 1 and positions.stride(1) != 1:
      positions = positions.contiguous()
    stride = positions.stride(0)
  if out is None:
    _on_gpu(data)
    out = torch.empty(data.shape, dtype=data.dtype, device=data.device)
  else:
    _require(torch.is_tensor(out) and out.shape == data.shape and out.dtype == data.dtype and out.device == data.device,
             "out must be a %s %s tensor on %s" % (tuple(data.shape), data.dtype, data.device))
    _own_rows(out, "out")
    same = out.data_ptr() == data.data_ptr() and out.stride() == data.stride()
    _apart(out, ([] if same else [data]) + [positions, frequencies], "out")
    _on_gpu(data)
  _call(data.device, "ocnn_octree_rotary", _ptr(out), _i64(out.stride(0)), _i64(out.stride(1)), _ptr(data),
        _i64(data.stride(0)), _i64(data.stride(1)), rows, heads, dim, _ptr(positions), kind, _i64(stride),
        _ptr(frequencies), (C.c_int * 4)(*pairs), len(pairs), int(bool(interleaved)), int(bool(inverse)), _dtype_code(data))
  return out


# ---- attention --------------------------------------------------------------------------------------
def _attention_params(q, k, v, q_offsets, k_offsets, k_lengths, left, right, sinks, scale, key_mask):
  q = _rows(q, "q", 3)
  k, v = _rows(k, "k", 3, q), _rows(v, "v", 3, q)
  _require(k.shape == v.shape, "k is %s, v is %s" % (tuple(k.shape), tuple(v.shape)))
  _require(k.size(2) == q.size(2), "q has %d channels a head, k has %d" % (q.size(2), k.size(2)))
  _require(k.size(1) > 0 and q.size(1) > 0 and q.size(1) % k.size(1) == 0,
           "%d query heads over %d key heads" % (q.size(1), k.size(1)))
  q_offsets = _table(q_offsets, "q_offsets", torch.int32, q)
  _require(q_offsets.numel() >= 2, "q_offsets needs an entry for each sequence and one more")
  if k_offsets is None:
    _require(k.size(0) == q.size(0), "%d query rows and %d key rows need k_offsets" % (q.size(0), k.size(0)))
    k_offsets = q_offsets
  else:
    k_offsets = _table(k_offsets, "k_offsets", torch.int32, q, q_offsets.numel())
  n_seq = q_offsets.numel() - 1
  if k_lengths is not None:
    k_lengths = _table(k_lengths, "k_lengths", torch.int32, q, n_seq)
  if key_mask is not None:
    _require(torch.is_tensor(key_mask) and key_mask.dtype == torch.bool and tuple(key_mask.shape) == (k.size(0),)
             and key_mask.device == q.device, "key_mask must be a bool [%d] tensor on %s" % (k.size(0), q.device))
    key_mask = key_mask.contiguous()
  if scale is None:
    scale = 1.0 / math.sqrt(max(q.size(2), 1))
  scale = float(scale)
  _require(math.isfinite(scale), "scale %r" % scale)
  q, k, v = _aligned(q), _aligned(k), _aligned(v)
  bound = 2 ** 31 - 1
  _require(-1 <= left <= bound and -1 <= right <= bound, "window %r, %r: -1 for no bound" % (left, right))
  _require(0 <= sinks <= bound, "%r sinks" % (sinks,))
  p = AttentionParams(q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), q.stride(1), k.stride(0), k.stride(1),
                      v.stride(0), v.stride(1), q_offsets.data_ptr(), k_offsets.data_ptr(),
                      k_lengths.data_ptr() if k_lengths is not None else 0, key_mask.data_ptr() if key_mask is not None else 0,
                      n_seq, q.size(0), k.size(0), q.size(1), k.size(1), q.size(2), int(left), int(right), int(sinks),
                      _dtype_code(q), scale)
  need, grad = C.c_size_t(), C.c_size_t()
  _lib.call("ocnn_attention_workspace_bytes", C.byref(p), C.byref(need), C.byref(grad))
  _on_gpu(q)
  return p, need.value, grad.value, q, (k, v, q_offsets, k_offsets, k_lengths, key_mask)


def _scratch(nbytes, device):
  return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def octree_attention(q, k, v, q_offsets, k_offsets=None, k_lengths=None, left=-1, right=-1, sinks=0, scale=None,
                     key_mask=None, out=None, return_lse=False):
  """Attention inside each sequence: q [rows_q, heads, dim], k and v [rows_k, kv_heads, dim] -> [rows_q, heads,
  dim].  Query head h reads key head h // (heads // kv_heads).  Sequence b owns the query rows q_offsets[b] ..
  q_offsets[b + 1] - 1 and the key rows k_offsets[b] .. (the same where k_offsets is None); k_lengths (int32
  [sequences]) says how many of the latter are keys, for a cache with room to grow.
  The queries are the last of a sequence's keys: query i stands at position p = i + keys - queries.  Key j is
  visible to it when j <= p + right and (j >= p - left or j < sinks), -1 for a bound that is absent
  (right=0: causal), and key_mask[row of j] (bool [rows_k]) holds.  A query that sees no key gets zeros; what
  invisible keys and values hold does not matter.
  dim: a multiple of 8 up to 128; heads // kv_heads and sinks: at most 64; scale: 1 / sqrt(dim) where None.
  `out`: where the result goes (rows of no sequence are left as they are; without `out` they are zero).
  return_lse=True returns (out, lse): lse [rows_q, heads] float32, the logarithm of each softmax's sum, which
  octree_attention_grad takes."""
  if out is None and _compiled():
    try:
      done = _fast.try_attention(q, k, v, q_offsets, k_offsets, k_lengths, left, right, sinks, scale, key_mask, return_lse)
      if done:
        return tuple(done) if return_lse else done[0]
    except TypeError:
      pass
  p, need, _, q, keep = _attention_params(q, k, v, q_offsets, k_offsets, k_lengths, left, right, sinks, scale, key_mask)
  fill = out is None
  if fill:
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
  else:
    _require(torch.is_tensor(out) and out.shape == q.shape and out.dtype == q.dtype and out.device == q.device,
             "out must be a %s %s tensor on %s" % (tuple(q.shape), q.dtype, q.device))
    _own_rows(out, "out")
    _apart(out, (q,) + keep, "out")
  lse = None
  if return_lse:             # (rows of no sequence: -inf, also where those of `out` are left alone)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    if not fill:
      lse.fill_(-math.inf)
  ws = _scratch(need, q.device)
  rows, heads = (s if n > 1 else 0 for n, s in zip(out.shape[:2], out.stride()))
  _call(q.device, "ocnn_octree_attention", _ptr(out), _i64(rows), _i64(heads), _ptr(lse), C.byref(p), int(fill), _ptr(ws),
        C.c_size_t(need))
  return (out, lse) if return_lse else out


def octree_attention_grad(grad_out, q, k, v, out, lse, q_offsets, k_offsets=None, k_lengths=None, left=-1, right=-1,
                          sinks=0, scale=None, key_mask=None):
  """Gradients of octree_attention with respect to q, k and v; `out` and `lse` are what the forward call with the
  same arguments returned.  Rows of no sequence and key rows that are no keys get zeros."""
  if _compiled():
    try:
      done = _fast.try_attention_grad(grad_out, q, k, v, out, lse, q_offsets, k_offsets, k_lengths, left, right, sinks, scale,
                                      key_mask)
      if done:
        return tuple(done)
    except TypeError:
      pass
  p, _, need, q, keep = _attention_params(q, k, v, q_offsets, k_offsets, k_lengths, left, right, sinks, scale, key_mask)
  out, grad_out = _rows(out, "out", 3, q), _rows(grad_out, "grad_out", 3, q)
  _require(out.shape == q.shape and grad_out.shape == q.shape, "out is %s, grad_out %s, expected %s"
           % (tuple(out.shape), tuple(grad_out.shape), tuple(q.shape)))
  lse = _require_lse(lse, q)
  out, grad_out = _aligned(out), _aligned(grad_out)
  grads = [torch.empty(t.shape, dtype=q.dtype, device=q.device) for t in (q, keep[0], keep[1])]
  ws = _scratch(need, q.device)
  strides = [a for g in grads for a in (_ptr(g), _i64(g.stride(0)), _i64(g.stride(1)))]
  _call(q.device, "ocnn_octree_attention_grad", *strides, _ptr(grad_out), _i64(grad_out.stride(0)),
        _i64(grad_out.stride(1)), _ptr(out), _i64(out.stride(0)), _i64(out.stride(1)), _ptr(lse), C.byref(p), _ptr(ws),
        C.c_size_t(need))
  return tuple(grads)


def _require_lse(lse, q):
  _require(torch.is_tensor(lse) and lse.dtype == torch.float32 and tuple(lse.shape) == tuple(q.shape[:2])
           and lse.device == q.device, "lse must be a float32 %s tensor on %s" % (tuple(q.shape[:2]), q.device))
  return lse.contiguous()


# ---- gated linear recurrence ------------------------------------------------------------------------
def _recurrence_args(gate, data, offsets, state, carries):
  data = _rows(data, "data", 2)
  gate = _rows(gate, "gate", 2, data)
  _require(gate.shape == data.shape, "gate is %s, data is %s" % (tuple(gate.shape), tuple(data.shape)))
  _require(data.size(1) > 0, "data has no channels")
  offsets = _table(offsets, "offsets", torch.int32, data)
  _require(offsets.numel() >= 2, "offsets needs an entry for each sequence and one more")
  n_seq = offsets.numel() - 1
  state = _state(state, "state", (n_seq, data.size(1)), data)
  carry, need, grad = C.c_int64(), C.c_size_t(), C.c_size_t()
  _lib.call("ocnn_recurrence_shape", data.size(0), data.size(1), n_seq, int(bool(carries)), C.byref(carry), C.byref(need), C.byref(grad))
  _on_gpu(data)
  return gate, data, offsets, state, n_seq, carry.value, need.value, grad.value


def octree_recurrence(gate, data, offsets, state=None, reverse=False, out=None, return_carries=False):
  """Gated linear recurrence along each sequence, channel by channel: gate and data [rows, channels],
    h_t = a_t h_{t-1} + (1 - a_t) data_t,  a = sigmoid(gate),
  from a sequence's first row to its last (reverse=True: from the last to the first), beginning with `state`
  (float32 [sequences, channels], zeros where None).  Returns (h, last): last = the state behind the last step
  (float32; of an empty sequence the one it began with), which the next call of a running sequence takes
  as `state`.  return_carries=True adds what octree_recurrence_grad needs: the states inside the sequences.
  `out`: where h goes (rows of no sequence are left as they are; without `out` they are zero)."""
  if out is None and _compiled():
    try:
      done = _fast.try_recurrence(gate, data, offsets, state, reverse, return_carries)
      if done:
        return tuple(done)
    except TypeError:
      pass
  gate, data, offsets, state, n_seq, carry_rows, need, _ = _recurrence_args(gate, data, offsets, state, return_carries)
  rows, channels = data.shape
  fill = out is None
  if fill:
    out = torch.empty(data.shape, dtype=data.dtype, device=data.device)
  else:
    _require(torch.is_tensor(out) and out.shape == data.shape and out.dtype == data.dtype and out.device == data.device,
             "out must be a %s %s tensor on %s" % (tuple(data.shape), data.dtype, data.device))
    _own_rows(out, "out")
    _apart(out, (gate, data, offsets, state), "out")
  last = torch.empty(n_seq, channels, dtype=torch.float32, device=data.device)
  carries = torch.empty(carry_rows, channels, dtype=torch.float32, device=data.device) if return_carries else None
  ws = _scratch(need, data.device)
  _call(data.device, "ocnn_octree_recurrence", _ptr(out), _i64(out.stride(0)), _ptr(last), _ptr(carries), _ptr(gate),
        _i64(gate.stride(0)), _ptr(data), _i64(data.stride(0)), _ptr(state), _ptr(offsets), n_seq, rows, channels,
        int(bool(reverse)), int(fill), _dtype_code(data), _ptr(ws), C.c_size_t(need))
  return (out, last, carries) if return_carries else (out, last)


def octree_recurrence_grad(grad_out, gate, data, offsets, carries, state=None, grad_last=None, reverse=False):
  """Gradients of octree_recurrence with respect to gate, data and state, from those of h (`grad_out`) and of
  the last state (`grad_last`, float32, zeros where None).  `carries` is what the forward call with the same
  arguments returned.  Rows of no sequence get zeros."""
  if _compiled():
    try:
      done = _fast.try_recurrence_grad(grad_out, gate, data, offsets, carries, state, grad_last, reverse)
      if done:
        return tuple(done)
    except TypeError:
      pass
  gate, data, offsets, state, n_seq, carry_rows, _, need = _recurrence_args(gate, data, offsets, state, True)
  rows, channels = data.shape
  grad_out = _rows(grad_out, "grad_out", 2, data)
  _require(grad_out.shape == data.shape, "grad_out is %s, expected %s" % (tuple(grad_out.shape), tuple(data.shape)))
  _require(carries is not None, "carries: the forward call returns them with return_carries=True")
  carries = _state(carries, "carries", (carry_rows, channels), data)
  grad_last = _state(grad_last, "grad_last", (n_seq, channels), data)
  grad_gate = torch.empty(data.shape, dtype=data.dtype, device=data.device)
  grad_data = torch.empty(data.shape, dtype=data.dtype, device=data.device)
  grad_state = torch.empty(n_seq, channels, dtype=torch.float32, device=data.device)
  ws = _scratch(need, data.device)
  _call(data.device, "ocnn_octree_recurrence_grad", _ptr(grad_gate), _i64(grad_gate.stride(0)), _ptr(grad_data),
        _i64(grad_data.stride(0)), _ptr(grad_state), _ptr(grad_out), _i64(grad_out.stride(0)), _ptr(grad_last), _ptr(gate),
        _i64(gate.stride(0)), _ptr(data), _i64(data.stride(0)), _ptr(state), _ptr(carries), _ptr(offsets), n_seq, rows,
        channels, int(bool(reverse)), _dtype_code(data), _ptr(ws), C.c_size_t(need))
  return grad_gate, grad_data, grad_state
