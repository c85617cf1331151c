"""The bounds that the GPU results of the recurrence are held to (test_gpu_sequence_precision.py): the formula's own results
lie inside, and those of a formula with a term missing do not.  No GPU."""
import pytest
import torch

import sequence_reference as ref
from test_gpu_sequence import BF16, offs, recurrence_inputs
from test_gpu_sequence_precision import held, recurrence_bounds


@pytest.mark.parametrize("name, term", [("dgate", "dl"), ("ddata", "dl"), ("dstate", "dl"), ("dgate", "state"), ("out", "state"),
                                        ("dgate", "x"), ("dgate", "dy"), ("ddata", "dy")])
def test_the_bounds_notice_a_missing_term(name, term):
  """Results without the state, the gradient of the last one, one row's data or gradient are beyond the bounds"""
  gate, data, state, dy, dl = recurrence_inputs([6, 400, 900], 8, BF16, 64)
  o = offs([6, 400, 900])
  want = recurrence_bounds(gate, data, o, state, False, dy, dl)
  held(want[name].to(BF16 if name in ("dgate", "ddata", "out") else torch.float32), want, name, BF16)
  if term == "dl":
    dl = None
  elif term == "state":
    state = None
  else:
    (data if term == "x" else dy)[700] = 0.0
  wrong = ref.recurrence(gate, data, o, state, False, dy, dl)
  with pytest.raises(AssertionError, match="over the bound"):
    held(wrong[name], want, name, BF16)
