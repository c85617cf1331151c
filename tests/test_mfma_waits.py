"""The wait states between a matrix instruction and the code that reads its result, in the assembly of attention.hip.
The compiler inserts them, but where a short block lies on one of two paths between the two it has counted along that path
only, and the other path read accumulators too early (wrong scores for the last key of a tile).  The source keeps
such branches away; this walks every path of every kernel and counts."""
import os
import re
import shutil
import subprocess

import pytest

from conftest import ROOT

# wait states from issue until a vector instruction may touch the result (16 and 8 passes)
NEED = {"v_mfma_f32_32x32x2_f32": 18, "v_mfma_f32_32x32x16_bf16": 11}


def registers(operands):
  out = set()
  for kind, a, b, c in re.findall(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)", operands):
    out |= {(kind, int(c))} if c else {(kind, i) for i in range(int(a), int(b) + 1)}
  return out


def early_uses(text):
  """(function, instruction) of every use that comes too early; the number of matrix instructions"""
  found, total = [], 0
  for name in re.findall(r"\n(_Z\S+):", text):
    at = text.index("\n" + name + ":")
    code, labels = [], {}
    for line in text[at:text.index(".Lfunc_end", at)].split("\n")[2:]:
      m = re.match(r"(\.LBB\S+):", line)
      if m:
        labels[m.group(1)] = len(code)
        continue
      line = line.split(";")[0].strip()
      if line and not line.startswith((".", "#")):
        code.append((line.split()[0], line))
    used = {}

    def regs(i):
      if i not in used:
        parts = code[i][1].split(None, 1)
        used[i] = registers(parts[1]) if len(parts) > 1 else set()
      return used[i]

    def after(i):
      op, line = code[i]
      if op == "s_endpgm":
        return []
      if op == "s_branch":
        return [labels[line.split()[1]]]
      return ([labels[line.split()[1]]] if op.startswith("s_cbranch") else []) + [i + 1]

    for i, (op, line) in enumerate(code):
      if not op.startswith("v_mfma"):
        continue
      total += 1
      need, result = NEED[op], registers(line.split(None, 1)[1].split(",")[0])
      seen, todo = {}, [(j, 0) for j in after(i)]
      while todo:
        j, waited = todo.pop()
        if j >= len(code) or waited >= need or seen.get(j, need) <= waited:
          continue
        seen[j] = waited
        o, l = code[j]
        if not o.startswith(("v_mfma", "s_")) and regs(j) & result:
          found.append((name, "%s: read after %d of %d wait states by: %s" % (line, waited, need, l)))
          break
        # (another matrix instruction holds the issue for at least four)
        waited += int(l.split()[1], 0) + 1 if o == "s_nop" else 4 if o.startswith("v_mfma") else 1
        todo += [(k, waited) for k in after(j)]
  return found, total


def test_the_walk_finds_an_early_read():
  text = """
_Zkernel:
; %bb.0:
\tv_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], 0
\ts_cbranch_vccnz .LBB0_2
; %bb.1:
\ts_nop 15
.LBB0_2:
\ts_nop WAIT
\tv_max_f32_e32 v30, v15, v15
\ts_endpgm
.Lfunc_end0:
"""
  assert len(early_uses(text.replace("WAIT", "8"))[0]) == 1
  assert early_uses(text.replace("WAIT", "9")) == ([], 1)


def test_no_kernel_reads_a_product_too_early(tmp_path):
  hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
  if shutil.which(hipcc) is None:
    pytest.skip("no hipcc")
  source = os.path.join(ROOT, "o-cnn_amd", "csrc", "attention.hip")
  flags = subprocess.run(["make", "-pn", "-C", os.path.dirname(source)], capture_output=True, text=True).stdout
  flags = re.search(r"^FLAGS := (.*)$", flags, re.M).group(1).split()
  out = str(tmp_path / "attention.s")
  subprocess.run([hipcc, *flags, "-S", "--cuda-device-only", source, "-o", out], check=True, capture_output=True)
  with open(out) as f:
    found, total = early_uses(f.read())
  assert total > 1000
  assert not found, found[:5]
