"""The frequencies of the rotary positions where modules and trunks keep them: calls in graphs, after inference, on moved modules."""
import copy

import pytest
import torch

from test_gpu_sequence_use import mixer_params, tree  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def rows_of(oc, tree, depth, nempty):
  info = oc.nn.octree_info(tree)
  return info.nnum_nempty(depth) if nempty else info.nnum(depth)


def captured(call, data):
  """`call` in a graph, replayed with other inputs and eager calls between"""
  g = torch.cuda.CUDAGraph()
  torch.cuda.synchronize()
  with torch.cuda.graph(g):
    got = call()
  for i in range(4):
    data.normal_(generator=torch.Generator("cuda").manual_seed(i))
    want = call()
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want), i


@pytest.mark.parametrize("nempty", [False, True])
def test_mixer_in_a_graph(oc, tree, nempty):
  """frequencies copied from the host in every call kept the mixer out of graphs"""
  mix = mixer_params(64, 4, 2, torch.float32)
  x = torch.randn(1, 64, rows_of(oc, tree, 4, nempty), 1, device="cuda")
  oc.stacks.node_mixer(x, tree, 4, mix, nempty)
  captured(lambda: oc.stacks.node_mixer(x, tree, 4, mix, nempty), x)


def test_first_call_of_a_rotary_module_in_a_graph(oc):
  m = oc.OctreeRotary([3, 2, 3]).cuda()
  x = torch.randn(50, 2, 24, device="cuda")
  pos = torch.randint(0, 99, (50, 3), dtype=torch.int32, device="cuda")
  captured(lambda: m(x, pos), x)


def test_training_after_inference(oc):
  """the table of a first call in inference mode can be saved for a backward pass"""
  m = oc.OctreeRotary([8])
  x = torch.randn(50, 2, 24, device="cuda")
  pos = torch.randint(0, 99, (50, 1), dtype=torch.int32, device="cuda")
  with torch.inference_mode():
    m(x, pos)
  leaf = x.requires_grad_(True)
  m(leaf, pos).square().sum().backward()
  assert float((leaf.grad - 2 * x).detach().abs().max()) < 2.0 ** -18 * float(x.abs().max())    # (a rotation keeps the squares)


def test_moved_modules_keep_64_bits(oc):
  m = oc.OctreeRotary([4, 4], base=50.0)
  for moved in (m.cuda(), m.cuda().bfloat16(), copy.deepcopy(m).cuda().half(), m.cpu().to("cuda", torch.float32)):
    table, = moved._frequencies.values()
    assert table.dtype == torch.float64 and table.is_cuda
    assert torch.equal(table.cpu(), oc.nn.rotary_frequencies([4, 4], 50.0, device="cpu"))
