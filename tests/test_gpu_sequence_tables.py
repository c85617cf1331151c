"""The frequencies of the rotary positions where modules and trunks keep them: calls in graphs."""
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
