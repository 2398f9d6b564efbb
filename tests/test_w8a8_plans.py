"""CPU: which pairs of 1x1 layers a plan marks for 8 bits."""
import pytest

from posehip import graph
from test_gpu_net import _tiny_net

CONVS = [("conv", "x", "image", 32, 3, "ReLU"), ("conv", "y", "image", 32, 3, "ReLU")]
NETS = {   # what the second layer reads beside the first one's output
    "nothing else": (CONVS[:1] + [("conv", "a", "x", 40, 1, "PReLU"), ("conv", "b", "a", 20, 1, None)], 1),
    "a later part": (CONVS + [("conv", "a", "y", 32, 1, "PReLU"), ("concat", "cat", ["a", "x"]), ("conv", "b", "cat", 20, 1, None)], 0),
    "a later part, odd widths": (CONVS + [("conv", "a", "y", 27, 1, "PReLU"), ("concat", "cat", ["a", "x"]), ("conv", "b", "cat", 20, 1, None)], 0),
    "an earlier part": (CONVS + [("conv", "a", "y", 32, 1, "PReLU"), ("concat", "cat", ["x", "a"]), ("conv", "b", "cat", 20, 1, None)], 0),
    "another 1x1 layer": (CONVS + [("conv", "c", "x", 24, 1, "ReLU"), ("conv", "a", "y", 32, 1, "PReLU"), ("concat", "cat", ["a", "c"]),
                                   ("conv", "b", "cat", 20, 1, None)], 0),
}


@pytest.mark.parametrize("case", sorted(NETS))
def test_a_pair_reads_only_its_first_layer(case):
    spec, pairs = NETS[case]
    net = _tiny_net(16, 24, spec)
    plan = graph.build_plan(net, graph.random_weights(net, seed=1), w8a8=True)
    assert sum(bool(o.get("w8a8")) for o in plan.ops) == 2 * pairs
