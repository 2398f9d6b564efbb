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


@pytest.mark.parametrize("value,on", [(True, True), (False, False), (None, False), (0, False), (1, True), ("0", False), ("False", False),
                                      ("no", False), ("1", True), ("true", True), ("Yes", True)])
def test_the_parameter_in_words(value, on):
    """What the estimators hand to build_plan."""
    from posehip import api_native, api_opencv, utils
    assert utils.as_bool(value) is on
    seen = []
    for module in (api_native, api_opencv):
        build_plan, module.graph.build_plan = module.graph.build_plan, lambda *a, **k: seen.append(k["w8a8"])
        try:
            if module is api_native:
                w = api_native.Wrapper()
                w.params = dict(posehip_w8a8=value)
                w._engine = type("E", (), {"build": lambda *a: None})()
                w._ensure(160, 128, 1)
            else:
                p = api_opencv.PyOpenPoseOpenCV.__new__(api_opencv.PyOpenPoseOpenCV)
                with pytest.raises(FileNotFoundError):
                    p.load("/nonexistent", "/nonexistent", w8a8=value)
                seen.append(p._w8a8)
        finally:
            module.graph.build_plan = build_plan
    assert seen == [on, on]


def test_a_parameter_that_is_no_word():
    from posehip import api_native
    with pytest.raises(ValueError, match="on or off"):
        api_native.PyOpenPoseNative(dict(posehip_random_weights=0, posehip_w8a8="maybe"))
