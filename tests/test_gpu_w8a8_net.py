"""The 8-bit pairs of 1x1 layers inside a network: each pair's outputs bit for bit from the pixels that it read."""
import numpy as np
import pytest

from oracle import w8a8 as ref
from posehip import _ffi, api_native, caffe_io, graph, synth
from test_gpu_net import CASES, _tiny_net

pytestmark = pytest.mark.gpu


def bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7fff + ((u >> 16) & 1)) & 0xffff0000
    return u.astype(np.uint32).view(np.float32)


def layer(op):
    """(int8 weights over the channels read, scales, bias, act, slope) of a plan's op"""
    w = op["weight"][:, :, 0, 0].astype(np.float64)
    m = op["cin_map"]
    w = np.where(m[None] >= 0, w[:, np.maximum(m, 0)], 0.0)
    q, s = ref.quantize_rows(w)
    slope = op["slope"]
    if slope is not None:
        slope = np.broadcast_to(slope, (op["cout"],))
    act = {_ffi.PH_ACT_NONE: "none", _ffi.PH_ACT_RELU: "relu", _ffi.PH_ACT_PRELU: "prelu"}[op["act"]]
    bias = op["bias"] if op["bias"] is not None else np.zeros(op["cout"], np.float32)
    return q, s, bias, act, slope


def check_pairs(engine, plan, B):
    """Every pair's network output and channel windows from the pixels in its input buffer; returns their number."""
    out = engine.net_out(B)
    n = 0
    for a, b in zip(plan.ops, plan.ops[1:]):
        if not (a.get("w8a8") and b.get("w8a8") and a["dst"] and a["dst"][0] == (b["in_buf"], b["in_coff"])):
            continue
        n += 1
        pad = plan.bufs[a["in_buf"]]["pad"]
        H, W = a["h"], a["w"]
        x = engine.get_buffer(a["in_buf"])[:B, pad:pad + H, pad:pad + W, a["in_coff"]:a["in_coff"] + a["cin_read"]]
        x = x.reshape(-1, a["cin_read"])
        l1, l2 = layer(a), layer(b)
        l2 = (l2[0][:, :a["cout"]],) + l2[1:]
        y = ref.feed_forward(x, l1, l2)
        if b["f32_coff"] >= 0:
            got = out[:, b["f32_coff"]:b["f32_coff"] + b["cout"]].transpose(0, 2, 3, 1).reshape(-1, b["cout"])
            assert np.array_equal(got, y), (a["name"], b["name"])
        for buf, coff in b["dst"]:
            d = engine.get_buffer(buf)[:B]
            p = plan.bufs[buf]["pad"]
            got = d[:, p:p + H, p:p + W, coff:coff + b["cout"]].reshape(-1, b["cout"])
            assert np.array_equal(got, bf16(y)), (a["name"], b["name"], buf)
            if p:   # the border stays zero
                d = d[..., coff:coff + b["cout"]]
                assert not d[:, :p].any() and not d[:, -p:].any() and not d[:, :, :p].any() and not d[:, :, -p:].any()
    return n


@pytest.mark.parametrize("case,pairs", [("dense_concat", 1), ("vgg_like", 0)])
@pytest.mark.parametrize("batch", [1, 3])
def test_small_nets(engine, case, pairs, batch):
    h, w, spec = CASES[case]
    net = _tiny_net(h, w, spec)
    weights = graph.random_weights(net, seed=3, out_gain=1.0)
    plan = graph.build_plan(net, weights, w8a8=True)
    engine.build(plan, 3)
    engine.preprocess(synth.synth_frames(2, batch, h, w), _ffi.PH_PRE_CV2)
    engine.forward(batch)
    assert check_pairs(engine, plan, batch) == pairs
    names = [k for k in engine.op_kernels() if k.startswith("w8_pair_kernel")]
    assert len(names) == pairs


@pytest.mark.parametrize("model,pairs", [("body25", 6), ("coco", 12)])
def test_whole_networks(engine, model, pairs):
    h, w = (184, 328) if model == "body25" else (96, 128)
    net = caffe_io.parse_prototxt(caffe_io.body25_prototxt(h, w) if model == "body25" else caffe_io.coco_prototxt(h, w))
    weights = graph.random_weights(net, seed=1, out_gain=1.0)
    plan = graph.build_plan(net, weights, w8a8=True)
    engine.build(plan, 2)
    frames = synth.synth_frames(5, 2, h, w)
    for _ in range(2):
        engine.preprocess(frames, _ffi.PH_PRE_CV2)
        engine.forward(2)
        assert check_pairs(engine, plan, 2) == pairs
    out = engine.net_out(2)
    assert np.isfinite(out).all()
    # without the flag nothing is in 8 bits, and the results are what they were
    plain = graph.build_plan(net, weights)
    engine.build(plain, 2)
    engine.preprocess(frames, _ffi.PH_PRE_CV2)
    engine.forward(2)
    assert not any(k.startswith("w8_pair") for k in engine.op_kernels())
    assert not np.array_equal(engine.net_out(2), out)


def test_refusals(engine):
    h, w, spec = CASES["dense_concat"]
    net = _tiny_net(h, w, spec)
    weights = graph.random_weights(net, seed=3)

    def build(mark):
        plan = graph.build_plan(net, weights)
        for o in plan.ops:
            if o["name"] in mark:
                o["w8a8"] = True
        engine.build(plan, 1)

    for mark in (["m6"], ["l2"], ["l1"], ["c0", "l1b"], ["a0"]):
        with pytest.raises(_ffi.PosehipError):
            build(mark)
    build(["m6", "l2"])
    bad = graph.build_plan(net, weights, w8a8=True)
    for o in bad.ops:
        if o["name"] == "m6":
            o["weight"] = o["weight"].copy()
            o["weight"][3, 5] = np.inf
    with pytest.raises(_ffi.PosehipError):
        engine.build(bad, 1)
    engine.build(graph.build_plan(net, weights, w8a8=True), 1)


def test_estimator_parameter():
    frames = synth.synth_frames(3, 1, 120, 160)
    outs = []
    for w8 in (False, True):
        pyop = api_native.PyOpenPoseNative(dict(posehip_random_weights=0, net_resolution="160x128", posehip_w8a8=w8))
        pyop.predict(frames[0])
        names = pyop.opWrapper._engine.op_kernels()
        assert any(k.startswith("w8_pair") for k in names) == w8
        outs.append(pyop.opWrapper._engine.net_out(1))
        pyop.opWrapper.close()
    assert np.isfinite(outs[1]).all() and not np.array_equal(outs[0], outs[1])
