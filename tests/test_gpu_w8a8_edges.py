"""posehip.w8a8 on the GPU at the edges of what its documents allow: the largest counts, kernels that only large products
take, padding that holds anything, tensors that are not what they look like."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from oracle import w8a8 as ref  # noqa: E402
from test_gpu_w8a8 import TYPES, make, rows, same, weights  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def w8():
    from posehip import w8a8
    return w8a8


def on_gpu(q, s, w, ws, bias):
    """The definition in torch, for sums below 2^24 (exact in f32 in any order); each operation is a kernel of its own."""
    assert q.shape[-1] * 127 * 127 < 1 << 24
    acc = torch.zeros(q.shape[0], w.shape[0], device="cuda")
    for k in range(q.shape[1]):
        acc += q[:, k:k + 1].float() * w[:, k].float()
    return acc * ws * s[:, None] + bias


@pytest.mark.parametrize("M,K,N", [(64 * 65535, 33, 5), (64 * 65535 + 1, 31, 16), (5_000_000, 31, 16)])
def test_rows_of_any_alignment_in_their_millions(w8, M, K, N):
    """More tokens than 65535 blocks of 64 hold."""
    rng = np.random.default_rng(K)
    w, ws, bias, _ = weights(rng, N, K)
    layer = make(w8, w, ws, bias)
    q = torch.randint(-127, 128, (M, K), dtype=torch.int8, device="cuda")
    s = torch.rand(M, device="cuda")
    y = w8.matmul(q, s, layer, dtype=torch.float32)
    c = [torch.from_numpy(a).cuda() for a in (w, ws, bias)]
    for a in range(0, M, 1 << 20):
        assert torch.equal(y[a:a + (1 << 20)], on_gpu(q[a:a + (1 << 20)], s[a:a + (1 << 20)], *c)), a


def test_threads_of_different_widths(w8):
    """First calls of a kernel at once, with different amounts of LDS."""
    import threading
    rng = np.random.default_rng(3)
    a = weights(rng, 512, 64)
    l1 = make(w8, a[0], a[1], a[2], "none")
    second = [weights(rng, n, 512) for n in (64, 48, 33, 17)]
    layers = [make(w8, *b[:3]) for b in second]
    x = rows(rng, 20500, 64, "f32")
    d = x.cuda()
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(3):
                y = w8.feed_forward(d, l1, layers[i])
            torch.cuda.current_stream().synchronize()
            got[i] = y.cpu()

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    for b, g in zip(second, got):
        same(g, ref.feed_forward(x.double().numpy(), (a[0], a[1], a[2], "none"), b[:3] + ("none", None)))


@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -1e38, 1e30])
@pytest.mark.parametrize("M,K,H,N", [(77, 100, 1, 21), (77, 100, 33, 21), (77, 100, 500, 21), (20100, 40, 33, 5), (77, 100, 600, 70), (9000, 64, 33, 300)])
def test_padding_of_parameters_may_be_anything(w8, M, K, H, N, junk):
    """Scale, bias and slope of the channels from n to the next multiple of 16."""
    rng = np.random.default_rng(H)
    a, b = weights(rng, H, K), weights(rng, N, H)
    x = rows(rng, M, K, "f32").cuda()
    l1, l2 = make(w8, a[0], a[1], a[2], "prelu", a[3]), make(w8, b[0], b[1], b[2], "prelu", b[3])
    want = w8.feed_forward(x, l1, l2), w8.linear(x, l1), w8.linear(x[:5], l1), w8.matmul(*w8.quantize_rows(x), l1)
    l1._par[:, H:] = junk
    l2._par[:, N:] = junk
    got = w8.feed_forward(x, l1, l2), w8.linear(x, l1), w8.linear(x[:5], l1), w8.matmul(*w8.quantize_rows(x), l1)
    for y, z in zip(got, want):
        assert torch.isfinite(z).all() and torch.equal(y, z)
    same(got[0], ref.feed_forward(x.double().cpu().numpy(), (a[0], a[1], a[2], "prelu", a[3]), (b[0], b[1], b[2], "prelu", b[3])))


def test_networks_whose_pairs_do_not_fit(engine):
    """They run as they do without 8 bits."""
    from posehip import _ffi, graph, synth
    from test_gpu_net import _tiny_net
    from test_w8a8_plans import NETS
    for spec, pairs in NETS.values():
        net = _tiny_net(16, 24, spec)
        w = graph.random_weights(net, seed=1, out_gain=1.0)
        outs = []
        for w8a8 in (False, True):
            engine.build(graph.build_plan(net, w, w8a8=w8a8), 2)
            engine.preprocess(synth.synth_frames(2, 2, 16, 24), _ffi.PH_PRE_CV2)
            engine.forward(2)
            outs.append(engine.net_out(2))
        assert np.array_equal(*outs) == (pairs == 0) and np.isfinite(outs[0]).all()


def test_outputs_over_scales(w8):
    rng = np.random.default_rng(5)
    w, ws, bias, _ = weights(rng, 20, 64)
    layer = make(w8, w, ws, bias)
    x = rows(rng, 30, 64, "f32").cuda()
    q, s = w8.quantize_rows(x)
    want = w8.matmul(q, s, layer, dtype=torch.float32)
    wide = torch.zeros(30 * 40 + 60, device="cuda")
    out = wide[30:30 + 1200].view(30, 40)[:, :20]
    for lo, ok in ((0, True), (1, False), (40, False), (1200, False), (1210, True), (1230, True)):
        sc = wide[lo:lo + 30]
        sc.copy_(s)
        if ok:
            w8.matmul(q, sc, layer, out=out)
            assert torch.equal(out, want) and torch.equal(sc, s)
        else:
            with pytest.raises(ValueError, match="scales"):
                w8.matmul(q, sc, layer, out=out)
    over = torch.zeros(30, 22, device="cuda")   # scales that are not side by side are copied first: their place may be written
    over[:, 3] = s
    assert torch.equal(w8.matmul(q, over[:, 3], layer, out=over[:, 1:21]), want)


def test_tangents_are_refused(w8):
    """Forward mode, also without gradients in the other direction; a detached tensor has none."""
    from torch.autograd import forward_ad as fw
    rng = np.random.default_rng(0)
    w, ws, bias, _ = weights(rng, 32, 32)
    layer = make(w8, w, ws, bias)
    x = torch.randn(4, 32, device="cuda")
    want = w8.linear(x, layer)
    q, s = w8.quantize_rows(x)
    with fw.dual_level():
        d, ds, out = (fw.make_dual(t, torch.ones_like(t)) for t in (x.clone(), s.clone(), torch.empty(4, 32, device="cuda")))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                for f in (lambda: w8.linear(d, layer), lambda: w8.quantize_rows(d), lambda: w8.feed_forward(d, layer, layer),
                          lambda: w8.matmul(q, ds, layer), lambda: w8.linear(x, layer, out=out)):
                    with pytest.raises(ValueError, match="no gradient"):
                        f()
        assert torch.equal(w8.linear(x, layer), want) and torch.equal(w8.linear(d.detach(), layer), want)
        W = torch.randn(20, 32, device="cuda")
        dual = w8.Layer(fw.make_dual(W, torch.ones_like(W)), bias=fw.make_dual(W[:, 0].contiguous(), torch.ones(20, device="cuda")))
        assert torch.equal(w8.linear(x, dual), w8.linear(x, w8.Layer(W, bias=W[:, 0])))
    assert torch.equal(w8.linear(x, layer), want)


def test_transforms_are_refused(w8):
    rng = np.random.default_rng(0)
    w, ws, bias, _ = weights(rng, 32, 32)
    layer = make(w8, w, ws, bias)
    x, W = torch.randn(4, 32, device="cuda"), torch.from_numpy(w).cuda()
    q, s = w8.quantize_rows(x)
    S, out = torch.from_numpy(ws).cuda(), torch.empty(4, 32, device="cuda")
    calls = [(x, lambda t: w8.linear(t, layer)), (x, lambda t: w8.quantize_rows(t)[1]), (x, lambda t: w8.feed_forward(t, layer, layer)),
             (s, lambda t: w8.matmul(q, t.expand(4), layer)), (x, lambda t: w8.linear(x, layer, out=t.expand(4, 32))),
             (S, lambda t: w8.Layer(W, scale=S, bias=t).packed), (x, lambda t: w8.Layer(t.expand(4, 32)).packed)]
    for t, f in calls:
        for transform in (torch.func.vmap(f), torch.func.functionalize(f), torch.func.grad(lambda v: f(v).sum()),
                          lambda v: torch.func.jvp(f, (v,), (torch.ones_like(v),))):
            with pytest.raises(ValueError):
                transform(t)
    with pytest.raises(ValueError):
        torch.func.vmap(lambda t: w8.matmul(t, s[0], layer))(q)
    with pytest.raises(ValueError):
        torch.func.functionalize(lambda t: w8.linear(x, layer) + t)(out)
    torch.func.vmap(lambda t: t + w8.linear(x, layer))(out)   # (x is no tensor of the transform's)
    assert torch.equal(w8.linear(x, layer), w8.matmul(q, s, layer, dtype=torch.float32))


def test_writes_into_tensors_that_a_gradient_needs_are_noticed(w8):
    rng = np.random.default_rng(0)
    w, ws, bias, _ = weights(rng, 32, 32)
    layer = make(w8, w, ws, bias)
    x = torch.randn(4, 32, device="cuda")
    q, s = w8.quantize_rows(x)
    for f in (lambda out: w8.linear(x, layer, out=out), lambda out: w8.feed_forward(x, layer, layer, out=out),
              lambda out: w8.matmul(q, s, layer, out=out)):
        buf = torch.rand(4, 40, device="cuda")
        p = torch.ones(4, 40, device="cuda", requires_grad=True)
        y = (buf * p).sum()
        f(buf[:, :32])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        y = (buf * p).sum()   # after the write: its values
        y.backward()
        assert torch.equal(p.grad, buf)
    with torch.inference_mode():
        out = torch.empty(4, 32, device="cuda")
        assert torch.equal(w8.linear(x, layer, out=out), w8.linear(x, layer))
    w8.linear(x, layer, out=out)   # (an inference tensor has no count)
    empty = torch.empty(0, 32, device="cuda")
    w8.linear(x[:0], layer, out=empty)
    assert empty._version == 0


def test_negated_views(w8):
    """Tensors whose memory holds the values' negatives: the imaginary part of a conjugate, and what torch makes like it."""
    rng = np.random.default_rng(0)
    w, ws, bias, _ = weights(rng, 20, 1)
    one, layer = make(w8, w, ws, bias), make(w8, *weights(rng, 64, 64)[:3])
    x = torch.randn(4, 1, dtype=torch.complex64, device="cuda").conj().imag
    y = torch._neg_view(torch.randn(4, 64, device="cuda"))
    q, s = w8.quantize_rows(y.clone())
    nq, ns = torch._neg_view(q), torch._neg_view(s)
    assert all(t.is_neg() for t in (x, y, nq, ns))
    for f, t, l in ((w8.linear, x, one), (w8.linear, y, layer)):
        assert torch.equal(f(t, l), f(t.clone(), l))
    assert torch.equal(w8.feed_forward(y, layer, layer), w8.feed_forward(y.clone(), layer, layer))
    assert torch.equal(w8.quantize_rows(y)[0], q)
    assert torch.equal(w8.matmul(nq, s, layer), w8.matmul(-q, s, layer)) and torch.equal(w8.matmul(q, ns, layer), w8.matmul(q, -s, layer))
    W = torch._neg_view(torch.randn(32, 64, device="cuda"))
    b = torch._neg_view(torch.randn(32, device="cuda"))
    assert torch.equal(w8.linear(y, w8.Layer(W, bias=b)), w8.linear(y, w8.Layer(W.clone(), bias=b.clone())))
    assert torch.equal(w8.Layer(nq, scale=s).packed, w8.Layer(-q, scale=s).packed)
    with pytest.raises(ValueError, match="negated"):
        w8.linear(y, layer, out=torch._neg_view(torch.empty(4, 64, device="cuda")))


def test_estimator_parameter_in_words_and_in_a_namespace():
    import argparse
    from posehip import api_native, synth
    frame = synth.synth_frames(3, 1, 120, 160)[0]
    args = argparse.Namespace(op_model_folder="/nonexistent/", op_model_pose="BODY_25", op_net_resolution="160x128", op_heatmaps_add_parts=False,
                              op_heatmaps_add_bkg=False, op_heatmaps_add_PAFs=False, op_heatmaps_scale=1, op_display=0, op_skel_thres=0.0,
                              op_max_true_body=8, op_patch_offset=2, posehip_random_weights=0)
    for value, on in (("0", False), ("yes", True), (False, False), (True, True), (None, False)):
        args.posehip_w8a8 = value
        pe = api_native.OpenPosePoseExtractor(args)
        pe.predict(frame, None)
        assert any(k.startswith("w8_pair") for k in pe.pyop.opWrapper._engine.op_kernels()) == on
        pe.pyop.opWrapper.close()
