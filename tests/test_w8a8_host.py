"""CPU: the oracle of the 8-bit layers against fractions, refusals of the C ABI and of posehip.w8a8 that need no GPU, and
the way row strides are taken apart."""
import ctypes as C
from fractions import Fraction

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from oracle import w8a8 as ref  # noqa: E402
from posehip import _ffi, w8a8  # noqa: E402


def nearest_even(f):
    lo = f.numerator // f.denominator
    r = f - lo
    return lo + (r > Fraction(1, 2) or (r == Fraction(1, 2) and lo % 2 == 1))


def test_oracle_quantisation_against_fractions():
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal((20, 40)).astype(np.float32), (np.arange(-20, 20)[None] * 0.5).astype(np.float32),
                        np.zeros((1, 40), np.float32), np.full((1, 40), 1e-44, np.float32)])
    x[20, 0] = 127 / 2   # a scale of exactly 1/2: every odd multiple of 1/4 ... is a border
    x[20, 1:] = (np.arange(39) - 19) * 0.25
    q, s = ref.quantize_rows(x)
    for i in range(x.shape[0]):
        for k in range(x.shape[1]):
            assert q[i, k] == nearest_even(Fraction(float(x[i, k])) / Fraction(float(s[i])))
    assert s[21] == np.float32(2.0 ** -126) and not q[21].any()
    q, s = ref.quantize_rows(np.array([[1, np.inf], [np.nan, 2], [3, 4]], np.float32))
    assert np.isnan(s[:2]).all() and not q[:2].any() and q[2, 1] == 127


def test_oracle_product_against_fractions():
    rng = np.random.default_rng(1)
    q, w = rng.integers(-128, 128, (4, 50)), rng.integers(-128, 128, (3, 50))
    s, ws, b = (rng.random(n).astype(np.float32) for n in (4, 3, 3))
    y = ref.matmul(q, s, w, ws, b)
    for m in range(4):
        for n in range(3):
            acc = int(sum(int(a) * int(c) for a, c in zip(q[m], w[n])))
            want = np.float32(np.float32(np.float32(np.float32(acc) * ws[n]) * s[m]) + b[n])
            assert y[m, n] == want
            exact = acc * Fraction(float(ws[n])) * Fraction(float(s[m])) + Fraction(float(b[n]))
            y64, mag = ref.matmul64(q, s, w, ws, b)
            assert abs(float(exact) - float(y[m, n])) <= 4 * 2.0 ** -24 * mag[m, n]
            assert abs(float(exact) - y64[m, n]) <= 4 * 2.0 ** -53 * mag[m, n]


def rows(n=(1, 1, 4), stride=(0, 0, 64)):
    return _ffi.PhRows((C.c_int64 * 3)(*n), (C.c_int64 * 3)(*stride))


def layer(n=16, k=64, act=0, slope=None):
    return _ffi.PhW8Layer(4096, 4096, None, slope, n, k, act)


def test_c_refusals():
    """Sizes, types and pointers are looked at before anything touches the GPU."""
    lib = _ffi.lib()
    st = (C.c_int64 * 3)(0, 0, 16)
    assert lib.ph_w8_packed_bytes(17, 65) == 32 * 128
    for n, k in ((0, 4), (4, 0), (4, w8a8.MAX_K + 1), ((1 << 20) + 1, 4), (-1, -1)):
        assert lib.ph_w8_packed_bytes(n, k) == -1
        assert lib.ph_w8_pack(0, None, 4096, 64, n, k, 4096) == -1
    assert lib.ph_w8_pack(0, None, None, 64, 4, 4, 4096) == -1 and lib.ph_w8_pack(0, None, 4096, 64, 4, 4, 4100) == -1
    assert lib.ph_w8_workspace(7, 4, 4, 0, 4) == -1 and lib.ph_w8_workspace(0, 1 << 31, 4, 0, 4) == -1
    assert lib.ph_w8_workspace(0, -1, 4, 0, 4) == -1 and lib.ph_w8_workspace(1, 4, 0, 0, 4) == -1
    q = lambda **k: lib.ph_w8_quantize_rows(0, None, k.get("x", 4096), k.get("t", 0), k.get("rows", rows()), k.get("k", 64),   # noqa: E731
                                            k.get("q", 4096), k.get("pitch", 64), k.get("s", 4096))
    assert q(t=3) == -1 and q(t=-1) == -1 and q(k=0) == -1 and q(k=(1 << 30) + 1, pitch=1 << 31) == -1 and q(pitch=48) == -1 and q(pitch=72) == -1 and q(q=4104) == -1
    assert q(x=None) == -1 and q(s=None) == -1 and q(q=None) == -1
    assert q(rows=rows((1, -1, 4))) == -1 and q(rows=rows((1, 1 << 16, 1 << 15))) == -1 and q(rows=rows((1 << 31, 1, 1))) == -1
    assert q(rows=rows((1, 0, 4)), x=None) == 0 and q(rows=rows((0, 1 << 40, 1 << 40))) == 0
    m = lambda **k: lib.ph_w8_matmul(0, None, k.get("q", 4096), k.get("rows", rows()), k.get("s", 4096), k.get("layer", layer()),   # noqa: E731
                                     k.get("out", 4096), k.get("t", 0), k.get("st", st), k.get("ws"), k.get("nws", 0))
    assert m(layer=layer(n=0)) == -1 and m(layer=layer(k=w8a8.MAX_K + 1)) == -1 and m(layer=layer(act=3)) == -1
    assert m(layer=layer(act=2)) == -1 and m(layer=None) == -1 and m(t=9) == -1 and m(q=None) == -1 and m(s=None) == -1
    assert m(out=None) == -1 and m(st=None) == -1 and m(rows=None) == -1
    odd = layer()
    odd.scale = 4104
    assert m(layer=odd) == -1
    r, big = rows((1, 1, 100000), (0, 0, 4096)), layer(n=640, k=4000)
    assert m(q=4097, rows=r, layer=big) == -3 and m(rows=rows((1, 1, 100000), (0, 0, 4097)), layer=big) == -3
    assert m(q=4097, rows=r, layer=big, ws=4096 + 16, nws=1 << 40) == -3
    assert b"workspace" in lib.ph_last_error()
    li = lambda **k: lib.ph_w8_linear(0, None, k.get("x", 4096), k.get("t", 0), k.get("rows", rows((1, 1, 100))), layer(k=4000), 4096, k.get("ot", 0),   # noqa: E731
                                      st, k.get("ws", 4096), k.get("nws", 1 << 20))
    assert li(x=None) == -1 and li(t=5) == -1 and li(ot=5) == -1 and li(ws=None) == -3 and li(nws=100) == -3
    ff = lambda a, b, **k: lib.ph_w8_feed_forward(0, None, 4096, 0, rows(), a, b, 4096, 0, st, 4096, k.get("nws", 1 << 20))   # noqa: E731
    assert ff(layer(n=16), layer(k=64)) == -1 and ff(layer(n=640), layer(k=640), nws=64) == -3
    assert ff(layer(n=64), layer(k=64, n=0)) == -1


def test_workspace_for_any_rows_holds_aligned_ones_too():
    lib = _ffi.lib()
    for m in (1, 5, 16, 33, 64, 65, 70, 130, 300, 1000, 5000, 100000):
        for k in (1, 15, 16, 31, 64, 301, 1001, 4001, 32500, w8a8.MAX_K):
            for n in (1, 16, 40, 187, 1000, 4096):
                assert lib.ph_w8_workspace(_ffi.PH_W8_MATMUL_ANY, m, k, 0, n) >= lib.ph_w8_workspace(_ffi.PH_W8_MATMUL, m, k, 0, n) >= 0


def test_python_refusals_without_a_gpu():
    x = torch.zeros(2, 4)
    for f in (lambda: w8a8.quantize_rows(x), lambda: w8a8.Layer(x), lambda: w8a8.Layer(x, act="tanh"),
              lambda: w8a8.linear(x, None), lambda: w8a8.matmul(x, x, None), lambda: w8a8.feed_forward(x, None, None)):
        with pytest.raises(ValueError):
            f()


def elements(r, m):
    n, s = list(r.n), list(r.stride)
    return [i * s[0] + j * s[1] + k * s[2] for i in range(n[0]) for j in range(n[1]) for k in range(n[2])][:m]


@pytest.mark.parametrize("view", ["whole", "window", "steps", "turned", "one", "expanded", "single", "vector"])
def test_rows_of_views(view):
    b = torch.arange(4 * 6 * 10 * 16).view(4, 6, 10, 16)
    v = {"whole": b, "window": b[1:3, 1:5, 2:9, 3:8], "steps": b[::2, ::3, 1::2], "turned": b.permute(2, 0, 1, 3), "one": b[:1, :, :1],
         "expanded": b[:, :1].expand(4, 7, 10, 16), "single": b[2:3, 3:4, 5:6], "vector": b[1, 2, 3]}[view]
    r, m = w8a8._rows(v.shape, v.stride())
    assert [v.storage_offset() + e for e in elements(r, m)] == v[..., 0].reshape(-1).tolist()
    out = torch.empty(v.shape[:-1] + (5,))
    r2, os, m2 = w8a8._out_rows(v.shape, v.stride(), out.shape, out.stride())
    assert m2 == m and [v.storage_offset() + e for e in elements(r2, m)] == v[..., 0].reshape(-1).tolist()
    assert elements(_ffi.PhRows(r2.n, os), m) == [i * 5 for i in range(m)]


def test_output_rows_that_overlap_are_refused():
    x = torch.empty(4, 8)
    for out in (torch.empty(1, 6).expand(4, 6), torch.empty(40).as_strided((4, 6), (5, 1)), torch.empty(8, 6).t()[:4, :6]):
        with pytest.raises(ValueError):
            w8a8._out_rows(x.shape, x.stride(), torch.Size((4, 6)), out.stride())
    w8a8._out_rows(x.shape, x.stride(), torch.Size((4, 6)), torch.empty(4, 9)[:, 2:8].stride())


def test_outputs_that_share_memory_with_the_rows_are_refused():
    b = torch.empty(6, 10, 64)
    flat = b.view(-1)

    def apart(x, out):
        return w8a8._apart(x.shape, x.stride(), x.element_size(), out.shape, out.stride(), out.element_size(), out.data_ptr() - x.data_ptr())

    half = flat.view(torch.bfloat16)
    for x, out, want in (
            (b, b, False), (b[0], b[0], False), (b[0], b[1], True), (b[1], b[0], True), (b[0, 0], b[0, 0], False),
            (b[..., :20], b[..., 20:40], True), (b[..., 20:40], b[..., :20], True), (b[..., :20], b[..., 19:40], False),
            (b[..., 1:20], b[..., 20:], True), (b[..., 30:50], b[..., 49:60], False), (b[:, ::2], b[:, 1::2], True), (b[:, :5], b[:, 5:], True),
            (b[:, 1:6], b[:, :5], False), (b[..., :20], b.transpose(0, 1)[..., 20:40].contiguous(), True),
            (b[:4, :4, :20], b[:4, :4].transpose(0, 1)[..., 20:40], False), (b[0, 0], b[0, 1], True), (b[0, 0, :8], b[0, 0, 8:9], True),
            (b[0, 0, :9], b[0, 0, 8:10], False), (b[0], half.view(6, 10, 128)[0, :, 64:], False), (b[:0], b[:0], True),
            (b[0, :1].expand(10, 64), b[0], False)):
        assert apart(x, out) == want, (x.shape, out.shape)
    wide = half.view(6, 10, 128)
    assert apart(b[..., :20], wide[..., 40:100]) and not apart(b[..., :20], wide[..., 39:100])


def test_plans_mark_the_pairs_that_fit():
    from posehip import caffe_io, graph
    for proto, pairs in ((caffe_io.body25_prototxt(64, 96), 6), (caffe_io.coco_prototxt(64, 96), 12)):
        net = caffe_io.parse_prototxt(proto)
        weights = graph.random_weights(net, seed=0)
        plan = graph.build_plan(net, weights)
        assert not any(o.get("w8a8") for o in plan.ops)
        plan8 = graph.build_plan(net, weights, w8a8=True)
        marked = [i for i, o in enumerate(plan8.ops) if o.get("w8a8")]
        assert len(marked) == 2 * pairs and all(b == a + 1 for a, b in zip(marked[::2], marked[1::2]))
        assert all(plan8.ops[i]["k"] == 1 for i in marked) and plan8.flops_per_frame() == plan.flops_per_frame()
        types = [d.type for d in plan8.to_ctypes()[1]]
        assert types.count(_ffi.PH_OP_CONV_W8A8) == 2 * pairs and [d.type for d in plan.to_ctypes()[1]].count(2) == 0
