"""posehip.w8a8 on the GPU against oracle/w8a8.py: bit for bit where the definition fixes every rounding, and against 64
bits within the roundings that the definition has."""
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from oracle import w8a8 as ref  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def w8():
    from posehip import w8a8
    return w8a8


def rows(rng, M, K, t):
    """Rows of very different sizes, some of them special."""
    x = rng.standard_normal((M, K)).astype(np.float32) * np.exp(rng.standard_normal((M, 1))).astype(np.float32)
    x = torch.from_numpy(x).to(TYPES[t])
    if M >= 3:
        x[M // 2] = 0
        x[M - 1, : K - 1] = 0
    return x


def weights(rng, N, K):
    return (rng.integers(-127, 128, (N, K)).astype(np.int8), (rng.random(N) * 0.01 + 1e-4).astype(np.float32),
            rng.standard_normal(N).astype(np.float32), (rng.random(N) * 0.3).astype(np.float32))


def make(w8, w, ws, bias=None, act="none", slope=None):
    c = lambda a: None if a is None else torch.from_numpy(a).cuda()   # noqa: E731
    return w8.Layer(c(w), scale=c(ws), bias=c(bias), act=act, slope=c(slope) if act == "prelu" else None)


def same(got, want32):
    """got (any float type) is want32 (f32) rounded once to got's type, bit for bit; NaN in the same places"""
    want = torch.from_numpy(np.ascontiguousarray(want32)).to(got.dtype)
    got = got.detach().cpu()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    bad = (got != want) & ~nan
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} differ, first at {torch.nonzero(bad)[0].tolist()}"


# ---- rows -----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,K", [(1, 1), (2, 7), (5, 8), (3, 17), (4, 64), (7, 384), (9, 511), (257, 512), (3, 513), (6, 1001),
                                 (5, 2047), (5, 2048), (4, 2049), (3, 4100), (2, 8192), (2, 8199), (3, 32500)])
def test_quantize_rows(w8, t, M, K):
    x = rows(np.random.default_rng(M * 100003 + K), M, K, t)
    q, s = w8.quantize_rows(x.cuda())
    wq, ws = ref.quantize_rows(x.double().numpy())
    assert q.shape == x.shape and s.shape == (M,) and q.data_ptr() % 16 == 0
    assert np.array_equal(s.cpu().numpy(), ws)
    assert np.array_equal(q.cpu().numpy(), wq)


def test_quantize_borders_and_special_rows(w8):
    """Ties at every step, both signs; neighbours of ties; subnormal, largest, infinite and NaN rows."""
    k = np.arange(-126, 126)
    tie = ((k + 0.5) / 8).astype(np.float32)
    r = np.zeros((10, 512), np.float32)
    r[0, :252], r[0, 511] = tie, 127 / 8
    r[1, :252], r[1, 511] = np.nextafter(tie, np.float32(99)), 127 / 8
    r[2, :252], r[2, 511] = np.nextafter(tie, np.float32(-99)), -127 / 8
    r[3, ::2] = np.float32(1e-44)
    r[4] = np.linspace(-1, 1, 512, dtype=np.float32) * np.float32(1.4e-36)
    r[5] = np.linspace(-1, 1, 512, dtype=np.float32) * np.float32(3.4028235e38)
    r[6, 3] = np.inf
    r[7, 5] = np.nan
    r[8, 7] = -np.inf
    r[8, 9] = 1.0
    r[9] = np.float32(2.0) ** -126
    q, s = w8.quantize_rows(torch.from_numpy(r).cuda())
    wq, ws = ref.quantize_rows(r)
    assert np.array_equal(s.cpu().numpy(), ws, equal_nan=True)
    assert np.array_equal(q.cpu().numpy(), wq)
    assert set(np.nonzero(np.isnan(ws))[0]) == {6, 7, 8}
    assert np.array_equal(q.cpu().numpy()[0, :252] % 2, np.zeros(252))   # ties go to the even step


def test_quantize_many_values_near_borders(w8):
    """Products of the reciprocal round onto a border now and then: the quotient decides."""
    rng = np.random.default_rng(5)
    amax = (rng.random(4096) * 3 + 0.5).astype(np.float32)
    s = (amax.astype(np.float64) / 127).astype(np.float32)
    k = rng.integers(-126, 126, (4096, 64))
    x = ((k + 0.5) * s[:, None].astype(np.float64)).astype(np.float32)
    x[:, ::3] = np.nextafter(x[:, ::3], np.float32(9))
    x[:, 0] = amax
    q, sc = w8.quantize_rows(torch.from_numpy(x).cuda())
    wq, ws = ref.quantize_rows(x)
    assert np.array_equal(sc.cpu().numpy(), ws) and np.array_equal(q.cpu().numpy(), wq)


@pytest.mark.parametrize("e", [-126, -125, -124, -100, -30, -1, 0, 1, 60, 120])
@pytest.mark.parametrize("step", [-1, 0, 1])
def test_quantize_next_to_every_border(w8, e, step):
    """The float next to each border k + 1/2, and those beside it, down to scales whose half is no float any more."""
    rng = np.random.default_rng(e + 200)
    M = 512
    amax = (127 * (1 + rng.integers(0, 1 << 22, M) * 2.0 ** -22) * 2.0 ** e).astype(np.float32)
    s = np.maximum((amax.astype(np.float64) / 127).astype(np.float32), np.float32(2.0 ** -126))
    k = np.arange(-127, 127)[None] + 0.5
    x = (k * s[:, None].astype(np.float64)).astype(np.float32)
    if step:
        x = np.nextafter(x, np.float32(step * np.inf), dtype=np.float32)
    x = np.where(np.abs(x) < amax[:, None], x, amax[:, None])
    x[:, 100] = amax
    q, sc = w8.quantize_rows(torch.from_numpy(x).cuda())
    wq, ws = ref.quantize_rows(x)
    assert np.array_equal(sc.cpu().numpy(), ws) and np.array_equal(q.cpu().numpy(), wq)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_quantize_strided_rows(w8, t):
    rng = np.random.default_rng(3)
    base = rows(rng, 4 * 6 * 10, 136, t).cuda().view(4, 6, 10, 136)
    for v in (base[1:4, ::2, 2:9, 3:100], base[:, :, :, 8:136], base.permute(2, 0, 1, 3)[..., :131], base[0, 0], base[2, 3, 5],
              base[:, :1].expand(4, 5, 10, 136), base[..., :1]):
        q, s = w8.quantize_rows(v)
        wq, ws = ref.quantize_rows(v.double().cpu().numpy().reshape(-1, v.shape[-1]))
        assert q.shape == v.shape and s.shape == v.shape[:-1]
        assert np.array_equal(q.cpu().numpy().reshape(wq.shape), wq) and np.array_equal(s.cpu().numpy().reshape(-1), ws)


# ---- products ---------------------------------------------------------------------------------------------------------------

SIZES = [(1, 1, 1), (1, 16, 16), (1, 384, 512), (1, 4096, 1000), (2, 63, 17), (3, 64, 15), (4, 1000, 257), (15, 129, 31),
         (16, 128, 64), (17, 127, 65), (31, 2048, 48), (33, 65, 300), (61, 4100, 187), (64, 256, 256), (65, 257, 255),
         (100, 31, 1025), (127, 640, 129), (128, 512, 128), (200, 1537, 96), (255, 192, 320), (256, 384, 512), (257, 385, 513),
         (300, 16, 26), (1000, 288, 256), (1023, 96, 52), (2500, 130, 130), (5000, 70, 700), (9000, 384, 52)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("out,act", [("f32", "prelu"), ("bf16", "relu"), ("f16", "none")])
def test_matmul(w8, M, K, N, out, act):
    rng = np.random.default_rng(M * 7919 + K * 31 + N)
    q = rng.integers(-127, 128, (M, K)).astype(np.int8)
    s = np.exp(rng.standard_normal(M)).astype(np.float32) * np.float32(0.01 / K)
    w, ws, bias, slope = weights(rng, N, K)
    bias = None if act == "none" else bias
    y = w8.matmul(torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda(), make(w8, w, ws, bias, act, slope), dtype=TYPES[out])
    assert y.dtype == TYPES[out]
    same(y, ref.matmul(q, s, w, ws, bias, act, slope))
    # against 64 bits: sum -> f32, two products, one addition and the slope's product, half a step each, the result's type
    y64, mag = ref.matmul64(q, s, w, ws, bias, act, slope)
    tol = 5 * 2.0 ** -24 * mag * 1.001 + torch.finfo(TYPES[out]).eps / 2 * np.abs(y64) * 1.001 + {"f16": 2.0 ** -25}.get(out, 1e-40)
    assert (np.abs(y.double().cpu().numpy() - y64) <= tol).all()


def test_matmul_extremes(w8):
    """-128 on both sides at the longest K: the sum fills 31 bits; scales of every size; NaN and infinite scales stay in
    their row and channel."""
    K = w8.MAX_K
    q = np.full((3, K), -128, np.int8)
    q[1] = 127
    q[2, ::2] = 0
    w = np.full((17, K), -128, np.int8)
    w[3] = 127
    ws = np.full(17, 1.0, np.float32)
    ws[5], ws[6], ws[7] = np.nan, np.inf, 1e-38
    s = np.array([1.0, 1e-38, 3e38], np.float32)
    y = w8.matmul(torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda(), make(w8, w, ws), dtype=torch.float32)
    same(y, ref.matmul(q, s, w, ws))
    z = w8.matmul(torch.zeros(2, K, dtype=torch.int8, device="cuda"), torch.tensor([3e38, np.nan], device="cuda"),
                  make(w8, w[:2], np.array([3e38, 1], np.float32)), dtype=torch.float32)
    assert torch.equal(z[0].cpu(), torch.zeros(2)) and torch.isnan(z[1]).all()


def test_matmul_strides_and_alignments(w8):
    rng = np.random.default_rng(11)
    w, ws, bias, slope = weights(rng, 70, 100)
    layer = make(w8, w, ws, bias, "prelu", slope)
    big = torch.from_numpy(rng.integers(-127, 128, (3, 5, 12, 165)).astype(np.int8)).cuda()
    scales = torch.rand(3, 5, 12, device="cuda")
    flat = torch.from_numpy(rng.integers(-127, 128, 40 * 112 + 64).astype(np.int8)).cuda()
    views = [(big[..., :100], scales), (big[..., 3:103], scales), (big[1:, ::2, 1:10, 16:116], scales[1:, ::2, 1:10]),
             (big.permute(2, 0, 1, 3)[..., 5:105], scales.permute(2, 0, 1)), (big[:, :1, :, :100].expand(3, 5, 12, 100), scales),
             (flat[:40 * 112].view(40, 112)[:, :100], torch.rand(40, device="cuda")),
             (flat[16:16 + 40 * 112].view(40, 112)[:, 12:], torch.rand(40, device="cuda")), (big[1, 2, 3, :100], scales[1, 2, 3])]
    for q, s in views:
        y = w8.matmul(q, s, layer, dtype=torch.float32)
        assert y.shape == q.shape[:-1] + (70,)
        want = ref.matmul(q.cpu().numpy().reshape(-1, 100), s.cpu().numpy().reshape(-1), w, ws, bias, "prelu", slope)
        same(y.reshape(-1, 70), want)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,off", [(52, 0), (52, 8), (33, 3), (64, 1), (256, 32)])
def test_output_windows_leave_the_rest(w8, t, N, off):
    """A channel window of a wider buffer with a border around the pixels, as the network's buffers have it."""
    rng = np.random.default_rng(N + off)
    w, ws, bias, slope = weights(rng, N, 96)
    layer = make(w8, w, ws, bias, "relu")
    x = rows(rng, 2 * 9 * 13, 96, "bf16").cuda().view(2, 9, 13, 96)
    buf = torch.full((2, 11, 15, N + off + 5), 7.5, dtype=TYPES[t], device="cuda")
    out = buf[:, 1:10, 1:14, off:off + N]
    r = w8.linear(x, layer, out=out)
    assert r.data_ptr() == out.data_ptr()
    same(out.reshape(-1, N), ref.linear(x.double().cpu().numpy().reshape(-1, 96), w, ws, bias, "relu"))
    buf[:, 1:10, 1:14, off:off + N] = 7.5
    assert bool((buf == 7.5).all())


@pytest.mark.parametrize("M,K,N", [(1, 384, 512), (1, 4096, 4096), (3, 1000, 70), (8, 130, 2047), (16, 512, 33), (37, 1001, 2047),
                                   (64, 64, 64), (300, 288, 256), (3772, 96, 52)])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_linear_is_the_two_calls(w8, M, K, N, t):
    rng = np.random.default_rng(M + K + N)
    w, ws, bias, slope = weights(rng, N, K)
    x = rows(rng, M, K, t).cuda()
    if M > 4:
        x[1, K // 2], x[2, 0], x[4, K - 1] = float("nan"), float("inf"), float("-inf")
    layer = make(w8, w, ws, bias, "prelu", slope)
    y = w8.linear(x, layer)
    assert y.dtype == x.dtype
    z = w8.matmul(*w8.quantize_rows(x), layer, dtype=x.dtype)
    assert torch.equal(y.view(torch.uint8), z.view(torch.uint8))
    same(y, ref.linear(x.double().cpu().numpy(), w, ws, bias, "prelu", slope))
    if M > 4:
        assert torch.isnan(y[[1, 2, 4]]).all() and torch.isfinite(y[3]).all()


FF = [(1, 384, 512, 52), (2, 40, 33, 17), (5, 96, 128, 26), (63, 288, 256, 52), (64, 384, 512, 26), (129, 385, 511, 19),
      (300, 100, 65, 130), (1000, 384, 512, 52), (257, 1024, 512, 64), (130, 640, 1100, 300), (40, 33, 2048, 512)]


@pytest.mark.parametrize("M,K,H,N", FF)
@pytest.mark.parametrize("t,out,act", [("bf16", "f32", "prelu"), ("f32", "bf16", "relu"), ("f16", "f16", "none")])
def test_feed_forward(w8, M, K, H, N, t, out, act):
    rng = np.random.default_rng(M + K + H + N)
    a, b = weights(rng, H, K), weights(rng, N, H)
    x = rows(rng, M, K, t).cuda()
    if M > 4:
        x[1, 0] = float("nan")
    l1, l2 = make(w8, a[0], a[1], a[2], act, a[3]), make(w8, b[0], b[1], b[2])
    y = w8.feed_forward(x, l1, l2, dtype=TYPES[out])
    same(y, ref.feed_forward(x.double().cpu().numpy(), (a[0], a[1], a[2], act, a[3]), (b[0], b[1], b[2])))
    z = w8.linear(w8.linear(x, l1, dtype=torch.float32), l2, dtype=TYPES[out])
    assert torch.equal(torch.nan_to_num(y.float()), torch.nan_to_num(z.float()))


# where one kernel hands over to another: row lengths, tokens, channels
@pytest.mark.parametrize("M,K,N", [(64, 512, 300), (65, 512, 300), (64, 513, 40), (65, 513, 40), (2, 16384, 20), (2, 16385, 20), (100, 7, 40),
                                   (64, 7, 40), (70, 8, 64), (70, 9, 65), (8192, 64, 130), (8193, 64, 130), (8193, 8, 520),
                                   (8200, 512, 260), (8200, 129, 60), (8200, 384, 128), (8200, 385, 129), (300, 100, 4096),
                                   (300, 100, 4097), (8200, 40, 2049)])
def test_linear_borders(w8, M, K, N):
    rng = np.random.default_rng(M * 3 + K * 5 + N)
    w, ws, bias, slope = weights(rng, N, K)
    layer = make(w8, w, ws, bias, "prelu", slope)
    for t, out in (("bf16", "bf16"), ("f32", "f32")):
        x = rows(rng, M, K, t).cuda()
        x[M // 3, K // 2] = float("nan")
        wide = torch.zeros(M, K + 3, dtype=x.dtype, device="cuda")
        wide[:, 3:] = x
        y = w8.linear(x, layer, dtype=TYPES[out])
        z = w8.linear(wide[:, 3:], layer, dtype=TYPES[out])   # rows that start at odd places
        assert torch.equal(y.view(torch.uint8), z.view(torch.uint8))
        same(y, ref.linear(x.double().cpu().numpy(), w, ws, bias, "prelu", slope))


@pytest.mark.parametrize("M,K,H,N", [(20000, 24, 40, 20), (20001, 24, 40, 20), (20001, 512, 512, 64), (130, 512, 512, 65), (130, 513, 512, 64),
                                     (130, 512, 513, 64), (130, 7, 64, 16), (130, 8, 1, 1), (33, 500, 17, 33), (64, 96, 500, 48)])
def test_feed_forward_borders(w8, M, K, H, N):
    rng = np.random.default_rng(M + 7 * K + H + N)
    a, b = weights(rng, H, K), weights(rng, N, H)
    x = rows(rng, M, K, "f16").cuda()
    x[M // 2, 0] = float("inf")
    l1, l2 = make(w8, a[0], a[1], a[2], "relu"), make(w8, b[0], b[1], b[2], "prelu", b[3])
    y = w8.feed_forward(x, l1, l2, dtype=torch.float32)
    same(y, ref.feed_forward(x.double().cpu().numpy(), (a[0], a[1], a[2], "relu"), (b[0], b[1], b[2], "prelu", b[3])))


@pytest.mark.parametrize("M,K,N", [(1, 15, 20), (1, 16, 20), (5, 17, 33), (64, 31, 100), (65, 33, 100), (64, 4099, 100), (200, 47, 70), (3, 40001, 5),
                                   (700, 1001, 90), (64, 64, 64), (70, 4001, 40), (200, 2001, 33), (64, 1001, 40), (48, 31, 3000),
                                   (3000, 55, 100), (300, 16, 20), (33, 1040, 50)])
def test_matmul_of_rows_that_start_anywhere(w8, M, K, N):
    """Nothing behind the last row's end is read: the storage ends there, and what stands before and between is noise."""
    rng = np.random.default_rng(K + M)
    w, ws, bias, _ = weights(rng, N, K)
    layer = make(w8, w, ws, bias)
    s = torch.rand(M, device="cuda")
    for gap, lead in ((0, 0), (1, 5), (7, 3)):
        store = torch.from_numpy(rng.integers(-127, 128, lead + (M - 1) * (K + gap) + K).astype(np.int8)).cuda()
        q = store.as_strided((M, K), (K + gap, 1), lead)
        same(w8.matmul(q, s, layer, dtype=torch.float32), ref.matmul(q.cpu().numpy(), s.cpu().numpy(), w, ws, bias))


def test_long_offsets(w8):
    """Rows behind the first 2^31 and 2^32 elements, of the input and of the output."""
    M, K = 70001, 65536
    q = torch.zeros(M, K, dtype=torch.int8, device="cuda")
    rng = np.random.default_rng(2)
    at = [0, 32767, 32768, 65535, 65536, M - 1]
    part = rng.integers(-127, 128, (len(at), K)).astype(np.int8)
    q[at] = torch.from_numpy(part).cuda()
    s = torch.full((M,), 0.5, device="cuda")
    w, ws, bias, _ = weights(rng, 20, K)
    out = torch.zeros(M, 70000, dtype=torch.float16, device="cuda")
    w8.matmul(q, s, make(w8, w, ws, bias), out=out[:, 69980:])
    same(out[at, 69980:], ref.matmul(part, np.full(len(at), 0.5, np.float32), w, ws, bias))
    assert bool((out[:, :69980] == 0).all())
    del out, q
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[at] = torch.from_numpy(part).cuda().to(torch.bfloat16)
    qq, sc = w8.quantize_rows(x)
    wq, wsc = ref.quantize_rows(part.astype(np.float64))
    assert np.array_equal(qq[at].cpu().numpy(), wq) and np.array_equal(sc[at].cpu().numpy(), wsc)


# ---- use ----------------------------------------------------------------------------------------------------------------------

def test_layer_from_float_weights(w8):
    rng = np.random.default_rng(8)
    W = rng.standard_normal((52, 384, 1, 1)).astype(np.float32)
    x = rows(rng, 50, 384, "bf16")
    y = w8.linear(x.cuda(), w8.Layer(torch.from_numpy(W).cuda()), dtype=torch.float32)
    wq, ws = ref.quantize_rows(W.reshape(52, 384))
    same(y, ref.linear(x.double().numpy(), wq, ws))
    # and near the float product: each factor is off by at most half a step of its row (and the product of both)
    xf, Wf = x.double().numpy(), W.reshape(52, 384).astype(np.float64)
    sx = np.abs(xf).max(1)[:, None] / 254 * 1.0001
    sw = np.abs(Wf).max(1)[None] / 254 * 1.0001
    tol = np.abs(xf).sum(1)[:, None] * sw + np.abs(Wf).sum(1)[None] * sx + 384 * sx * sw + 1e-5
    assert (np.abs(y.double().cpu().numpy() - xf @ Wf.T) <= tol).all()
    Wt = torch.from_numpy(np.ascontiguousarray(W.reshape(52, 384).T)).cuda().t()   # K is not the fast axis
    assert torch.equal(w8.linear(x.cuda(), w8.Layer(Wt), dtype=torch.float32), y)


def test_no_rows(w8):
    rng = np.random.default_rng(1)
    w, ws, bias, _ = weights(rng, 20, 32)
    layer = make(w8, w, ws, bias)
    for shape in ((0, 32), (3, 0, 32)):
        x = torch.empty(shape, device="cuda")
        q, s = w8.quantize_rows(x)
        assert q.shape == shape and s.shape == shape[:-1]
        assert w8.matmul(q, s, layer).shape == shape[:-1] + (20,) and w8.linear(x, layer).shape == shape[:-1] + (20,)
        assert w8.feed_forward(x, layer, make(w8, *weights(rng, 7, 20)[:2])).shape == shape[:-1] + (7,)


def test_streams(w8):
    """Each stream's calls stand in that stream's order, with no wait of the host."""
    rng = np.random.default_rng(4)
    w, ws, bias, _ = weights(rng, 96, 384)
    layer = make(w8, w, ws, bias)
    xs = [rows(rng, 700, 384, "bf16") for _ in range(3)]
    want = [ref.linear(x.double().numpy(), w, ws, bias) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, st in zip(xs, streams):
        with torch.cuda.stream(st):
            d = x.cuda(non_blocking=True)
            d = (d * 2) * 0.5
            got.append(w8.linear(d, layer, dtype=torch.float32) + 0)
    torch.cuda.synchronize()
    for g, v in zip(got, want):
        same(g, v)


def test_threads(w8):
    rng = np.random.default_rng(6)
    w, ws, bias, _ = weights(rng, 130, 200)
    layer = make(w8, w, ws, bias)
    xs = [rows(rng, 40 + 30 * i, 200, "f32") for i in range(4)]
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            d = xs[i].cuda()
            for _ in range(20):
                y = w8.linear(d, layer)
            torch.cuda.current_stream().synchronize()
            got[i] = y.cpu()

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    for x, g in zip(xs, got):
        same(g, ref.linear(x.double().numpy(), w, ws, bias))


@pytest.mark.parametrize("M", [1, 37, 700])
def test_graphs(w8, M):
    """Two captured graphs, replayed in turn with new inputs and eager calls between them."""
    rng = np.random.default_rng(M)
    a, b = weights(rng, 512, 384), weights(rng, 52, 512)
    l1, l2 = make(w8, a[0], a[1], a[2], "prelu", a[3]), make(w8, b[0], b[1], b[2])
    big = make(w8, *weights(rng, 40, 5000)[:2])
    bufs, graphs, outs = [], [], []
    for g in range(2):
        x = torch.zeros(M, 384, dtype=torch.bfloat16, device="cuda")
        v = torch.zeros(M, 5000, dtype=torch.float32, device="cuda")
        w8.feed_forward(x, l1, l2), w8.linear(x, l1), w8.linear(v, big)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            q, s = w8.quantize_rows(x)
            outs.append((w8.matmul(q, s, l1, dtype=torch.float32), w8.feed_forward(x, l1, l2, dtype=torch.float32), w8.linear(v, big)))
        bufs.append((x, v))
        graphs.append(graph)
    for rep in range(4):
        for g in range(2):
            x, v = rows(rng, M, 384, "bf16"), rows(rng, M, 5000, "f32")
            bufs[g][0].copy_(x)
            bufs[g][1].copy_(v)
            graphs[g].replay()
            e = (w8.linear(bufs[g][0], l1, dtype=torch.float32), w8.feed_forward(bufs[g][0], l1, l2, dtype=torch.float32),
                 w8.linear(bufs[g][1], big))
            torch.cuda.synchronize()
            for o, w_ in zip(outs[g], e):
                assert torch.equal(o, w_)
            same(outs[g][0], ref.linear(x.double().numpy(), a[0], a[1], a[2], "prelu", a[3]))


def test_same_results_every_time(w8):
    rng = np.random.default_rng(9)
    w, ws, bias, _ = weights(rng, 187, 32500)
    layer = make(w8, w, ws, bias)
    x = rows(rng, 61, 32500, "f32").cuda()
    y = w8.linear(x, layer)
    for _ in range(5):
        assert torch.equal(w8.linear(x, layer), y)
    same(y, ref.linear(x.double().cpu().numpy(), w, ws, bias))


def test_first_calls_inside_a_capture(w8):
    """Nothing that a first call sets up needs a call outside of a capture."""
    rng = np.random.default_rng(12)
    a, b = weights(rng, 500, 300), weights(rng, 33, 500)
    l1, l2, l3 = make(w8, a[0], a[1], a[2], "relu"), make(w8, b[0], b[1], b[2]), make(w8, *weights(rng, 600, 2000)[:2])
    x, v = rows(rng, 21000, 300, "f16"), rows(rng, 400, 2000, "f32")
    dx, dv = x.cuda(), v.cuda()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = (w8.feed_forward(dx, l1, l2, dtype=torch.float16), w8.linear(dx, l1, dtype=torch.float16), w8.linear(dv, l3, dtype=torch.float16))
    for _ in range(3):
        g.replay()
        e = (w8.feed_forward(dx, l1, l2), w8.linear(dx, l1), w8.linear(dv, l3, dtype=torch.float16))
        torch.cuda.synchronize()
        assert all(torch.equal(p, r) for p, r in zip(o, e))


def test_outputs_beside_their_rows_and_over_them(w8):
    rng = np.random.default_rng(4)
    w, ws, bias, _ = weights(rng, 40, 40)
    layer = make(w8, w, ws, bias)
    buf = rows(rng, 300, 100, "f32").cuda()
    x, out = buf[:, :40], buf[:, 50:90]
    want = ref.linear(x.double().cpu().numpy(), w, ws, bias)
    w8.linear(x, layer, out=out)
    same(out, want)
    assert torch.equal(w8.feed_forward(x, layer, layer, out=out), w8.feed_forward(x, layer, layer))
    for f in (lambda: w8.linear(x, layer, out=x), lambda: w8.linear(x, layer, out=buf[:, 39:79]),
              lambda: w8.feed_forward(x[1:], layer, layer, out=x[:-1])):
        with pytest.raises(ValueError, match="shares memory"):
            f()


def test_a_device_that_is_not_there(w8):
    """A call for one is refused, and nothing of it is left for the next call."""
    from posehip import _ffi
    x = torch.ones(4, 64, device="cuda")
    rows, _ = w8._rows(x.shape, x.stride())
    for device in (torch.cuda.device_count() + 3, -1):
        assert _ffi.lib().ph_w8_quantize_rows(device, None, x.data_ptr(), _ffi.PH_F32, rows, 64, x.data_ptr(), 64, x.data_ptr()) == -1
        q, s = w8.quantize_rows(x)
        assert q.min() == 127 and s.max() > 0


def test_more_rows_than_a_launch_holds(w8):
    """Refused before anything is launched."""
    import ctypes as C
    from posehip import _ffi
    lib, buf = _ffi.lib(), torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    n = (1 << 31) - 1
    r = _ffi.PhRows((C.c_int64 * 3)(1, 1, n), (C.c_int64 * 3)(0, 0, 0))
    st = torch.cuda.current_stream().cuda_stream
    assert lib.ph_w8_quantize_rows(0, st, buf.data_ptr(), _ffi.PH_F32, r, 300, buf.data_ptr(), 304, buf.data_ptr()) == -1
    assert b"launch" in lib.ph_last_error()
    rng = np.random.default_rng(0)
    layer = make(w8, *weights(rng, 16, 64)[:2])
    os = (C.c_int64 * 3)(0, 0, 16)
    assert lib.ph_w8_matmul(0, st, buf.data_ptr(), r, buf.data_ptr(), layer.desc, buf.data_ptr(), 0, os, None, 0) == -1
    assert lib.ph_w8_linear(0, st, buf.data_ptr(), 0, r, layer.desc, buf.data_ptr(), 0, os, None, 0) == -1
    torch.cuda.synchronize()
    assert not buf.any()


def test_refusals(w8):
    rng = np.random.default_rng(0)
    w, ws, bias, slope = weights(rng, 20, 32)
    layer = make(w8, w, ws, bias)
    W = torch.from_numpy(w).cuda()
    S = torch.from_numpy(ws).cuda()
    x = torch.randn(4, 32, device="cuda")
    q, s = w8.quantize_rows(x)
    bad = [lambda: w8.Layer(W), lambda: w8.Layer(W.float(), scale=S), lambda: w8.Layer(W, scale=S[:3]),
           lambda: w8.Layer(W, scale=S.cpu()), lambda: w8.Layer(W, scale=S, act="gelu"), lambda: w8.Layer(W, scale=S, act="prelu"),
           lambda: w8.Layer(W, scale=S, slope=S), lambda: w8.Layer(W, scale=S, bias=S[:19]), lambda: w8.Layer(W.view(-1), scale=S),
           lambda: w8.Layer(torch.zeros(1, w8.MAX_K + 1, dtype=torch.int8, device="cuda"), scale=S[:1]),
           lambda: w8.Layer(W[:, :0], scale=S), lambda: w8.Layer(W.int(), scale=S), lambda: w8.Layer(W.double()),
           lambda: w8.linear(x[:, :31], layer), lambda: w8.linear(x.double(), layer), lambda: w8.linear(x.cpu(), layer),
           lambda: w8.linear(x.t().contiguous().t(), layer), lambda: w8.linear(x, W), lambda: w8.linear(x, layer, dtype=torch.int8),
           lambda: w8.linear(x, layer, out=torch.empty(4, 19, device="cuda")),
           lambda: w8.linear(x, layer, out=torch.empty(4, 20, device="cuda").cpu()),
           lambda: w8.linear(x, layer, out=torch.empty(20, 4, device="cuda").t()),
           lambda: w8.linear(x, layer, out=torch.empty(1, 20, device="cuda").expand(4, 20)),
           lambda: w8.linear(x, layer, out=torch.empty(4, 20, device="cuda"), dtype=torch.float16),
           lambda: w8.linear(x.clone().requires_grad_(), layer), lambda: w8.linear(x[0, 0], layer),
           lambda: w8.matmul(q, s[:3], layer), lambda: w8.matmul(q, s.double(), layer), lambda: w8.matmul(x, s, layer),
           lambda: w8.matmul(q[:, :16], s, layer), lambda: w8.matmul(q, s.cpu(), layer),
           lambda: w8.feed_forward(x, layer, layer), lambda: w8.quantize_rows(x[:, :0]), lambda: w8.quantize_rows(x.to(torch.int32)),
           lambda: w8.linear(torch.randn(3, 3, 3, 3, 64, device="cuda")[::2, ::2, ::2, ::2, :32], layer)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    with torch.no_grad():
        w8.linear(x.clone().requires_grad_(), layer)
    assert torch.equal(w8.linear(x, layer), w8.matmul(q, s, layer, dtype=torch.float32))
