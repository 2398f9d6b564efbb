"""Every kernel that a product can take, at ragged sizes: bit for bit what the definition's f32 roundings give from sums in
64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from test_gpu_w8a8 import TYPES  # noqa: E402

pytestmark = pytest.mark.gpu

# (kernel as the launch names it, M, K, N)
TILE = "w8_tile_kernelILi{}ELi{}E"
PRODUCTS = [
    (TILE.format(256, 256), False, 776, 17, 15019), (TILE.format(256, 256), False, 8190, 1001, 2040),
    (TILE.format(256, 256), True, 163, 43475, 6255),
    (TILE.format(128, 128) + "Li2ELi4ELi2E", False, 135, 33, 32739), (TILE.format(128, 128) + "Li2ELi4ELi2E", False, 13699, 700, 841),
    (TILE.format(128, 128) + "Li2ELi4ELi2E", True, 137, 17005, 6197),
    (TILE.format(128, 128) + "Li2ELi4ELi3E", False, 9837, 1537, 259), (TILE.format(128, 128) + "Li2ELi4ELi3E", False, 29417, 2030, 65),
    (TILE.format(128, 128) + "Li2ELi4ELi3E", True, 3117, 14270, 68), (TILE.format(128, 128) + "Li2ELi4ELi3E", True, 401, 25437, 1553),
    (TILE.format(128, 64), False, 8369, 113, 2153), (TILE.format(128, 64), False, 50065, 100, 1),
    (TILE.format(128, 64), True, 3163, 15611, 7), (TILE.format(128, 64), True, 2315, 50000, 66),
    (TILE.format(64, 64), False, 3000, 2500, 129), (TILE.format(64, 64), True, 777, 20000, 200),
    ("w8_few_kernelILi1E", False, 9, 449, 295), ("w8_few_kernelILi1E", True, 5, 47072, 132),
    ("w8_few_kernelILi2E", False, 19, 433, 713), ("w8_few_kernelILi2E", True, 17, 10704, 149),
    ("w8_few_kernelILi3E", False, 43, 1696, 201), ("w8_few_kernelILi3E", True, 34, 36624, 46),
    ("w8_few_kernelILi4E", False, 62, 1791, 177), ("w8_few_kernelILi4E", True, 57, 73376, 19),
]
# two dimensions of rows that do not merge: M = a x b
SPLIT_M = {776: (8, 97), 135: (9, 15), 3117: (3, 1039), 3000: (30, 100), 57: (3, 19)}


@pytest.fixture(scope="module")
def w8():
    from posehip import w8a8
    return w8a8


def expected(q, s, w, ws, bias, act, slope, dtype):
    y = torch.mm(q.double(), w.double().t()).float()   # (whole numbers below 2^31: exact in 64 bits)
    y = y * ws
    y = y * s[:, None]
    y = y + bias
    if act == "relu":
        y = torch.where(y < 0, torch.zeros_like(y), y)
    elif act == "prelu":
        y = torch.where(y < 0, y * slope, y)
    return y.to(dtype)


def same(got, want):
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got.masked_fill(nan, 0), want.masked_fill(nan, 0))


@pytest.mark.parametrize("kernel,split,M,K,N", PRODUCTS, ids=[f"{M}x{K}-{N}" for _, _, M, K, N in PRODUCTS])
def test_products(w8, kernel, split, M, K, N):
    g = torch.Generator(device="cuda")
    g.manual_seed(M + K + N)
    pitch = (K + 15) // 16 * 16 + 16
    dims = SPLIT_M.get(M) or (M,)
    wide = torch.randint(-128, 128, dims[:-1] + (dims[-1] + 2, pitch), generator=g, device="cuda", dtype=torch.int8)
    q = wide[..., 1:-1, :K]   # a window: noise beside and behind the rows
    s = torch.rand(M, generator=g, device="cuda") * (1e-2 / K) + 1e-9
    s[M // 2] = float("nan")
    w = torch.randint(-128, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    ws, slope = torch.rand(N, generator=g, device="cuda") + 0.5, torch.rand(N, generator=g, device="cuda")
    bias = torch.randn(N, generator=g, device="cuda")
    flat = q.reshape(M, K)
    for out, act in (("f32", "prelu"), ("bf16", "relu"), ("f16", "none")):
        layer = w8.Layer(w, scale=ws, bias=bias, act=act, slope=slope if act == "prelu" else None)
        want = expected(flat, s, w, ws, bias, act, slope, TYPES[out])
        same(w8.matmul(q, s.view(dims), layer, dtype=TYPES[out]).reshape(M, N), want)
        buf = torch.full(dims + (N + 5,), 7.5, dtype=TYPES[out], device="cuda")
        same(w8.matmul(q, s.view(dims), layer, out=buf[..., 3:3 + N]).reshape(M, N), want)
        assert bool((buf[..., :3] == 7.5).all()) and bool((buf[..., 3 + N:] == 7.5).all())


@pytest.mark.parametrize("M,K,N", [(8190, 1001, 2040), (163, 43475, 6255), (9837, 1537, 259), (3117, 14270, 68), (8369, 513, 2153), (2315, 50000, 66)])
@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_linear_is_the_two_calls(w8, M, K, N, t):
    g = torch.Generator(device="cuda")
    g.manual_seed(M + K + N)
    x = (torch.randn(M, K, generator=g, device="cuda") * torch.exp(torch.randn(M, 1, generator=g, device="cuda"))).to(TYPES[t])
    x[M // 2, K // 3], x[M - 1, K - 1] = float("nan"), float("inf")
    layer = w8.Layer(torch.randn(N, K, generator=g, device="cuda"), bias=torch.randn(N, generator=g, device="cuda"), act="relu")
    y = w8.linear(x, layer)
    z = w8.matmul(*w8.quantize_rows(x), layer, dtype=x.dtype)
    assert torch.equal(y.view(torch.uint8), z.view(torch.uint8))
    assert torch.isnan(y[[M // 2, M - 1]]).all() and torch.isfinite(y[:M // 2]).all()


def test_every_scale_is_the_division(w8):
    """The scale of every float from 0 to the largest, against its division by 127 in 64 bits, rounded to 32 (which a
    division in 32 bits gives, 53 >= 2 * 24 + 2)."""
    m = torch.arange(1 << 23, dtype=torch.int32, device="cuda")
    for e in range(255):
        x = (m + (e << 23)).view(torch.float32).view(-1, 1)
        q, s = w8.quantize_rows(x)
        want = (x[:, 0].double() / 127).float().clamp_min(2.0 ** -126)
        assert torch.equal(s, want), e
        if e > 7:   # (smaller values are less than 127 of the smallest scale)
            assert int(q.min()) == 127


# ---- rows, and layers that quantise them ----------------------------------------------------------------------------------

# lanes of a row, M, K: more than one chunk of 8 values a lane, also past those kept in registers
QUANTIZE = [(8, 40001, 203), (16, 20001, 401), (32, 10001, 1001), (64, 5003, 2005), (256, 1101, 8001), (1024, 301, 32767), (1024, 7, 40001),
            (1024, 3, 100003)]


def quantized(x):
    """The definition in 64 bits: (whole numbers, scales f32)"""
    x = x.double()
    amax = x.abs().amax(1)
    ok = torch.isfinite(amax)
    s = (torch.where(ok, amax, 0.0) / 127).float().clamp_min(2.0 ** -126)
    q = torch.round(torch.where(ok[:, None], x, 0.0) / s.double()[:, None])   # (to even)
    return q, torch.where(ok, s, float("nan"))


def values(M, K, t, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = (torch.randn(M, K, generator=g, device="cuda") * torch.exp(torch.randn(M, 1, generator=g, device="cuda"))).to(TYPES[t])
    if M > 2:
        x[M // 2, K // 3] = float("nan")
        x[M - 1] = 0
        x[M - 1, K - 1] = -3
    return x


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lanes,M,K", QUANTIZE)
def test_quantize_rows(w8, lanes, M, K, t):
    x = values(M, K, t, M + K)
    for v in (x, torch.nn.functional.pad(x, (3, 2), value=1e4)[:, 3:3 + K]):
        q, s = w8.quantize_rows(v)
        wq, ws = quantized(v)
        same(s, ws)
        assert torch.equal(q.double(), wq)


def layer_and(w8, N, K, act, seed):
    """(Layer, the function that its definition is: 8-bit rows' whole numbers and scales -> f32)"""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    w = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    ws, slope = torch.rand(N, generator=g, device="cuda") * 0.01 + 1e-3, torch.rand(N, generator=g, device="cuda")
    bias = torch.randn(N, generator=g, device="cuda")
    layer = w8.Layer(w, scale=ws, bias=bias, act=act, slope=slope if act == "prelu" else None)
    return layer, lambda q, s: expected(q, s, w, ws, bias, act, slope, torch.float32)


# (kernel, M, K, N)
LINEAR = [("w8_few_kernelILi1E", 5, 300, 70), ("w8_few_kernelILi4E", 40, 500, 70), ("w8_rows_kernelILi2ELi4E", 4000, 300, 500),
          ("w8_rows_kernelILi4ELi8E", 8300, 500, 300), ("w8_rows_kernelILi4ELi4E", 8300, 130, 200), ("w8_rows_kernelILi4ELi2E", 8300, 64, 52),
          ("quantize_rows_kernel", 700, 2000, 300)]
# (kernel, M, K, H, N)
FEED_FORWARD = [("w8_pair_kernelILi2E", 300, 100, 200, 40), ("w8_pair_kernelILi4E", 20100, 200, 500, 33), ("w8_few_kernelILi4E", 50, 300, 600, 40),
                ("w8_rows_kernelILi2ELi4E", 300, 200, 700, 90)]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "prelu"])
def test_layers_of_every_type(w8, t, out, act):
    for _, M, K, N in LINEAR:
        x = values(M, K, t, M + K + N)
        layer, f = layer_and(w8, N, K, act, N)
        same(w8.linear(x, layer, dtype=TYPES[out]), f(*quantized(x)).to(TYPES[out]))
    for _, M, K, H, N in FEED_FORWARD:
        x = values(M, K, t, M + K + H + N)
        a, fa = layer_and(w8, H, K, act, H)
        b, fb = layer_and(w8, N, H, "relu" if act == "prelu" else "prelu", N)
        same(w8.feed_forward(x, a, b, dtype=TYPES[out]), fb(*quantized(fa(*quantized(x)))).to(TYPES[out]))
