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
