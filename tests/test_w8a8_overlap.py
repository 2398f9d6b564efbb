"""CPU: outputs that share memory with the scales that a product reads."""
import random

import pytest

torch = pytest.importorskip("torch")
from posehip import w8a8  # noqa: E402


def clear(scale, out):
    return w8a8._clear_of(scale.numel() * 4, out.shape, out.stride(), out.element_size(), out.data_ptr() - scale.data_ptr())


def test_outputs_over_scales():
    b = torch.zeros(20, 10, 64)
    f = b.view(-1)
    half = f.view(torch.bfloat16)
    for scale, out, want in (
            (f[:20], b[:, 0], False), (b[19, 9, 44:], b[:19].reshape(190, 64), True), (f[:10], b[0], False), (f[64:74], b[:, 0], True),
            (f[63:73], b[:, 0], False), (f[50:60], b[:, 0, :50], True), (f[50:60], b[:, 0, :51], False), (f[100:150], b[:, 1:3, 10:20], False),
            (f[84:138], b[:, 1:3, 10:20], True), (f[84:139], b[:, 1:3, 10:20], False), (f[:74], b[:, 1:3, 10:20], True), (f[:75], b[:, 1:3, 10:20], False),
            (f[-40:], b[..., :24], True), (f[-41:], b[..., :24], False), (f[:0], b, True), (f[:5], b[:0], True), (f[2:3], f[2:3], False),
            (f[3:4], f[2:3], True), (f[2:3], half[4:5], False), (f[2:3], half[6:7], True), (f[2:3], half[3:4], True), (f[2:700], f[4:5], False),
            (f[0:700], b.transpose(0, 1)[..., 60:], False)):
        assert clear(scale, out) == want, (scale.shape, scale.storage_offset(), out.shape, out.stride())


def test_against_marked_bytes():
    rng = random.Random(0)
    seen = [0, 0]
    for _ in range(3000):
        f = torch.zeros(400)
        n = [rng.randint(1, 4) for _ in range(rng.randint(0, 3))] + [rng.randint(1, 6)]
        t = rng.choice([torch.float32, torch.float16])
        stride, reach = [1], n[-1]
        for k in reversed(n[:-1]):
            stride.insert(0, reach + rng.randint(0, 3))
            reach += (k - 1) * stride[0]
        if reach > 300:
            continue
        order = list(range(len(n) - 1))
        rng.shuffle(order)
        out = f.view(t).as_strided(n, stride, rng.randint(0, 40)).permute(order + [len(n) - 1])
        m = rng.randint(1, 20)
        at = rng.randint(0, 400 - m) if rng.random() < 0.3 else rng.randint(0, 60)
        out.fill_(1)
        want = not f.view(torch.int32)[at:at + m].any()
        assert clear(f[at:at + m], out) == want
        seen[want] += 1
    assert min(seen) > 300
