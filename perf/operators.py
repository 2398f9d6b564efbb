"""The 8-bit matrix products of posehip.w8a8, measured: a product of 8-bit rows with a scale for each token (row) and
each output channel, the quantisation of float rows that feeds it, the two in one call, and two layers in one call.

Every case runs in a plain form too (elementary torch operations); both take the same inputs.

    s[m]    = max(f32(max_k |x[m,k]| / 127), 2^-126)
    q[m,k]  = round_half_even(x[m,k] / s[m])                      of the exact quotient
    y[m,n]  = act((f32(sum_k q[m,k] w[n,k]) * sw[n]) * s[m] + b[n])   each operation rounded to f32
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
TINY = 2.0 ** -126

# a drawn case's largest sizes: those of the largest listed case
MAX_MACS = 16384 * 4096 * 4096
MAX_X = 1 << 26
MAX_W = 1 << 25
MAX_Y = 1 << 26


def listed():
    return [
        # one token through a 1x1 layer's matrix: the smallest call, a launch
        dict(name="matmul 1 token 384x512", op="matmul", M=1, K=384, N=512, out="bf16", act="prelu", x="pixels"),
        # the 1x1 layer that widens a stage of BODY_25, 32 frames of 46 x 82 pixels
        dict(name="matmul 32 frames 384x512", op="matmul", M=120704, K=384, N=512, out="bf16", act="prelu", x="pixels"),
        # appearance features (25 x 50 x 26 values) of one frame's people against a gallery: a long sum, odd sizes
        dict(name="matmul features 61x187", op="matmul", M=61, K=32500, N=187, out="f32", act="none", x="features"),
        # a square product
        dict(name="matmul 4096 square", op="matmul", M=4096, K=4096, N=4096, out="bf16", act="none", x="tokens"),
        # one token through a wide layer: the weights are read once
        dict(name="linear 1 token 4096x4096", op="linear", M=1, K=4096, N=4096, out="bf16", x_type="bf16", act="none", x="tokens"),
        # a few tokens, odd sizes, half precision
        dict(name="linear 37 tokens 1001x2047", op="linear", M=37, K=1001, N=2047, out="f16", x_type="f16", act="relu", x="tokens"),
        # one frame through the first refinement stage's 1x1 layer
        dict(name="linear 1 frame 288x256", op="linear", M=3772, K=288, N=256, out="bf16", x_type="bf16", act="prelu", x="pixels"),
        # many tokens through a wide layer: the largest
        dict(name="linear 16384 tokens 4096x4096", op="linear", M=16384, K=4096, N=4096, out="bf16", x_type="bf16", act="relu", x="tokens"),
        # the rows of 32 frames' feature maps in 8 bits
        dict(name="quantize 32 frames 384", op="quantize", M=120704, K=384, x_type="bf16", x="pixels"),
        # few long rows of an odd length, 32 bits
        dict(name="quantize 300 rows 32500", op="quantize", M=300, K=32500, x_type="f32", x="features"),
        # the two 1x1 layers that close a stage of BODY_25: one frame, and 32
        dict(name="feed_forward 1 frame", op="feed_forward", M=3772, K=384, H=512, N=26, out="f32", x_type="bf16", act="prelu", x="pixels"),
        dict(name="feed_forward 32 frames", op="feed_forward", M=120704, K=384, H=512, N=52, out="bf16", x_type="bf16", act="prelu", x="pixels"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["matmul", "matmul", "linear", "linear", "quantize", "feed_forward"])
    while True:
        M = _log(rng, 1, 131072)
        act = rng.choice(["none", "relu", "prelu"])
        out = rng.choice(["bf16", "f16", "f32"])
        x_type = rng.choice(["bf16", "f16", "f32"])
        x = rng.choice(["pixels", "tokens"])
        K = _log(rng, 16, 32768)
        N = _log(rng, 16, 8192)
        if op == "quantize":
            if M * K <= MAX_X:
                return dict(op=op, M=M, K=K, x_type=x_type, x=x)
        elif op == "feed_forward":
            K, H, N = _log(rng, 32, 1024), _log(rng, 64, 2048), _log(rng, 16, 512)
            if M * K <= MAX_X and M * H <= MAX_X and M * H * (K + N) <= MAX_MACS:
                return dict(op=op, M=M, K=K, H=H, N=N, out=out, x_type=x_type, act=act, x=x)
        elif M * K <= MAX_X and N * K <= MAX_W and M * N <= MAX_Y and M * N * K <= MAX_MACS:
            d = dict(op=op, M=M, K=K, N=N, out=out, act=act, x=x)
            if op == "linear":
                d["x_type"] = x_type
            return d


# ---- inputs -------------------------------------------------------------------------------------------------------


def _values(g, kind, M, K):
    """f32 [M,K]: what such rows hold. "tokens": normal, each token with a size of its own and a few wide channels;
    "pixels": a layer's output after PReLU, each pixel with a size of its own; "features": maps of blobs, near zero
    almost everywhere, never negative."""
    dev = g.device
    x = torch.randn(M, K, generator=g, device=dev)
    size = torch.exp(torch.randn(M, 1, generator=g, device=dev))
    if kind == "tokens":
        wide = 1.0 + 7.0 * (torch.rand(1, K, generator=g, device=dev) < 0.01)
        return x * wide * size
    if kind == "pixels":
        return torch.where(x > 0, x, 0.2 * x) * size
    return torch.exp(-torch.rand(M, K, generator=g, device=dev) * 12.0)


def _weight(g, N, K, positive):
    """int8 [N,K] and a scale for each channel, as a model file in 8 bits holds them."""
    w = _values(g, "features", N, K) if positive else torch.randn(N, K, generator=g, device=g.device) * math.sqrt(2.0 / K)
    s = w.abs().amax(1) / 127
    return torch.round(w / s[:, None]).clamp(-127, 127).to(torch.int8), s


def _layer(g, N, K, act, positive=False):
    w, s = _weight(g, N, K, positive)
    d = dict(w=w, s=s, act=act, bias=None, slope=None)
    if not positive:
        d["bias"] = torch.randn(N, generator=g, device=g.device) * 0.1
    if act == "prelu":
        d["slope"] = torch.rand(N, generator=g, device=g.device) * 0.2 + 0.1
    if own:
        from posehip import w8a8
        d["layer"] = w8a8.Layer(w, scale=s, bias=d["bias"], act=act, slope=d["slope"])
    return d


def _import():
    """The package's folder is not on the path by itself."""
    import os
    import sys
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pose-estimation_amd")
    if at not in sys.path:
        sys.path.insert(0, at)


def prepare(case, seed):
    if own:
        _import()
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op, M, K = case["op"], case["M"], case["K"]
    st = dict(case=case)
    x = _values(g, case["x"], M, K)
    if op == "matmul":
        s = x.abs().amax(1) / 127
        st["q"], st["s"] = torch.round(x / s[:, None]).clamp(-127, 127).to(torch.int8), s
        st["layer"] = _layer(g, case["N"], K, case["act"], case["x"] == "features")
        return st
    st["x"] = x.to(DTYPES[case["x_type"]])
    if op == "linear":
        st["layer"] = _layer(g, case["N"], K, case["act"])
    elif op == "feed_forward":
        st["layer1"] = _layer(g, case["H"], K, case["act"])
        st["layer2"] = _layer(g, case["N"], case["H"], "none")
    return st


# ---- the plain form ------------------------------------------------------------------------------------------------


def _quantize(x):
    """(whole numbers in f32, scale f32 [M,1]). The quotient in 64 bits: in 32 it may round onto the border between two
    steps."""
    s = (x.abs().amax(1, keepdim=True).double() / 127).float().clamp_min(TINY)
    return torch.round(x.double() / s.double()).float(), s


def _act(y, layer):
    if layer["act"] == "relu":
        return torch.clamp_min(y, 0)
    if layer["act"] == "prelu":
        return torch.where(y < 0, y * layer["slope"], y)
    return y


def _product(q, s, layer):
    y = (q @ layer["w"].float().t()) * layer["s"] * s
    if layer["bias"] is not None:
        y = y + layer["bias"]
    return _act(y, layer)


def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        from posehip import w8a8
        if op == "matmul":
            return w8a8.matmul(st["q"], st["s"], st["layer"]["layer"], dtype=DTYPES[case["out"]])
        if op == "linear":
            return w8a8.linear(st["x"], st["layer"]["layer"], dtype=DTYPES[case["out"]])
        if op == "feed_forward":
            return w8a8.feed_forward(st["x"], st["layer1"]["layer"], st["layer2"]["layer"], dtype=DTYPES[case["out"]])
        q, s = w8a8.quantize_rows(st["x"])
        return q * s[:, None], s
    if op == "matmul":
        return _product(st["q"].float(), st["s"][:, None], st["layer"]).to(DTYPES[case["out"]])
    q, s = _quantize(st["x"])
    if op == "quantize":
        return q * s, s[:, 0]
    if op == "linear":
        return _product(q, s, st["layer"]).to(DTYPES[case["out"]])
    q, s = _quantize(_product(q, s, st["layer1"]))
    return _product(q, s, st["layer2"]).to(DTYPES[case["out"]])


def work(case):
    op, M, K = case["op"], case["M"], case["K"]
    if op == "quantize":  # the values come back in 32 bits
        return {"bytes": M * K * (BYTES[case["x_type"]] + 4) + 4 * M, "flops": 2 * M * K}
    N = case["N"]
    par = 12 if case["act"] == "prelu" else 8  # scale, bias, slope of a channel
    if op == "feed_forward":
        H = case["H"]
        return {"bytes": M * K * BYTES[case["x_type"]] + H * K + N * H + par * H + 8 * N + M * N * BYTES[case["out"]],
                "flops": 2 * M * H * (K + N)}
    x = M * K + 4 * M if op == "matmul" else M * K * BYTES[case["x_type"]]
    return {"bytes": x + N * K + par * N + M * N * BYTES[case["out"]], "flops": 2 * M * N * K}


# ---- 64 bits ---------------------------------------------------------------------------------------------------------


def _rounded(v):
    """64-bit values, each rounded to the nearest 32-bit one."""
    return v.to(torch.float32).to(torch.float64)


def _exact_rows(x):
    x = x.to(torch.float64)
    scale = torch.maximum(_rounded(x.abs().max(dim=1).values / 127.0), torch.tensor(TINY, dtype=torch.float64, device=x.device))
    t = x / scale.unsqueeze(1)
    below = torch.floor(t)
    part = t - below
    up = (part > 0.5) | ((part == 0.5) & (torch.remainder(below, 2) == 1))
    return below + up.to(torch.float64), scale


def _exact_sums(q, layer):
    w = layer["w"].to(torch.float64)
    return torch.cat([torch.mm(p, w.t()) for p in torch.split(q, 8192)])


def _exact_layer(q, scale, layer, held=False):
    """`held`: the layer's result as the definition holds it between two layers, rounded to 32 bits at each step."""
    r = _rounded if held else (lambda v: v)
    y = r(r(r(_exact_sums(q, layer)) * layer["s"].to(torch.float64)[None]) * scale[:, None])
    if layer["bias"] is not None:
        y = r(y + layer["bias"].to(torch.float64)[None])
    if layer["act"] == "relu":
        y = y * (y > 0)
    elif layer["act"] == "prelu":
        y = torch.maximum(y, torch.zeros_like(y)) + r(torch.minimum(y, torch.zeros_like(y)) * layer["slope"].to(torch.float64)[None])
    return y


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "matmul":
        return _exact_layer(st["q"].to(torch.float64), st["s"].to(torch.float64), st["layer"])
    q, scale = _exact_rows(st["x"])
    if op == "quantize":
        return q * scale[:, None], scale
    if op == "linear":
        return _exact_layer(q, scale, st["layer"])
    q, scale = _exact_rows(_exact_layer(q, scale, st["layer1"], held=True))
    return _exact_layer(q, scale, st["layer2"])
