"""Layers in 8-bit integers: products of int8 rows with int8 weights, a scale for each token (row: a pixel, a feature
vector) and each output channel.  What a 1x1 convolution, or any other matrix product of a network, computes when the
network runs in 8 bits; ``cv2.dnn``'s quantised networks do the same per channel on the CPU.

::

    layer = Layer(weight, bias=bias, act="prelu", slope=slope)      # once: weight [N,K] float or int8 + scale
    y = linear(x, layer)                                            # x [..,K] float -> [..,N]
    q, s = quantize_rows(x)                                         # once, for several layers that read x
    y1, y2 = matmul(q, s, layer1), matmul(q, s, layer2)
    y = feed_forward(x, layer1, layer2)                             # two layers, in one kernel where they fit

    s[m]   = max(f32(max_k |x[m,k]| / 127), 2^-126)      q[m,k] = round_half_even(x[m,k] / s[m])   (exact quotient)
    y[m,n] = act((f32(sum_k q[m,k] w[n,k]) * ws[n]) * s[m] + bias[n])

The sum is an exact 32-bit integer (K <= 131071), each later operation is rounded to f32, the result once to its type;
so ``linear(x, l)`` is ``matmul(*quantize_rows(x), l)`` and ``feed_forward(x, a, b)`` is
``linear(linear(x, a, dtype=torch.float32), b)``, both bit for bit, whatever the sizes.  A row with a NaN or an infinity
gives NaN outputs and touches no other row.  There are no gradients: inputs and outputs that ask
for one, or carry a tangent (forward mode), are refused (a Layer takes a parameter's values as they are); so are the tensors that
torch.func's transforms hand out.

Tensors are CUDA tensors of f32 / f16 / bf16 with the values of a row consecutive (last stride 1) and any other strides;
leading dimensions that do not merge into three are refused.  Work is put on torch's current stream of the tensors'
device, waits for nothing, and can be captured into a graph; a tensor (a layer's weights among them) that is used on
another stream than the one it was made on has to stay alive until that stream is done with it, as with any torch
operation.  All arithmetic happens in libposehip.so.
"""
import ctypes as C
from functools import lru_cache

import torch
from torch.autograd import forward_ad

from . import _ffi

_TYPES = {torch.float32: _ffi.PH_F32, torch.float16: _ffi.PH_F16, torch.bfloat16: _ffi.PH_BF16}
_ACTS = {"none": _ffi.PH_ACT_NONE, "relu": _ffi.PH_ACT_RELU, "prelu": _ffi.PH_ACT_PRELU}
MAX_K = 131071


# torch.cuda.current_stream().cuda_stream without the Stream object around it (0.1 against 1.9 us a call)
_raw_stream = torch._C._cuda_getCurrentRawStream


def _merge(shape, stride):
    """Leading dimensions as few as they go: [(n, stride)], outermost first."""
    dims = []
    for n, s in zip(shape, stride):
        if n == 1:
            continue
        if dims and dims[-1][1] == n * s:
            dims[-1] = (dims[-1][0] * n, s)
        else:
            dims.append((n, s))
    return dims


@lru_cache(maxsize=4096)
def _rows(shape, stride):
    """(ph_rows, number of rows) of a tensor [.., K] of this shape and these strides."""
    if stride[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"the values of a row must be consecutive (last stride 1), got strides {stride}")
    m = 1
    for n in shape[:-1]:
        m *= n
    r = _ffi.PhRows()
    dims = _merge(shape[:-1], stride[:-1]) if m else [(0, 0)]
    if len(dims) > 3:
        raise ValueError(f"rows of shape {tuple(shape)}, strides {stride} do not merge into three dimensions")
    dims = [(1, 0)] * (3 - len(dims)) + dims
    for i, (n, s) in enumerate(dims):
        r.n[i], r.stride[i] = n, s
    return r, m


@lru_cache(maxsize=4096)
def _out_rows(in_shape, in_stride, shape, stride):
    """ph_rows of the input and int64[3] strides of the output over the same three dimensions, and the number of rows."""
    if stride[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"the values of an output row must be consecutive (last stride 1), got strides {stride}")
    if in_stride[-1] != 1 and in_shape[-1] > 1:
        raise ValueError(f"the values of a row must be consecutive (last stride 1), got strides {in_stride}")
    m = 1
    for n in shape[:-1]:
        m *= n
    dims = []          # (n, input stride, output stride), merged where both merge
    for n, s, o in zip(shape[:-1], in_stride[:-1], stride[:-1]):
        if n == 1:
            continue
        if dims and dims[-1][1] == n * s and dims[-1][2] == n * o:
            dims[-1] = (dims[-1][0] * n, s, o)
        else:
            dims.append((n, s, o))
    reach = shape[-1]
    for n, o in sorted(((n, o) for n, _, o in dims), key=lambda d: d[1]):
        if m and o < reach:
            raise ValueError(f"output rows of shape {tuple(shape)}, strides {stride} overlap")
        reach = (n - 1) * o + reach
    if not m:
        dims = [(0, 0, 0)]
    if len(dims) > 3:
        raise ValueError(f"rows of shape {tuple(shape)}, strides {in_stride} do not merge into three dimensions")
    dims = [(1, 0, 0)] * (3 - len(dims)) + dims
    r, os = _ffi.PhRows(), (C.c_int64 * 3)()
    for i, (n, s, o) in enumerate(dims):
        r.n[i], r.stride[i], os[i] = n, s, o
    r.by_16 = all(s % 16 == 0 for _, s, _ in dims)   # (of 8-bit rows)
    return r, os, m


@lru_cache(maxsize=4096)
def _apart(shape, stride, size, out_shape, out_stride, out_size, diff):
    """Whether an output that starts diff bytes behind an input shares no byte with it, as far as that is easily told: it ends
    before, starts after, or both are parts of one wider buffer (the same strides) that do not meet."""
    if 0 in shape or 0 in out_shape:
        return True
    end = sum((n - 1) * s for n, s in zip(shape, stride)) * size + size
    out_end = sum((n - 1) * s for n, s in zip(out_shape, out_stride)) * out_size + out_size
    if diff >= end or diff + out_end <= 0:
        return True
    dims = [(s * size, n) for n, s in zip(shape[:-1], stride[:-1]) if n > 1]
    if dims != [(s * out_size, n) for n, s in zip(out_shape[:-1], out_stride[:-1]) if n > 1] or any(s == 0 for s, _ in dims):
        return False
    dims.sort(reverse=True)
    width, out_width = shape[-1] * size, out_shape[-1] * out_size

    def meet(diff, dims):   # some row of the output, diff + k . strides behind some row of the input, shares a byte with it
        if not dims:
            return -out_width < diff < width
        (s, n), rest = dims[0], dims[1:]
        reach = sum(t * (m - 1) for t, m in rest) + max(width, out_width)
        low, high = max(1 - n, -((reach + diff) // s)), min(n - 1, (reach - diff) // s)
        return high - low > 8 or any(meet(diff + k * s, rest) for k in range(low, high + 1))

    return not meet(diff, dims)


@lru_cache(maxsize=4096)
def _clear_of(size, out_shape, out_stride, out_size, diff):
    """Whether an output of rows that do not overlap, diff bytes behind one piece of `size` bytes, shares no byte with it."""
    if 0 in out_shape or not size:
        return True
    dims = sorted(((s * out_size, n) for n, s in zip(out_shape[:-1], out_stride[:-1]) if n > 1), reverse=True)

    def meet(low, high, dims):   # bytes low .. high - 1, from the output's first on, hold one of a row's
        if not dims:
            return low < out_shape[-1] * out_size and high > 0
        (s, n), rest = dims[0], dims[1:]
        a, b = max(low // s, 0), min((high - 1) // s, n - 1)
        return b - a > 1 or any(meet(low - k * s, high - k * s, rest) for k in range(a, b + 1))   # (between two: a whole step)

    return not meet(-diff, size - diff, dims)


@lru_cache(maxsize=4096)
def _plan(shape, stride, n):
    """_out_rows for a new, contiguous output of n values a row, and that output's shape."""
    out = tuple(shape[:-1]) + (n,)
    ostride, step = [], 1
    for d in reversed(out):
        ostride.append(step)
        step *= max(d, 1)
    return _out_rows(shape, stride, out, tuple(reversed(ostride))) + (out,)


@lru_cache(maxsize=4096)
def _workspace(op, m, k, h, n):
    b = _ffi.lib().ph_w8_workspace(op, m, k, h, n)
    if b < 0:
        _ffi.check(-1, "ph_w8_workspace")
    return b


def _wants_gradient(t):
    """In either direction: a tensor that requires one, or that carries a tangent."""
    if t.requires_grad and torch.is_grad_enabled():
        return True
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


_transforms = torch._C._functorch.maybe_current_level


def _check_memory(*tensors):
    """The transforms of torch.func hand out tensors without memory of their own."""
    for t in tensors + (torch.empty(0),):
        if t is not None and torch._C._functorch.is_functorch_wrapped_tensor(t):
            raise ValueError("8-bit layers read and write memory: the transforms of torch.func do not go through them")


def _check_x(x, k, what):
    if not x.is_cuda or x.dtype not in _TYPES:
        raise ValueError(f"{what} must be a CUDA tensor of f32, f16 or bf16, got {x.dtype} on {x.device}")
    shape = x.shape
    if not shape or (k is not None and shape[-1] != k):
        raise ValueError(f"{what} must be [.., {k}], got {tuple(x.shape)}")
    if _wants_gradient(x):
        raise ValueError("8-bit layers have no gradient: call them under torch.no_grad() or detach their inputs")


@lru_cache(maxsize=4096)
def _q_shape(shape):
    return tuple(shape[:-1]) + ((shape[-1] + 15) // 16 * 16,), tuple(shape[:-1])


def quantize_rows(x):
    """x [.., K] float -> (q int8 [.., K], scale f32 [..]); x ~ q * scale[.., None].  q's rows start at multiples of 16
    bytes (a view of a wider buffer where K is no multiple of 16)."""
    _check_x(x, None, "x")
    if x.is_neg():
        x = x.resolve_neg()
    if _transforms() is not None:
        _check_memory(x)
    shape, device = x.shape, x.device
    k = shape[-1]
    if k < 1:
        raise ValueError("rows of no values have no scale")
    rows, m = _rows(shape, x.stride())
    qshape, lead = _q_shape(shape)
    pitch = qshape[-1]
    q = torch.empty(qshape, dtype=torch.int8, device=device)
    scale = torch.empty(lead, dtype=torch.float32, device=device)
    if m:
        _ffi.check(_ffi.lib().ph_w8_quantize_rows(device.index, _raw_stream(device.index), x.data_ptr(), _TYPES[x.dtype], rows, k,
                                                  q.data_ptr(), pitch, scale.data_ptr()), "ph_w8_quantize_rows")
    return (q if pitch == k else q[..., :k]), scale


class Layer:
    """Weights of a layer, laid out once for the matrix instructions.

    weight: [N,K] (or [N,K,1,1], a 1x1 convolution's) CUDA tensor, float (then quantised per channel as
    ``quantize_rows`` does) or int8 with ``scale`` f32 [N].  bias [N]; act "none" / "relu" / "prelu" with slope [N] or
    [1].  The inputs are not kept."""

    def __init__(self, weight, scale=None, bias=None, act="none", slope=None):
        if act not in _ACTS:
            raise ValueError(f"act must be one of {sorted(_ACTS)}, got {act!r}")
        if not weight.is_cuda:
            raise ValueError("weight must be a CUDA tensor")
        if _transforms() is not None:
            _check_memory(weight, scale, bias, slope)
        weight = weight.detach().resolve_neg()
        if weight.dim() == 4 and tuple(weight.shape[2:]) == (1, 1):
            weight = weight[:, :, 0, 0]
        if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
            raise ValueError(f"weight must be [N,K] or [N,K,1,1], got {tuple(weight.shape)}")
        n, k = weight.shape
        if k > MAX_K:
            raise ValueError(f"K = {k}: sums of more than {MAX_K} products can overflow 32 bits")
        if weight.stride(1) != 1:
            weight = weight.contiguous()
        if weight.dtype == torch.int8:
            if scale is None:
                raise ValueError("an int8 weight needs the scale of each channel")
            q = weight
        else:
            if scale is not None:
                raise ValueError("scale goes with an int8 weight")
            q, scale = quantize_rows(weight)
        if (act == "prelu") != (slope is not None):
            raise ValueError("slope goes with act='prelu'")
        dev = weight.device
        lib = _ffi.lib()
        nbytes = lib.ph_w8_packed_bytes(n, k)
        if nbytes < 0:
            _ffi.check(-1, "ph_w8_packed_bytes")
        par = torch.zeros(3, (n + 15) // 16 * 16, dtype=torch.float32, device=dev)
        for i, (name, v) in enumerate((("scale", scale), ("bias", bias), ("slope", slope))):
            if v is None:
                continue
            v = v.detach()
            if v.device != dev or not v.is_floating_point() or (tuple(v.shape) != (n,) and not (i == 2 and v.numel() == 1)):
                raise ValueError(f"{name} must be a float tensor [{n}] on {dev}, got {v.dtype} {tuple(v.shape)} on {v.device}")
            par[i, :n] = v.reshape(-1) if i == 2 else v
        self.packed = torch.empty(nbytes, dtype=torch.int8, device=dev)
        self.n, self.k, self.act, self.device = n, k, act, dev
        self._par = par
        _ffi.check(lib.ph_w8_pack(dev.index, _raw_stream(dev.index), q.data_ptr(), q.stride(0) if n > 1 else k, n, k,
                                  self.packed.data_ptr()), "ph_w8_pack")
        row = par.stride(0) * 4
        self.desc = _ffi.PhW8Layer(self.packed.data_ptr(), par.data_ptr(), par.data_ptr() + row if bias is not None else None,
                                   par.data_ptr() + 2 * row if slope is not None else None, n, k, _ACTS[act])
        if not torch.cuda.is_current_stream_capturing():   # a layer can be used on any stream once it exists
            torch.cuda.current_stream(dev).synchronize()


def _check_layer(layer, x):
    if not isinstance(layer, Layer):
        raise ValueError(f"a w8a8.Layer is wanted, got {type(layer).__name__}")
    if layer.device != x.device:
        raise ValueError(f"the layer is on {layer.device}, the rows on {x.device}")


# autograd's count of writes: a tensor that was saved for a gradient and then written by a kernel is noticed
_written = torch.autograd.graph.increment_version


def _output(x, n, out, dtype, default):
    """(out, ph_rows of x, strides of out, number of rows)"""
    if out is None:
        dtype = dtype or default
        if dtype not in _TYPES:
            raise ValueError(f"dtype must be f32, f16 or bf16, got {dtype}")
        rows, ostride, m, shape = _plan(x.shape, x.stride(), n)
        return torch.empty(shape, dtype=dtype, device=x.device), rows, ostride, m
    shape = x.shape[:-1] + (n,)
    if out.shape != shape or out.device != x.device or out.dtype not in _TYPES or (dtype is not None and dtype != out.dtype):
        raise ValueError(f"out must be {tuple(shape)} f32 / f16 / bf16 on {x.device}, got {tuple(out.shape)} {out.dtype} on {out.device}")
    if out.is_neg():
        raise ValueError("out must hold its values as they are, not negated (torch.Tensor.is_neg)")
    if _wants_gradient(out):
        raise ValueError("8-bit layers have no gradient: out must not ask for one")
    if not _apart(x.shape, x.stride(), x.element_size(), out.shape, out.stride(), out.element_size(), out.data_ptr() - x.data_ptr()):
        raise ValueError("out shares memory with the rows that are read")
    return (out,) + _out_rows(x.shape, x.stride(), out.shape, out.stride())


def matmul(q, scale, layer, out=None, dtype=None):
    """8-bit rows q int8 [.., K] with scale f32 [..] (``quantize_rows``' or any other's) x layer -> [.., N] of ``dtype``
    (default bf16), or into ``out`` (a tensor or a view; rows must not overlap each other or an input: rows side by side in a wider buffer are fine)."""
    _check_layer(layer, q)
    if not q.is_cuda or q.dtype != torch.int8 or q.dim() < 1 or q.shape[-1] != layer.k:
        raise ValueError(f"q must be a CUDA int8 tensor [.., {layer.k}], got {q.dtype} {tuple(q.shape)} on {q.device}")
    if scale.shape != q.shape[:-1] or scale.dtype != torch.float32 or scale.device != q.device:
        raise ValueError(f"scale must be f32 {tuple(q.shape[:-1])} on {q.device}, got {scale.dtype} {tuple(scale.shape)} on {scale.device}")
    if _wants_gradient(scale):
        raise ValueError("8-bit layers have no gradient: call them under torch.no_grad() or detach their inputs")
    if _transforms() is not None:
        _check_memory(q, scale, out)
    if q.is_neg():
        q = q.resolve_neg()
    if scale.is_neg() or not scale.is_contiguous():
        scale = scale.resolve_neg().contiguous()
    y, rows, ostride, m = _output(q, layer.n, out, dtype, torch.bfloat16)
    if out is not None and not _clear_of(scale.numel() * 4, out.shape, out.stride(), out.element_size(), out.data_ptr() - scale.data_ptr()):
        raise ValueError("out shares memory with the scales that are read")
    if m:
        need = _workspace(_ffi.PH_W8_MATMUL if rows.by_16 and not q.data_ptr() % 16 else _ffi.PH_W8_MATMUL_ANY, m, layer.k, 0, layer.n)
        ws = torch.empty(need, dtype=torch.int8, device=q.device) if need else None
        device = q.device.index
        _ffi.check(_ffi.lib().ph_w8_matmul(device, _raw_stream(device), q.data_ptr(), rows, scale.data_ptr(), layer.desc,
                                           y.data_ptr(), _TYPES[y.dtype], ostride, ws.data_ptr() if need else None, need),
                   "ph_w8_matmul")
        if out is not None:
            _written(out)
    return y


def linear(x, layer, out=None, dtype=None):
    """Float rows x [.., K] x layer -> [.., N] of ``dtype`` (default x's), or into ``out`` (as for ``matmul``; not x
    itself): the rows are quantised on the way."""
    _check_layer(layer, x)
    _check_x(x, layer.k, "x")
    if x.is_neg():
        x = x.resolve_neg()
    if _transforms() is not None:
        _check_memory(x, out)
    y, rows, ostride, m = _output(x, layer.n, out, dtype, x.dtype)
    if m:
        need = _workspace(_ffi.PH_W8_LINEAR, m, layer.k, 0, layer.n)
        ws = torch.empty(need, dtype=torch.int8, device=x.device) if need else None
        device = x.device.index
        _ffi.check(_ffi.lib().ph_w8_linear(device, _raw_stream(device), x.data_ptr(), _TYPES[x.dtype], rows, layer.desc,
                                           y.data_ptr(), _TYPES[y.dtype], ostride, ws.data_ptr() if need else None, need),
                   "ph_w8_linear")
        if out is not None:
            _written(out)
    return y


def feed_forward(x, layer1, layer2, out=None, dtype=None):
    """Two layers: x [.., K] -> [.., N] of ``dtype`` (default x's), or into ``out``; the values between them are f32,
    quantised per row like x."""
    _check_layer(layer1, x)
    _check_layer(layer2, x)
    _check_x(x, layer1.k, "x")
    if x.is_neg():
        x = x.resolve_neg()
    if _transforms() is not None:
        _check_memory(x, out)
    if layer1.n != layer2.k:
        raise ValueError(f"the first layer has {layer1.n} outputs, the second {layer2.k} inputs")
    y, rows, ostride, m = _output(x, layer2.n, out, dtype, x.dtype)
    if m:
        need = _workspace(_ffi.PH_W8_FEED_FORWARD, m, layer1.k, layer1.n, layer2.n)
        ws = torch.empty(need, dtype=torch.int8, device=x.device) if need else None
        device = x.device.index
        _ffi.check(_ffi.lib().ph_w8_feed_forward(device, _raw_stream(device), x.data_ptr(), _TYPES[x.dtype], rows,
                                                 layer1.desc, layer2.desc, y.data_ptr(), _TYPES[y.dtype], ostride,
                                                 ws.data_ptr() if need else None, need), "ph_w8_feed_forward")
        if out is not None:
            _written(out)
    return y
