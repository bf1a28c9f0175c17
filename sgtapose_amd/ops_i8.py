"""Token products in 8-bit integers, beside ``ops.linear``: a scale for each token (row of x), one for each output channel (row of w).

    xq, xs = quantize_rows(x)                       # activations, each call
    wq, ws = quantize_rows(w)                       # weights [N, K], once
    out = linear_i8(xq, xs, wq, ws, bias, relu=..., dtype=torch.bfloat16)

x, bias and out are float32, float16 or bfloat16; scales are float32; the sums are exact whole numbers.  Outputs share no memory with what a call reads.  Everything is enqueued on
the current stream of the tensors' device.
"""
import functools

import torch

from . import _lib
from .ops_attn import DTYPES, _fail, raw_stream

MAX_COUNT = (1 << 31) - 1
MAX_K = 131071                 # 127 * 128 * K stays below 2^31


def _rows(name, shape, stride, dtype, dtypes, want=None):
    """2-D rows of consecutive elements: checks, and the rows' stride."""
    if len(shape) != 2 or dtype not in dtypes or (want is not None and tuple(shape) != tuple(want)):
        _fail("%s: %s %s where %s of %s is expected", name, dtype, tuple(shape), "a matrix" if want is None else list(want),
              " / ".join(str(d).replace("torch.", "") for d in dtypes))
    M, K = shape
    if M < 1 or K < 1:
        _fail("%s is empty: %s", name, tuple(shape))
    if max(M, K) > MAX_COUNT:
        _fail("%s: %s, at most %d rows and columns (the kernels count in 32 bits)", name, tuple(shape), MAX_COUNT)
    if (K > 1 and stride[1] != 1) or (M > 1 and stride[0] < K):
        _fail("%s: rows of consecutive elements that do not overlap expected, strides %s", name, tuple(stride))
    return stride[0] if M > 1 else max(K, stride[0])


def _vector(name, t, n, dtype):
    if t.shape != (n,) or t.dtype != dtype or not t.is_contiguous():
        _fail("%s: %s %s where %s [%d] is expected", name, t.dtype, tuple(t.shape), dtype, n)


def _together(first, *others):
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            _fail("tensors on %s and %s", dev, t.device)
    if not first.is_cuda:
        _fail("expected tensors on the GPU, got %s (there is no CPU fallback)", dev)
    return dev


def _enqueue(device, name, *args, meta=None):
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _enqueue(device, name, *args, meta=meta)
    _lib.call(name, *args, raw_stream(device.index), meta=meta)


@functools.lru_cache(maxsize=1024)
def _quant_plan(shape, stride, dtype):
    """What follows from x alone: (rows, columns, row stride, type, row stride of an xq allocated here)."""
    ld = _rows("x", shape, stride, dtype, DTYPES)
    return (*shape, ld, DTYPES[dtype], (shape[1] + 15) // 16 * 16)


def quantize_rows(x, xq=None, xs=None):
    """x [M, K] -> (xq int8 [M, K], xs float32 [M]): xs = max|row| / 127, xq = x / xs to the nearest, ties to even (a row of zeros:
    zeros).  An ``xq`` allocated here has rows of whole 16 bytes."""
    M, K, ldx, ty, ldq = _quant_plan(x.shape, x.stride(), x.dtype)
    if xq is not None:
        ldq = _rows("xq", xq.shape, xq.stride(), xq.dtype, (torch.int8,), x.shape)
    if xs is not None:
        _vector("xs", xs, M, torch.float32)
    dev = _together(x, xq, xs)
    if xq is None:
        xq = torch.empty((M, ldq), dtype=torch.int8, device=dev)
        if ldq != K:
            xq = xq[:, :K]
    if xs is None:
        xs = torch.empty(M, dtype=torch.float32, device=dev)
    meta = None
    if _lib.PROFILE is not None:
        meta = {"kernel": "quant_rows_kernel", "flops": 2.0 * M * K, "exec_flops": 2.0 * M * K, "bytes": M * K * (x.element_size() + 1.0)}
    _enqueue(dev, "sgta_quant_rows_i8", x.data_ptr(), ldx, ty, xq.data_ptr(), ldq, xs.data_ptr(), M, K, meta=meta)
    return xq, xs


@functools.lru_cache(maxsize=1024)
def _linear_plan(xshape, xstride, xtype, wshape, wstride, wtype):
    """What follows from the operands alone: (M, N, K, row strides)."""
    ldx, ldw = _rows("xq", xshape, xstride, xtype, (torch.int8,)), _rows("wq", wshape, wstride, wtype, (torch.int8,))
    (M, K), N = xshape, wshape[0]
    if wshape[1] != K:
        _fail("xq %s and wq %s differ in their last dimension", tuple(xshape), tuple(wshape))
    if K > MAX_K or max(ldx, ldw) > 1 << 22:
        _fail("linear_i8: K = %d (at most %d: sums in 32 bits are exact), rows of %d and %d bytes (at most 2^22)", K, MAX_K, ldx, ldw)
    return M, N, K, ldx, ldw


def linear_i8(xq, xs, wq, ws, bias=None, out=None, relu=False, dtype=None):
    """out[m, n] = relu?( (xq[m] . wq[n]) xs[m] ws[n] + bias[n] ) in ``out``'s type (``dtype`` where it is allocated here; else
    the bias's; else float32)."""
    M, N, K, ldx, ldw = _linear_plan(xq.shape, xq.stride(), xq.dtype, wq.shape, wq.stride(), wq.dtype)
    _vector("xs", xs, M, torch.float32)
    _vector("ws", ws, N, torch.float32)
    if dtype is None:
        dtype = out.dtype if out is not None else bias.dtype if bias is not None else torch.float32
    ty = DTYPES.get(dtype)
    if ty is None:
        _fail("linear_i8 writes float32, float16 or bfloat16, not %s", dtype)
    pb = None
    if bias is not None:
        _vector("bias", bias, N, dtype)
        pb = bias.data_ptr()
    ldo = N if out is None else _rows("out", out.shape, out.stride(), out.dtype, (dtype,), (M, N))
    dev = _together(xq, xs, wq, ws, bias, out)
    if out is None:
        out = torch.empty((M, N), dtype=dtype, device=dev)
    meta = None
    if _lib.PROFILE is not None:
        meta = {"kernel": "linear_i8_kernel", "flops": 2.0 * M * N * K, "exec_flops": 2.0 * M * N * K,
                "bytes": 1.0 * M * K + N * K + out.element_size() * M * N}
    _enqueue(dev, "sgta_linear_i8", xq.data_ptr(), ldx, xs.data_ptr(), wq.data_ptr(), ldw, ws.data_ptr(), pb, out.data_ptr(), ldo, M, N, K,
             int(relu), ty, meta=meta)
    return out
