"""Token products in 8-bit integers, beside ``ops.linear``: a scale for each token (row of x), one for each output channel (row of w).

    xq, xs = quantize_rows(x)                       # activations, each call
    wq, ws = quantize_rows(w)                       # weights [N, K], once
    out = linear_i8(xq, xs, wq, ws, bias, relu=..., dtype=torch.bfloat16)

x, bias and out are float32, float16 or bfloat16; scales are float32; the sums are exact whole numbers.  Everything is enqueued on
the current stream of the tensors' device.
"""
import torch

from . import _lib
from .ops_attn import DTYPES, _fail

MAX_K = 131071                 # 127 * 128 * K stays below 2^31


def _rows(name, t, dtypes, shape=None):
    """2-D rows of consecutive elements on the GPU; returns their stride."""
    if t.dim() != 2 or t.dtype not in dtypes or (shape is not None and t.shape != shape):
        _fail("%s: %s %s where %s of %s is expected", name, t.dtype, tuple(t.shape), "a matrix" if shape is None else list(shape),
              " / ".join(str(d).replace("torch.", "") for d in dtypes))
    M, K = t.shape
    if M < 1 or K < 1:
        _fail("%s is empty: %s", name, tuple(t.shape))
    ld, one = t.stride()
    if (K > 1 and one != 1) or (M > 1 and ld < K):
        _fail("%s: rows of consecutive elements that do not overlap expected, strides %s", name, tuple(t.stride()))
    return ld if M > 1 else max(K, ld)


def _vector(name, t, n, dtype):
    if t.shape != (n,) or t.dtype != dtype or (n > 1 and t.stride(0) != 1):
        _fail("%s: %s %s where %s [%d] is expected", name, t.dtype, tuple(t.shape), dtype, n)


def _together(first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            _fail("tensors on %s and %s", first.device, t.device)
    if not first.is_cuda:
        _fail("expected tensors on the GPU, got %s (there is no CPU fallback)", first.device)


def _enqueue(device, name, *args, meta=None):
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _enqueue(device, name, *args, meta=meta)
    _lib.call(name, *args, torch.cuda.current_stream(device).cuda_stream, meta=meta)


def quantize_rows(x, xq=None, xs=None):
    """x [M, K] -> (xq int8 [M, K], xs float32 [M]): xs = max|row| / 127, xq = x / xs to the nearest, ties to even (a row of zeros:
    zeros).  An ``xq`` allocated here has rows of whole 16 bytes."""
    ldx = _rows("x", x, DTYPES)
    M, K = x.shape
    if xq is not None:
        _rows("xq", xq, (torch.int8,), x.shape)
    if xs is not None:
        _vector("xs", xs, M, torch.float32)
    _together(x, xq, xs)
    if xq is None:
        xq = torch.empty(M, (K + 15) // 16 * 16, dtype=torch.int8, device=x.device)[:, :K]
    if xs is None:
        xs = torch.empty(M, dtype=torch.float32, device=x.device)
    meta = None
    if _lib.PROFILE is not None:
        meta = {"kernel": "quant_rows_kernel", "flops": 2.0 * M * K, "exec_flops": 2.0 * M * K, "bytes": M * K * (x.element_size() + 1.0)}
    _enqueue(x.device, "sgta_quant_rows_i8", x.data_ptr(), ldx, DTYPES[x.dtype], xq.data_ptr(),
             xq.stride(0) if M > 1 else max(K, xq.stride(0)), xs.data_ptr(), M, K, meta=meta)
    return xq, xs


def linear_i8(xq, xs, wq, ws, bias=None, out=None, relu=False, dtype=None):
    """out[m, n] = relu?( (xq[m] . wq[n]) xs[m] ws[n] + bias[n] ) in ``out``'s type (``dtype`` where it is allocated here; else
    the bias's; else float32)."""
    ldx, ldw = _rows("xq", xq, (torch.int8,)), _rows("wq", wq, (torch.int8,))
    (M, K), N = xq.shape, wq.shape[0]
    if wq.shape[1] != K:
        _fail("xq %s and wq %s differ in their last dimension", tuple(xq.shape), tuple(wq.shape))
    if K > MAX_K or max(ldx, ldw) > 1 << 22:
        _fail("linear_i8: K = %d (at most %d: sums in 32 bits are exact), rows of %d and %d bytes (at most 2^22)", K, MAX_K, ldx, ldw)
    _vector("xs", xs, M, torch.float32)
    _vector("ws", ws, N, torch.float32)
    if dtype is None:
        dtype = out.dtype if out is not None else bias.dtype if bias is not None else torch.float32
    if dtype not in DTYPES:
        _fail("linear_i8 writes float32, float16 or bfloat16, not %s", dtype)
    if bias is not None:
        _vector("bias", bias, N, dtype)
    if out is not None:
        _rows("out", out, (dtype,), (M, N))
    _together(xq, xs, wq, ws, bias, out)
    if out is None:
        out = torch.empty(M, N, dtype=dtype, device=xq.device)
    meta = None
    if _lib.PROFILE is not None:
        meta = {"kernel": "linear_i8_kernel", "flops": 2.0 * M * N * K, "exec_flops": 2.0 * M * N * K,
                "bytes": 1.0 * M * K + N * K + out.element_size() * M * N}
    _enqueue(xq.device, "sgta_linear_i8", xq.data_ptr(), ldx, xs.data_ptr(), wq.data_ptr(), ldw, ws.data_ptr(),
             None if bias is None else bias.data_ptr(), out.data_ptr(), out.stride(0) if M > 1 else max(N, out.stride(0)), M, N, K,
             int(relu), DTYPES[dtype], meta=meta)
    return out
