"""Attention over sequences of any length, beside the fixed-window ``ops.mhca``: a learned relative position bias by buckets
(``rel_attention``), and the difference of two softmax maps with a learned weight (``diff_attention``), each with its gradients.

    q [B, Lq, H, D], k [B, Lk, Hkv, D], v [B, Lk, Hkv, Dv] -> out [B, Lq, H, Dv];  differential: q [B, Lq, H, 2, D], k [B, Lk, Hkv, 2, D]

Element types float32, float16, bfloat16 (one for all tensors of a call); sums, softmax statistics and the bias are held in
float32.  Query head h reads key / value head h // (H // Hkv).  The last dimension is contiguous; the others may have any
non-negative stride of whole 16 bytes (slices of a fused projection, caches).  D and Dv are multiples of 8: up to 128 for
``rel_attention`` (Dv = D), up to 64 and 128 for ``diff_attention``.

Lengths: ``kv_len`` / ``q_len`` int32 [B] on the GPU (None: all).  What lies behind them is never read, output rows behind
``q_len`` are left as they are (an output that a call allocates itself holds zeros there).  ``q_start`` int32 [B] is the position of
the first query among the keys (None: 0); a new token against a cache that already holds it has q_start = kv_len - 1.
``causal``: a query at position p sees keys j <= p.  A query that sees no key has an output and gradients of zero.

Everything is enqueued on the current stream of the tensors' device; workspaces come from torch's allocator anew in each call, so
calls on several streams and calls captured into several graphs do not share any.
"""
import ctypes
import functools
import math

import torch

from . import _lib

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_REACH = 1024               # distances that may have buckets of their own (the kernels keep them in LDS)


def _fail(msg, *args):
    raise _lib.SgtaHipError(msg % args)


def _first_distances(n, far):
    """First distance of each of the logarithmic buckets n/2 + 1 ... n - 1 of one side: the least r with
    n/2 + log(r / (n/2)) / log(far / (n/2)) (n - n/2) >= bucket, by integer powers (no rounding at a border)."""
    e = n // 2
    m = n - e
    out, r = [], e
    for k in range(1, m):
        while r ** m < e ** (m - k) * far ** k:
            r += 1
        out.append(r)
    return out


def bucket_reach(num_buckets, max_distance, bidirectional):
    """The distance from which on the bucket stays the same (checks the arguments)."""
    n = num_buckets // 2 if bidirectional else num_buckets
    if num_buckets < 2 or (bidirectional and num_buckets % 2) or n < 2:
        _fail("rel_attention: %d buckets (at least 2 a direction, an even number for two directions)", num_buckets)
    if not n // 2 < max_distance <= MAX_REACH:
        _fail("rel_attention: max_distance %d is not in %d ... %d", max_distance, n // 2 + 1, MAX_REACH)
    first = _first_distances(n, max_distance)
    return max(first[-1] if first else 1, n // 2, 1)


def relative_buckets(num_buckets, max_distance, bidirectional):
    """Bucket of each distance key - query in -reach ... reach, as a list.  Half the buckets (all of them when not
    ``bidirectional``, where keys behind the query count as distance 0) hold: distances below half of them one each, larger
    ones up to ``max_distance`` logarithmically, the last one everything beyond."""
    reach = bucket_reach(num_buckets, max_distance, bidirectional)
    n = num_buckets // 2 if bidirectional else num_buckets
    first = _first_distances(n, max_distance)

    def one_side(r):
        return r if r < n // 2 else n // 2 + sum(r >= f for f in first)
    return [(n if bidirectional and d > 0 else 0) + one_side(abs(d) if bidirectional else max(-d, 0)) for d in range(-reach, reach + 1)]


@functools.lru_cache(maxsize=None)
def _lut(num_buckets, max_distance, bidirectional, device):
    """``relative_buckets`` on the device: depends on nothing but the arguments, as ops.gauss_taps."""
    return torch.tensor(relative_buckets(num_buckets, max_distance, bidirectional), dtype=torch.int32).to(device)


def _strides(t, maps):
    """Element strides {batch, position, head, map} of [B, L, heads(, 2), D]."""
    s = t.stride()
    return (ctypes.c_long * 4)(s[0], s[1], s[2], s[3] if maps == 2 else 0)


def _layout(name, t, shape, like):
    """Shape, type, device and 16-byte layout of one strided operand."""
    if tuple(t.shape) != tuple(shape):
        _fail("%s is %s, expected %s", name, tuple(t.shape), tuple(shape))
    if t.dtype != like.dtype or t.device != like.device:
        _fail("%s is %s on %s, q is %s on %s", name, t.dtype, t.device, like.dtype, like.device)
    whole = 16 // t.element_size()
    if t.stride(-1) != 1 or any(s % whole or s < 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1) or t.data_ptr() % 16:
        _fail("%s: the last dimension must be contiguous, the others' strides and the pointer whole 16 bytes (strides %s)",
              name, tuple(t.stride()))


def _dense(t):
    """``t`` with the strides of dimensions of one element set to what a kernel may multiply (torch leaves them arbitrary)."""
    if any(n == 1 for n in t.shape[:-1]):
        whole = 16 // t.element_size()
        t = t.as_strided(t.shape, [s if n > 1 or i == t.dim() - 1 else whole for i, (s, n) in enumerate(zip(t.stride(), t.shape))])
    return t


def _operands(maps, q, k, v, w, causal, scale, q_len, kv_len, q_start):
    """Checks what every call has in common -> AttnArgs (w and outputs still to be set)."""
    mp = (2,) if maps == 2 else ()
    nd = 4 + len(mp)
    if q.dim() != nd or k.dim() != nd or v.dim() != 4:
        _fail("q %s, k %s, v %s: expected [B, L, heads%s, D] and [B, L, heads, Dv]", tuple(q.shape), tuple(k.shape), tuple(v.shape),
              ", 2" if mp else "")
    if q.dtype not in DTYPES:
        _fail("attention takes float32, float16 or bfloat16, got %s", q.dtype)
    B, Lq, H, D = q.shape[0], q.shape[1], q.shape[2], q.shape[-1]
    Lk, Hkv, Dv = v.shape[1], v.shape[2], v.shape[3]
    if min(B, Lq, Lk, H, Hkv) < 1 or H % Hkv:
        _fail("B %d, Lq %d, Lk %d, %d heads on %d key / value heads: none may be zero, the heads shared evenly", B, Lq, Lk, H, Hkv)
    most = (128, 128) if maps == 1 else (64, 128)
    if D % 8 or Dv % 8 or not 8 <= D <= most[0] or not 8 <= Dv <= most[1] or (maps == 1 and D != Dv):
        _fail("head sizes %d, %d: multiples of 8 up to %d, %d%s", D, Dv, *most, ", equal" if maps == 1 else "")
    if max(Lq, Lk) >= 1 << 29:
        _fail("sequences of %d, %d: below 2^29", Lq, Lk)
    if scale is None:
        scale = D ** -0.5
    if not (scale > 0 and math.isfinite(scale)):
        _fail("scale %r: a positive number", scale)
    _layout("q", q, (B, Lq, H, *mp, D), q)
    _layout("k", k, (B, Lk, Hkv, *mp, D), q)
    _layout("v", v, (B, Lk, Hkv, Dv), q)
    for name, t in (("q_len", q_len), ("kv_len", kv_len), ("q_start", q_start)):
        if t is not None and (tuple(t.shape) != (B,) or t.dtype != torch.int32 or t.device != q.device or not t.is_contiguous()):
            _fail("%s: int32 [%d] on %s expected, got %s %s on %s", name, B, q.device, t.dtype, tuple(t.shape), t.device)
    if w.dtype != q.dtype or w.device != q.device or not w.is_contiguous():
        _fail("the learned weights are %s on %s: %s, contiguous, on %s expected", w.dtype, w.device, q.dtype, q.device)
    if not q.is_cuda:
        _fail("expected tensors on the GPU, got %s (there is no CPU fallback)", q.device)
    q, k, v = _dense(q), _dense(k), _dense(v)
    a = _lib.AttnArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), w=w.data_ptr(), sq=_strides(q, maps), sk=_strides(k, maps),
                      sv=_strides(v, 1), B=B, Lq=Lq, Lk=Lk, H=H, Hkv=Hkv, D=D, Dv=Dv, causal=int(causal), dtype=DTYPES[q.dtype],
                      scale=scale, q_len=_ptr(q_len), kv_len=_ptr(kv_len), q_start=_ptr(q_start))
    return a


def _ptr(t):
    return None if t is None else t.data_ptr()


def _overlaps(t):
    """Whether two elements of ``t`` may share memory (an expanded or overlapping view)."""
    need = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s < need:
            return True
        need = s * (n - 1) + need
    return False


def _output(name, t, shape, like, partial=False):
    """The caller's tensor, checked, or a new one (zeros where a call may leave rows as they are)."""
    if t is None:
        return torch.zeros(shape, dtype=like.dtype, device=like.device) if partial else torch.empty(shape, dtype=like.dtype, device=like.device)
    _layout(name, t, shape, like)
    if _overlaps(t):
        _fail("%s: elements that share memory (strides %s) cannot be written", name, tuple(t.stride()))
    return t


def _work(floats, device):
    return torch.empty(floats, dtype=torch.float32, device=device) if floats else None


def _enqueue(name, a, device, meta):
    _lib.call(name, ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream), meta=meta)


def _meta(kernel, a, maps, products):
    """Algorithmic work for the live profile: ``products`` of D and of Dv per pair of positions (full, unmasked lengths)."""
    if _lib.PROFILE is None:
        return None
    pairs = 2.0 * a.B * a.H * a.Lq * a.Lk * (0.5 if a.causal and a.Lq == a.Lk else 1.0)
    flops = pairs * (products[0] * a.D + products[1] * a.Dv)
    size = 4 if a.dtype == 0 else 2
    return {"kernel": kernel, "flops": flops, "exec_flops": flops,
            "bytes": size * (a.B * a.Lq * a.H * (maps * a.D + a.Dv) + a.B * a.Lk * a.Hkv * (maps * a.D + a.Dv))}


def _check_table(table, H, max_distance, bidirectional):
    if table.dim() != 2 or table.shape[1] != H:
        _fail("table is %s, expected [num_buckets, %d]", tuple(table.shape), H)
    return bucket_reach(table.shape[0], int(max_distance), bool(bidirectional))


def _check_lam(lam, D):
    if tuple(lam.shape) != (4, D):
        _fail("lam is %s, expected [4, %d]", tuple(lam.shape), D)


def _forward(name, maps, a, like, out, q_len, save):
    shape = (a.B, a.Lq, a.H, a.Dv)
    out = _output("out", out, shape, like, partial=q_len is not None)
    o = _dense(out)
    a.out, a.so = o.data_ptr(), _strides(o, 1)
    stats = out2 = None
    if save:
        stats = torch.empty(maps, a.B, a.H, a.Lq, 2, dtype=torch.float32, device=like.device)
        a.stats = stats.data_ptr()
        if maps == 2:
            out2 = torch.empty(shape, dtype=like.dtype, device=like.device)
            a.out2 = out2.data_ptr()
    ws = _work(_lib.load().sgta_attn_fwd_ws_floats(ctypes.byref(a), maps), like.device)
    if ws is not None:
        a.ws, a.ws_floats = ws.data_ptr(), ws.numel()
    _enqueue(name, a, like.device, _meta(name, a, maps, (maps, maps)))
    return (out, (stats, out2)) if save else out


def rel_attention(q, k, v, table, out=None, *, max_distance=128, bidirectional=True, causal=False, scale=None, q_len=None, kv_len=None,
                  q_start=None, save=False):
    """softmax(scale q k^T + table[bucket(key - query), head]) v, one pass, nothing of size Lq x Lk in memory.

    ``table`` [num_buckets, H] is the learned bias; buckets as ``relative_buckets(num_buckets, max_distance, bidirectional)``.
    ``scale`` None: D ** -0.5.  ``save``: returns (out, saved) for ``rel_attention_bwd``."""
    reach = _check_table(table, q.shape[2], max_distance, bidirectional)
    a = _operands(1, q, k, v, table, causal, scale, q_len, kv_len, q_start)
    with torch.cuda.device(q.device):
        lut = _lut(table.shape[0], int(max_distance), bool(bidirectional), q.device)
        a.lut, a.reach, a.num_buckets = lut.data_ptr(), reach, table.shape[0]
        return _forward("sgta_rel_attn_fwd", 1, a, q, out, q_len, save)


def diff_attention(q, k, v, lam, out=None, *, lam_init=0.8, causal=False, scale=None, q_len=None, kv_len=None, q_start=None, save=False):
    """(softmax(scale q1 k1^T) - lambda softmax(scale q2 k2^T)) v; ``lam`` [4, D] holds the learned vectors of
    lambda = exp(lam[0].lam[1]) - exp(lam[2].lam[3]) + lam_init, one for all heads.  V is read once for both maps.
    ``save``: returns (out, saved) for ``diff_attention_bwd``."""
    _check_lam(lam, q.shape[-1])
    a = _operands(2, q, k, v, lam, causal, scale, q_len, kv_len, q_start)
    a.lam_init = lam_init
    with torch.cuda.device(q.device):
        return _forward("sgta_diff_attn_fwd", 2, a, q, out, q_len, save)


def _backward(name, maps, a, like, dout, w, out, saved, grads, q_len, kv_len):
    mp = (2,) if maps == 2 else ()
    stats, out2 = saved
    shape = (a.B, a.Lq, a.H, a.Dv)
    _layout("dout", dout, shape, like)
    _layout("out", out, shape, like)
    if tuple(stats.shape) != (maps, a.B, a.H, a.Lq, 2) or stats.device != like.device or (maps == 2 and tuple(out2.shape) != shape):
        _fail("saved does not come from a forward call of this shape")
    dq, dk, dv, dw = grads
    dq = _output("dq", dq, (a.B, a.Lq, a.H, *mp, a.D), like, q_len is not None)
    dk = _output("dk", dk, (a.B, a.Lk, a.Hkv, *mp, a.D), like, kv_len is not None)
    dv = _output("dv", dv, (a.B, a.Lk, a.Hkv, a.Dv), like, kv_len is not None)
    if dw is None:
        dw = torch.empty_like(w)
    elif dw.shape != w.shape or dw.dtype != w.dtype or dw.device != w.device or not dw.is_contiguous():
        _fail("the learned weights' gradient is %s %s, expected %s %s, contiguous", dw.dtype, tuple(dw.shape), w.dtype, tuple(w.shape))
    g, o, q_, k_, v_ = (_dense(t) for t in (dout, out, dq, dk, dv))
    a.dout, a.sdo, a.out, a.so = g.data_ptr(), _strides(g, 1), o.data_ptr(), _strides(o, 1)
    a.dq, a.sdq, a.dk, a.sdk, a.dv, a.sdv = q_.data_ptr(), _strides(q_, maps), k_.data_ptr(), _strides(k_, maps), v_.data_ptr(), _strides(v_, 1)
    a.dw, a.stats, a.out2 = dw.data_ptr(), stats.data_ptr(), _ptr(out2)
    ws = _work(_lib.load().sgta_attn_bwd_ws_floats(ctypes.byref(a), maps), like.device)
    a.ws, a.ws_floats = ws.data_ptr(), ws.numel()
    _enqueue(name, a, like.device, _meta(name, a, maps, (5 * maps, 3)))
    return dq, dk, dv, dw


def rel_attention_bwd(dout, q, k, v, table, out, saved, dq=None, dk=None, dv=None, dtable=None, *, max_distance=128, bidirectional=True,
                      causal=False, scale=None, q_len=None, kv_len=None, q_start=None):
    """Gradients (dq, dk, dv, dtable) of ``rel_attention`` for the gradient ``dout`` of its ``out``; the other arguments as in the
    forward call, ``saved`` from its ``save=True``.  Shared heads' gradients are summed; rows behind q_len / kv_len are left as they
    are (zeros where allocated here).  The same inputs give the same bits."""
    reach = _check_table(table, q.shape[2], max_distance, bidirectional)
    a = _operands(1, q, k, v, table, causal, scale, q_len, kv_len, q_start)
    with torch.cuda.device(q.device):
        lut = _lut(table.shape[0], int(max_distance), bool(bidirectional), q.device)
        a.lut, a.reach, a.num_buckets = lut.data_ptr(), reach, table.shape[0]
        return _backward("sgta_rel_attn_bwd", 1, a, q, dout, table, out, saved, (dq, dk, dv, dtable), q_len, kv_len)


def diff_attention_bwd(dout, q, k, v, lam, out, saved, dq=None, dk=None, dv=None, dlam=None, *, lam_init=0.8, causal=False, scale=None,
                       q_len=None, kv_len=None, q_start=None):
    """Gradients (dq, dk, dv, dlam) of ``diff_attention``, as ``rel_attention_bwd``; dlam [4, D]."""
    _check_lam(lam, q.shape[-1])
    a = _operands(2, q, k, v, lam, causal, scale, q_len, kv_len, q_start)
    a.lam_init = lam_init
    with torch.cuda.device(q.device):
        return _backward("sgta_diff_attn_bwd", 2, a, q, dout, lam, out, saved, (dq, dk, dv, dlam), q_len, kv_len)
