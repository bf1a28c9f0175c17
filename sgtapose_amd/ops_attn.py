"""Attention over sequences of any length, beside the fixed-window ``ops.mhca``: a learned relative position bias by buckets
(``rel_attention``), and the difference of two softmax maps with a learned weight (``diff_attention``), each with its gradients.

    q [B, Lq, H, D], k [B, Lk, Hkv, D], v [B, Lk, Hkv, Dv] -> out [B, Lq, H, Dv];  differential: q [B, Lq, H, 2, D], k [B, Lk, Hkv, 2, D]

Element types float32, float16, bfloat16 (one for all tensors of a call); sums, softmax statistics and the bias are held in
float32.  Query head h reads key / value head h // (H // Hkv).  The last dimension is contiguous; the others may have any
non-negative stride of whole 16 bytes (slices of a fused projection, caches).  D and Dv are multiples of 8: up to 128 for
``rel_attention`` (Dv = D), up to 64 and 128 for ``diff_attention``.  Positions lie at most 16 MB apart.

Lengths: ``kv_len`` / ``q_len`` int32 [B] on the GPU (None: all).  What lies behind them is never read, output rows behind
``q_len`` are left as they are (an output that a call allocates itself holds zeros there).  ``q_start`` int32 [B] is the position of
the first query among the keys (None: 0); a new token against a cache that already holds it has q_start = kv_len - 1.
``causal``: a query at position p sees keys j <= p.  A query that sees no key has an output and gradients of zero.

Table values of any size: -inf hides a bucket's keys; finite ones keep the scores' accuracy up to 7e8 in magnitude (2^30 in units of log2)
and, up to twice that, the accuracy of scores below 40 (a mask of -1e9).  Beyond, down to a type's lowest value, they absorb the scores,
so that a query that only such keys are left for weighs them evenly.

Within the lengths a value that is not finite may also reach positions from which the mask hides it (0 times infinity), as in the
plain products.  float32 operands are split into three bfloat16 numbers, so that an infinity among them gives not-a-numbers.

Nothing is recorded for autograd: outside ``torch.no_grad()`` operands that require a gradient are refused unless ``save=True`` says that
the caller takes the backward operator.  Its ``dout`` is laid out as the other operands are (an expanded one: ``.contiguous()`` first).

Everything is enqueued on the current stream of the tensors' device; workspaces come from torch's allocator anew in each call, so
calls on several streams and calls captured into several graphs do not share any.  Outputs share no memory with each other or with
what a call reads.  ``rel_attention`` puts the table of buckets on the device at its first call with given settings, which cannot be
captured: run it once before a graph is.
"""
import ctypes
import functools
import math

import torch

from . import _lib

raw_stream = torch._C._cuda_getCurrentRawStream      # (device index) -> the current stream's handle; 2 us less a call than the Stream object
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_PITCH = 1 << 24            # bytes from one position to the next
MAX_GROUPS = 1 << 24           # blocks of 128 positions of all sequences and heads
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


@functools.lru_cache(maxsize=None)
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
    """``relative_buckets`` on the device, and each bucket's first entry and number of entries: depends on nothing but the arguments,
    as ops.gauss_taps."""
    if torch.cuda.is_current_stream_capturing():
        _fail("the table of %d buckets to distance %d is not on the device yet and cannot be copied there in a captured graph: call the operator "
              "once before", num_buckets, max_distance)
    of = relative_buckets(num_buckets, max_distance, bidirectional)
    count = [of.count(b) for b in range(num_buckets)]
    first = [of.index(b) if n else 0 for b, n in enumerate(count)]
    return torch.tensor(of + first + count, dtype=torch.int32).to(device)


def _whole(name, shape, stride, size):
    """Checks a strided operand's layout -> its strides, those of dimensions of one element (which torch leaves arbitrary) set to
    what a kernel may multiply."""
    whole = 16 // size
    st = [s if n > 1 else whole for s, n in zip(stride[:-1], shape[:-1])]
    if (stride[-1] != 1 and shape[-1] != 1) or any(s % whole or s < 0 for s in st):
        _fail("%s: the last dimension must be contiguous, the other strides whole 16 bytes (strides %s)", name, tuple(stride))
    if st[1] * size > MAX_PITCH:
        _fail("%s: positions lie at most %d bytes apart (strides %s)", name, MAX_PITCH, tuple(stride))
    return st


def _set_strides(a, field, st, map_dim):
    """Element strides {batch, position, head, map} of [B, L, heads(, 2), D]."""
    f = getattr(a, field)
    f[0], f[1], f[2], f[3] = st[0], st[1], st[2], st[3] if map_dim else 0


@functools.lru_cache(maxsize=1024)
def _plan(maps, qs, qst, ks, kst, vs, vst, dtype, causal, scale, w_shape, max_distance, bidirectional, lam_init):
    """Everything that follows from shapes, strides and settings: the checks, and AttnArgs with all but pointers."""
    nd = 5 if maps == 2 else 4
    if len(qs) != nd or len(ks) != nd or len(vs) != 4:
        _fail("q %s, k %s, v %s: expected [B, L, heads%s, D] and [B, L, heads, Dv]", tuple(qs), tuple(ks), tuple(vs), ", 2" if maps == 2 else "")
    if dtype not in DTYPES:
        _fail("attention takes float32, float16 or bfloat16, got %s", dtype)
    B, Lq, H, D = qs[0], qs[1], qs[2], qs[-1]
    Lk, Hkv, Dv = vs[1], vs[2], vs[3]
    if min(B, Lq, Lk, H, Hkv) < 1 or H % Hkv:
        _fail("B %d, Lq %d, Lk %d, %d heads on %d key / value heads: none may be zero, the heads shared evenly", B, Lq, Lk, H, Hkv)
    mp = (2,) if maps == 2 else ()
    if tuple(qs) != (B, Lq, H, *mp, D) or tuple(ks) != (B, Lk, Hkv, *mp, D) or vs[0] != B:
        _fail("q %s, k %s, v %s do not fit together", tuple(qs), tuple(ks), tuple(vs))
    most = (128, 128) if maps == 1 else (64, 128)
    if D % 8 or Dv % 8 or not 8 <= D <= most[0] or not 8 <= Dv <= most[1] or (maps == 1 and D != Dv):
        _fail("head sizes %d, %d: multiples of 8 up to %d, %d%s", D, Dv, *most, ", equal" if maps == 1 else "")
    if max(Lq, Lk) >= 1 << 29:
        _fail("sequences of %d, %d: below 2^29", Lq, Lk)
    if B * H * ((max(Lq, Lk) + 127) // 128) >= MAX_GROUPS:
        _fail("%d sequences of %d, %d with %d heads: B * H * ceil(longest / 128) stays below 2^24", B, Lq, Lk, H)
    if scale is None:
        scale = D ** -0.5
    if not 1e-36 <= scale <= 1e36:
        _fail("scale %r: a positive number, from 1e-36 to 1e36 (it and its inverse are formed in units of log2)", scale)
    a = _lib.AttnArgs(B=B, Lq=Lq, Lk=Lk, H=H, Hkv=Hkv, D=D, Dv=Dv, causal=int(causal), dtype=DTYPES[dtype], scale=scale)
    size = 4 if dtype == torch.float32 else 2
    _set_strides(a, "sq", _whole("q", qs, qst, size), maps == 2)
    _set_strides(a, "sk", _whole("k", ks, kst, size), maps == 2)
    _set_strides(a, "sv", _whole("v", vs, vst, size), False)
    if maps == 1:
        if len(w_shape) != 2 or w_shape[1] != H:
            _fail("table is %s, expected [num_buckets, %d]", tuple(w_shape), H)
        a.num_buckets, a.reach = w_shape[0], bucket_reach(w_shape[0], max_distance, bidirectional)
    else:
        if tuple(w_shape) != (4, D):
            _fail("lam is %s, expected [4, %d]", tuple(w_shape), D)
        a.lam_init = lam_init
    a.so[0], a.so[1], a.so[2] = Lq * H * Dv, H * Dv, Dv
    return a


def _operands(maps, q, k, v, w, causal, scale, q_len, kv_len, q_start, max_distance=0, bidirectional=False, lam_init=0.0):
    """Checks what every call has in common -> AttnArgs (outputs still to be set)."""
    dev, dtype = q.device, q.dtype
    scale = None if scale is None else float(scale)
    a = _lib.AttnArgs.from_buffer_copy(_plan(maps, q.shape, q.stride(), k.shape, k.stride(), v.shape, v.stride(), dtype, bool(causal), scale,
                                             w.shape, max_distance, bidirectional, lam_init))
    for name, t in (("k", k), ("v", v), ("the learned weights", w)):
        if t.dtype != dtype or t.device != dev:
            _fail("%s: %s on %s, q is %s on %s", name, t.dtype, t.device, dtype, dev)
    if not w.is_contiguous():
        _fail("the learned weights must be contiguous")
    a.q, a.k, a.v, a.w = pq, pk, pv, _ = q.data_ptr(), k.data_ptr(), v.data_ptr(), w.data_ptr()
    if (pq | pk | pv) & 15:
        _fail("q, k and v must start at whole 16 bytes")
    if q_len is not None:
        a.q_len = _lengths("q_len", q_len, a.B, dev)
    if kv_len is not None:
        a.kv_len = _lengths("kv_len", kv_len, a.B, dev)
    if q_start is not None:
        a.q_start = _lengths("q_start", q_start, a.B, dev)
    if not q.is_cuda:
        _fail("expected tensors on the GPU, got %s (there is no CPU fallback)", dev)
    if maps == 1:
        a.lut = _lut(a.num_buckets, max_distance, bidirectional, dev).data_ptr()
    return a


def _lengths(name, t, B, dev):
    if t.shape != (B,) or t.dtype != torch.int32 or t.device != dev or (B > 1 and t.stride(0) != 1):
        _fail("%s: int32 [%d] on %s expected, got %s %s on %s", name, B, dev, t.dtype, tuple(t.shape), t.device)
    return t.data_ptr()


def _like(name, t, shape, like):
    """A further operand: shape, type, device, layout -> its strides."""
    if tuple(t.shape) != tuple(shape):
        _fail("%s is %s, expected %s", name, tuple(t.shape), tuple(shape))
    if t.dtype != like.dtype or t.device != like.device:
        _fail("%s is %s on %s, q is %s on %s", name, t.dtype, t.device, like.dtype, like.device)
    if t.data_ptr() & 15:
        _fail("%s must start at whole 16 bytes", name)
    return _whole(name, t.shape, t.stride(), t.element_size())


def _overlaps(t):
    """Whether two elements of ``t`` may share memory (an expanded or overlapping view)."""
    need = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s < need:
            return True
        need = s * (n - 1) + need
    return False


def _output(a, field, strides, t, shape, like, partial):
    """The caller's tensor, checked, or a new one (zeros where a call may leave rows as they are), set in ``a``."""
    if t is None:
        t = (torch.zeros if partial else torch.empty)(shape, dtype=like.dtype, device=like.device)
        st = t.stride()
    else:
        st = _like(field, t, shape, like)
        if _overlaps(t):
            _fail("%s: elements that share memory (strides %s) cannot be written", field, tuple(t.stride()))
    setattr(a, field, t.data_ptr())
    _set_strides(a, strides, st, len(shape) == 5)
    return t


def _enqueue(name, a, device, ws_name, maps, meta):
    """Launches on the device's current stream, with the workspace the call needs."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _enqueue(name, a, device, ws_name, maps, meta)
    n = getattr(_lib.load(), ws_name)(ctypes.byref(a), maps)
    if n:
        ws = torch.empty(n, dtype=torch.float32, device=device)
        a.ws, a.ws_floats = ws.data_ptr(), n
    _lib.call(name, ctypes.byref(a), raw_stream(device.index), meta=meta)


def _meta(kernel, a, maps, backward=False):
    """Work for the live profile (full, unmasked lengths): ``flops`` of the formulas' products of D and of Dv per pair of positions,
    ``exec_flops`` with the scores and dO V^T that the backward kernels compute twice, ``bytes`` with each tensor once."""
    if _lib.PROFILE is None:
        return None
    pairs = 2.0 * a.B * a.H * a.Lq * a.Lk * (0.5 if a.causal and a.Lq == a.Lk else 1.0)
    need, does = ((3 * maps, 2), (4 * maps, 3)) if backward else ((maps, maps),) * 2
    flops, execs = (pairs * (d * a.D + dv * a.Dv) for d, dv in (need, does))
    size = 4 if a.dtype == 0 else 2
    q, kv, o = a.B * a.Lq * a.H * maps * a.D, a.B * a.Lk * a.Hkv * (maps * a.D + a.Dv), a.B * a.Lq * a.H * a.Dv
    count = 2 * q + 2 * kv + (maps + 1) * o if backward else q + kv + o          # and each gradient; out, the second map's, dout
    return {"kernel": kernel, "flops": flops, "exec_flops": execs, "bytes": size * count}


def _no_graph(save, *tensors):
    """These operators record nothing for autograd: a result that looks as if it did would train without its share of the gradient."""
    if not save and torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        _fail("an operand requires a gradient, which this call does not record: call it under torch.no_grad(), or with save=True and the "
              "backward operator (inside an autograd.Function, say)")


def _forward(name, maps, a, like, out, q_len, save):
    shape = (a.B, a.Lq, a.H, a.Dv)
    out = _output(a, "out", "so", out, shape, like, q_len is not None)
    stats = out2 = None
    if save:
        stats = torch.empty(maps, a.B, a.H, a.Lq, 2, dtype=torch.float32, device=like.device)
        a.stats = stats.data_ptr()
        if maps == 2:
            out2 = torch.empty(shape, dtype=like.dtype, device=like.device)
            a.out2 = out2.data_ptr()
    _enqueue(name, a, like.device, "sgta_attn_fwd_ws_floats", maps, _meta(name, a, maps))
    return (out, (stats, out2)) if save else out


def rel_attention(q, k, v, table, out=None, *, max_distance=128, bidirectional=True, causal=False, scale=None, q_len=None, kv_len=None,
                  q_start=None, save=False):
    """softmax(scale q k^T + table[bucket(key - query), head]) v, one pass, nothing of size Lq x Lk in memory.

    ``table`` [num_buckets, H] is the learned bias; buckets as ``relative_buckets(num_buckets, max_distance, bidirectional)``.
    ``scale`` None: D ** -0.5; 1e-36 to 1e36.  ``save``: returns (out, saved) for ``rel_attention_bwd``."""
    _no_graph(save, q, k, v, table)
    a = _operands(1, q, k, v, table, causal, scale, q_len, kv_len, q_start, int(max_distance), bool(bidirectional))
    return _forward("sgta_rel_attn_fwd", 1, a, q, out, q_len, save)


def diff_attention(q, k, v, lam, out=None, *, lam_init=0.8, causal=False, scale=None, q_len=None, kv_len=None, q_start=None, save=False):
    """(softmax(scale q1 k1^T) - lambda softmax(scale q2 k2^T)) v; ``lam`` [4, D] holds the learned vectors of
    lambda = exp(lam[0].lam[1]) - exp(lam[2].lam[3]) + lam_init, one for all heads.  V is read once for both maps.
    ``save``: returns (out, saved) for ``diff_attention_bwd``."""
    _no_graph(save, q, k, v, lam)
    a = _operands(2, q, k, v, lam, causal, scale, q_len, kv_len, q_start, lam_init=float(lam_init))
    return _forward("sgta_diff_attn_fwd", 2, a, q, out, q_len, save)


def _saved(stats, out2, maps, shape, like):
    """Checks what the forward call kept: the kernels read it as it was written, whole and contiguous."""
    B, Lq, H, _ = shape
    ok = [stats is not None and tuple(stats.shape) == (maps, B, H, Lq, 2) and stats.dtype == torch.float32 and stats.device == like.device
          and stats.is_contiguous(), (out2 is None) == (maps == 1)]
    if all(ok) and maps == 2:
        ok.append(tuple(out2.shape) == tuple(shape) and out2.dtype == like.dtype and out2.device == like.device and out2.is_contiguous()
                  and out2.data_ptr() % 16 == 0)
    if not all(ok):
        _fail("saved does not come from a forward call of this shape")


def _backward(name, maps, a, like, dout, w, out, saved, grads, q_len, kv_len):
    mp = (2,) if maps == 2 else ()
    stats, out2 = saved
    shape = (a.B, a.Lq, a.H, a.Dv)
    _set_strides(a, "sdo", _like("dout", dout, shape, like), False)
    _set_strides(a, "so", _like("out", out, shape, like), False)
    _saved(stats, out2, maps, shape, like)
    a.dout, a.out, a.stats = dout.data_ptr(), out.data_ptr(), stats.data_ptr()
    if maps == 2:
        a.out2 = out2.data_ptr()
    dq, dk, dv, dw = grads
    dq = _output(a, "dq", "sdq", dq, (a.B, a.Lq, a.H, *mp, a.D), like, q_len is not None)
    dk = _output(a, "dk", "sdk", dk, (a.B, a.Lk, a.Hkv, *mp, a.D), like, kv_len is not None)
    dv = _output(a, "dv", "sdv", dv, (a.B, a.Lk, a.Hkv, a.Dv), like, kv_len is not None)
    if dw is None:
        dw = torch.empty_like(w)
    elif dw.shape != w.shape or dw.dtype != w.dtype or dw.device != w.device or not dw.is_contiguous():
        _fail("the learned weights' gradient is %s %s, expected %s %s, contiguous", dw.dtype, tuple(dw.shape), w.dtype, tuple(w.shape))
    a.dw = dw.data_ptr()
    _enqueue(name, a, like.device, "sgta_attn_bwd_ws_floats", maps, _meta(name, a, maps, backward=True))
    return dq, dk, dv, dw


def rel_attention_bwd(dout, q, k, v, table, out, saved, dq=None, dk=None, dv=None, dtable=None, *, max_distance=128, bidirectional=True,
                      causal=False, scale=None, q_len=None, kv_len=None, q_start=None):
    """Gradients (dq, dk, dv, dtable) of ``rel_attention`` for the gradient ``dout`` of its ``out``; the other arguments as in the
    forward call, ``saved`` from its ``save=True``.  Shared heads' gradients are summed; rows behind q_len / kv_len are left as they
    are (zeros where allocated here).  The same inputs give the same bits."""
    a = _operands(1, q, k, v, table, causal, scale, q_len, kv_len, q_start, int(max_distance), bool(bidirectional))
    return _backward("sgta_rel_attn_bwd", 1, a, q, dout, table, out, saved, (dq, dk, dv, dtable), q_len, kv_len)


def diff_attention_bwd(dout, q, k, v, lam, out, saved, dq=None, dk=None, dv=None, dlam=None, *, lam_init=0.8, causal=False, scale=None,
                       q_len=None, kv_len=None, q_start=None):
    """Gradients (dq, dk, dv, dlam) of ``diff_attention``, as ``rel_attention_bwd``; dlam [4, D]."""
    a = _operands(2, q, k, v, lam, causal, scale, q_len, kv_len, q_start, lam_init=float(lam_init))
    return _backward("sgta_diff_attn_bwd", 2, a, q, dout, lam, out, saved, (dq, dk, dv, dlam), q_len, kv_len)
