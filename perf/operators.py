"""The attention and token operators beside the windowed attention and the token products: what is timed, on which inputs.

Three operators: attention with a learned relative position bias by buckets, differential attention (the difference of two
softmax maps), and the token product in 8-bit integers with a scale for each token and each output channel.  ``own`` selects the
framework's kernels; otherwise ``run`` is the plain form in elementary torch operations.

Tensors: q [B, Lq, H, D] (two maps: [B, Lq, H, 2, D]), k the same with the key / value heads, v [B, Lk, Hkv, Dv].
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one camera, the next frame's token against a short history: latency of the smallest call
        dict(name="rel_step_one", op="rel", mode="step", dtype="f16", B=1, Lq=1, Lk=197, H=8, Hkv=8, D=32, Dv=32,
             causal=True, ragged=False, buckets=32, far=128),
        # 16 cameras in different places of their caches, one new token each, shared key / value heads
        dict(name="rel_step", op="rel", mode="step", dtype="bf16", B=16, Lq=1, Lk=4096, H=16, Hkv=4, D=64, Dv=64,
             causal=True, ragged=True, buckets=32, far=128),
        # a batch of padded clips with the token count of the finest attention level, both directions
        dict(name="rel_encoder", op="rel", mode="fwd", dtype="bf16", B=8, Lq=1183, Lk=1183, H=8, Hkv=8, D=64, Dv=64,
             causal=False, ragged=True, buckets=32, far=128),
        # a long clip read causally in one go
        dict(name="rel_long", op="rel", mode="fwd", dtype="f16", B=1, Lq=8192, Lk=8192, H=16, Hkv=4, D=128, Dv=128,
             causal=True, ragged=False, buckets=32, far=128),
        # fine-tuning the middle attention level in full precision: 343 tokens a sample, small heads
        dict(name="rel_windows_train", op="rel", mode="train", dtype="f32", B=32, Lq=343, Lk=343, H=8, Hkv=8, D=16, Dv=16,
             causal=False, ragged=False, buckets=32, far=128),
        # an ordinary training step's attention: forward, and the gradients of everything
        dict(name="rel_train", op="rel", mode="train", dtype="bf16", B=4, Lq=2048, Lk=2048, H=16, Hkv=16, D=64, Dv=64,
             causal=False, ragged=False, buckets=32, far=128),
        # differential attention, one new token for each of 8 caches
        dict(name="diff_step", op="diff", mode="step", dtype="bf16", B=8, Lq=1, Lk=4095, H=8, Hkv=4, D=64, Dv=128,
             causal=True, ragged=True),
        # in full precision, an odd length, forward and gradients
        dict(name="diff_train_f32", op="diff", mode="train", dtype="f32", B=2, Lq=777, Lk=777, H=8, Hkv=8, D=32, Dv=64,
             causal=False, ragged=False),
        # an ordinary training step's attention, causal
        dict(name="diff_train", op="diff", mode="train", dtype="bf16", B=2, Lq=2048, Lk=2048, H=8, Hkv=8, D=64, Dv=128,
             causal=True, ragged=False),
        # the projection of four new tokens: the weights' bytes are what it costs
        dict(name="i8_step", op="i8", mode="fwd", dtype="bf16", M=4, N=4096, K=4096, bias=True, relu=False),
        # the first product of the feed-forward block on one frame pair's tokens
        dict(name="i8_tokens", op="i8", mode="fwd", dtype="f32", M=1183, N=1024, K=256, bias=True, relu=True),
        # a large batch of tokens through a square projection
        dict(name="i8_large", op="i8", mode="fwd", dtype="bf16", M=16384, N=4096, K=4096, bias=False, relu=False),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rel", "diff", "i8"])
    dtype = rng.choice(["bf16", "f16", "bf16", "f16", "f32"])
    if op == "i8":
        n, k = _spread(rng, 64, 4096), _spread(rng, 64, 4096)
        k = k if rng.random() < 0.25 else (k + 15) // 16 * 16
        return dict(op="i8", mode="fwd", dtype=dtype, M=_spread(rng, 1, 16384), N=n, K=k, bias=rng.random() < 0.5,
                    relu=rng.random() < 0.3)
    mode = rng.choice(["step", "fwd", "train"])
    hkv = rng.choice([1, 2, 4, 8])
    h = hkv * rng.choice([1, 2, 4])
    d = rng.choice([16, 32, 40, 64, 96, 128]) if op == "rel" else rng.choice([16, 32, 64])
    dv = d if op == "rel" else 2 * d
    causal, ragged = rng.random() < 0.5, rng.random() < 0.5
    if mode == "step":
        b, lq, lk, causal = _spread(rng, 1, 32), rng.choice([1, 1, 1, 2, 4]), _spread(rng, 5, 8192), True
    else:
        # scores of all heads and samples: at most what one long clip or one training step has
        most = (2 ** 28 if mode == "fwd" else 2 ** 25) // (4 if dtype == "f32" else 1)
        b = _spread(rng, 1, 16)
        lq = lk = _spread(rng, 33, max(64, min(8192 if mode == "fwd" else 2048, math.isqrt(most // (b * h)))))
    c = dict(op=op, mode=mode, dtype=dtype, B=b, Lq=lq, Lk=lk, H=h, Hkv=hkv, D=d, Dv=dv, causal=causal, ragged=ragged)
    if op == "rel":
        c.update(buckets=rng.choice([16, 32, 64]), far=rng.choice([64, 128, 200]))
    return c


def _lengths(case):
    """The samples' lengths (keys): all full, or spread evenly down to a small part of the longest."""
    B, Lk, Lq = case["B"], case["Lk"], case["Lq"]
    if not case["ragged"]:
        return [Lk] * B
    least = Lq if case["mode"] == "step" else 1
    return [max(least, Lk - (Lk * 9 // 10) * b // max(1, B - 1)) for b in range(B)]


def _maps(case):
    return 2 if case["op"] == "diff" else 1


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "i8":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": size * M * K + N * K + 4 * N + (size * N if case["bias"] else 0) + size * M * N, "flops": 2.0 * M * N * K}
    H, Hkv, D, Dv, maps, Lq = case["H"], case["Hkv"], case["D"], case["Dv"], _maps(case), case["Lq"]
    step = case["mode"] == "step"
    pairs = keys = rows = 0
    for n in _lengths(case):
        q = Lq if step else min(n, Lq)
        start = n - Lq if step else 0
        pairs += sum(min(n, start + i + 1) for i in range(q)) if case["causal"] else q * n
        keys += n
        rows += q
    kv = size * keys * Hkv * (maps * D + Dv)
    qo = size * rows * H * (maps * D + Dv)
    small = size * (case["buckets"] * H if case["op"] == "rel" else 4 * D)
    fwd = 2.0 * pairs * H * (maps * D + maps * Dv)
    if case["mode"] != "train":
        return {"bytes": kv + qo + small, "flops": fwd}
    # backward: the maps again, dO V^T, dV, and dQ, dK of each map; reads q, k, v and the output's gradient, writes four gradients
    bwd = 2.0 * pairs * H * (3 * maps * D + 2 * Dv)
    return {"bytes": 2 * (kv + qo + small) + size * rows * H * Dv, "flops": fwd + bwd}


# ----------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev, T = "cuda", TYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device=dev, generator=g)                                        # noqa: E731
    st = dict(case=case)
    if case["op"] == "i8":
        M, N, K = case["M"], case["N"], case["K"]
        # activations with a few strong channels, weights as a program holds them: 8-bit, with a scale for each row
        st["x"] = (rn(M, K) * torch.exp(0.7 * rn(K))).to(T)
        w = rn(N, K) / math.sqrt(K)
        st["ws"] = w.abs().amax(1) / 127
        st["wq"] = torch.round(w / st["ws"][:, None]).to(torch.int8)
        st["bias"] = (0.1 * rn(N)).to(T) if case["bias"] else None
        return st
    B, Lq, Lk, H, Hkv, D, Dv = (case[k] for k in ("B", "Lq", "Lk", "H", "Hkv", "D", "Dv"))
    maps = _maps(case)
    mp = (2,) if maps == 2 else ()
    if case["mode"] == "step":                                       # the caches, and the new tokens' queries
        st["q"] = rn(B, Lq, H, *mp, D).to(T)
        st["k"], st["v"] = rn(B, Lk, Hkv, *mp, D).to(T), rn(B, Lk, Hkv, Dv).to(T)
    else:                                                            # slices of one projection's output
        qkv = rn(B, Lk, (H + Hkv) * maps * D + Hkv * Dv).to(T)
        a, b = H * maps * D, (H + Hkv) * maps * D
        st["q"] = qkv[..., :a].unflatten(-1, (H, *mp, D))
        st["k"] = qkv[..., a:b].unflatten(-1, (Hkv, *mp, D))
        st["v"] = qkv[..., b:].unflatten(-1, (Hkv, Dv))
    n = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
    n = n[torch.randperm(B, device=dev, generator=g)]
    step = case["mode"] == "step"
    st["kv_len"] = n if case["ragged"] or step else None
    st["q_len"] = n if case["ragged"] and not step else None
    st["q_start"] = n - Lq if step else None
    if case["op"] == "rel":
        st["table"] = (0.7 * rn(case["buckets"], H)).to(T)
        st["bounds"] = torch.tensor(_bucket_bounds(case["buckets"] // (1 if case["causal"] else 2), case["far"]), device=dev)
    else:
        st["lam"] = (0.1 * rn(4, D)).to(T)
    if case["mode"] == "train":
        st["dout"] = rn(B, Lq, H, Dv).to(T)
    return st


# ------------------------------------------------------------------------------------------- plain forms
LAM_INIT = 0.8


def _bucket_bounds(n, far):
    """Least distances of the buckets n/2 + 1 ... n - 1: r with r^(n - n/2) >= (n/2)^(n - n/2 - k) far^k, in whole numbers."""
    e = n // 2
    m = n - e
    return [next(r for r in range(e, far + 1) if r ** m >= e ** (m - k) * far ** k) for k in range(1, m)]


def _buckets(rel, n, bounds, both):
    """Bucket of the key's position minus the query's: half the buckets for each side where both directions are seen."""
    if both:
        n //= 2
        first, r = n * (rel > 0), rel.abs()
    else:
        first, r = 0, (-rel).clamp(min=0)
    return first + torch.where(r < n // 2, r, n // 2 + torch.bucketize(r, bounds, right=True))


def _seen(st, B, Lq, Lk, dev):
    """[B or 1, Lq, Lk]: key positions minus query positions, and which keys a query sees."""
    i, j = torch.arange(Lq, device=dev)[None, :, None], torch.arange(Lk, device=dev)[None, None, :]
    pos = i if st["q_start"] is None else i + st["q_start"].long()[:, None, None]
    rel = j - pos
    seen = torch.ones_like(rel, dtype=torch.bool)
    if st["case"]["causal"]:
        seen = rel <= 0
    if st["kv_len"] is not None:
        seen = seen & (j < st["kv_len"][:, None, None])
    if st["q_len"] is not None:
        seen = seen & (i < st["q_len"][:, None, None])
    return rel, seen


def _softmax(s, seen):
    s = torch.where(seen, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _heads(t, G):
    """[B, L, heads, ...] as [B, all query heads, L, ...] in 32 bits."""
    t = t.float().transpose(1, 2)
    return t if G == 1 else t.repeat_interleave(G, 1)


def _back(t, heads, T):
    """[B, all query heads, L, d] summed over the query heads that share one, as [B, L, heads, d]."""
    B, H, L, d = t.shape
    return (t.reshape(B, heads, H // heads, L, d).sum(2) if H != heads else t).transpose(1, 2).to(T).contiguous()


def _plain_rel(st):
    c = st["case"]
    q, k, v, table = st["q"], st["k"], st["v"], st["table"]
    T, (B, Lq, H, D), Lk, Hkv = q.dtype, q.shape, k.shape[1], k.shape[2]
    G, scale = H // Hkv, D ** -0.5
    rel, seen = _seen(st, B, Lq, Lk, q.device)
    bucket = _buckets(rel, c["buckets"], st["bounds"], not c["causal"])
    bias = table.float().t()[:, bucket].transpose(0, 1)                             # [B or 1, H, Lq, Lk]
    Q, K, V = _heads(q, 1), _heads(k, G), _heads(v, G)
    p = _softmax(scale * (Q @ K.transpose(-1, -2).contiguous()) + bias, seen[:, None])
    out = (p @ V).transpose(1, 2).to(T).contiguous()
    if c["mode"] != "train":
        return out
    dO = _heads(st["dout"], 1)
    dP = dO @ V.transpose(-1, -2).contiguous()
    dS = p * (dP - (p * dP).sum(-1, keepdim=True))
    dq = scale * (dS @ K)
    dk = scale * (dS.transpose(-1, -2).contiguous() @ Q)
    dv = p.transpose(-1, -2).contiguous() @ dO
    # the table's gradient, in 64 bits: sums along the diagonals, by reading the rows of Lq + Lk again in rows of one more, so
    # that (i, j) stands in column j - i (mod the rows' length); then sums of the diagonals of one bucket
    W = Lq + Lk + 1
    wide = torch.zeros(H, Lq, W, dtype=torch.float64, device=q.device)
    wide.view(H, -1)[:, : Lq * (W - 1)].view(H, Lq, W - 1)[..., :Lk] = dS.sum(0, dtype=torch.float64)
    away = torch.arange(1 - Lq, Lk, device=q.device)
    of = _buckets(away, c["buckets"], st["bounds"], not c["causal"])
    hit = (of[:, None] == torch.arange(c["buckets"], device=q.device)).double()
    dtable = (wide.sum(1)[:, away % W] @ hit).t()
    return out, _back(dq, H, T), _back(dk, Hkv, T), _back(dv, Hkv, T), dtable.to(T).contiguous()


def _lambda(lam):
    a, b = (lam[0] * lam[1]).sum(), (lam[2] * lam[3]).sum()
    return torch.exp(a), torch.exp(b)


def _plain_diff(st):
    c = st["case"]
    q, k, v = st["q"], st["k"], st["v"]
    T, (B, Lq, H, _, D), Lk, Hkv = q.dtype, q.shape, k.shape[1], k.shape[2]
    G, scale = H // Hkv, D ** -0.5
    lam = st["lam"].float()
    e1, e2 = _lambda(lam)
    lm = e1 - e2 + LAM_INIT
    seen = _seen(st, B, Lq, Lk, q.device)[1][:, None]
    Q1, Q2, K1, K2 = (_heads(t[:, :, :, m], g) for t, g in ((q, 1), (k, G)) for m in (0, 1))
    V = _heads(v, G)
    p1 = _softmax(scale * (Q1 @ K1.transpose(-1, -2).contiguous()), seen)
    p2 = _softmax(scale * (Q2 @ K2.transpose(-1, -2).contiguous()), seen)
    p = p1 - lm * p2
    out = (p @ V).transpose(1, 2).to(T).contiguous()
    if c["mode"] != "train":
        return out
    dO = _heads(st["dout"], 1)
    X = dO @ V.transpose(-1, -2).contiguous()
    d2 = (p2 * X).sum(-1, keepdim=True)
    dS1 = p1 * (X - (p1 * X).sum(-1, keepdim=True))
    dS2 = -lm * p2 * (X - d2)
    dq = torch.stack([_back(scale * (dS1 @ K1), H, T), _back(scale * (dS2 @ K2), H, T)], 3)
    dk = torch.stack([_back(scale * (dS1.transpose(-1, -2).contiguous() @ Q1), Hkv, T),
                      _back(scale * (dS2.transpose(-1, -2).contiguous() @ Q2), Hkv, T)], 3)
    dv = _back(p.transpose(-1, -2).contiguous() @ dO, Hkv, T)
    dlm = -d2.double().sum()
    dlam = torch.stack([dlm * e1 * lam[1], dlm * e1 * lam[0], -dlm * e2 * lam[3], -dlm * e2 * lam[2]])
    return out, dq, dk, dv, dlam.to(T)


def _plain_i8(st):
    c, x = st["case"], st["x"].float()
    xs = x.abs().amax(1, keepdim=True) / 127
    # in 64 bits: quotients next to a half, and sums of whole numbers beyond 2^24
    xq = torch.where(xs > 0, torch.round(x.double() / xs), 0.0).clamp(-127, 127)
    y = (xq @ st["wq"].double().t()).float() * (xs * st["ws"])
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return (y.clamp(min=0) if c["relu"] else y).to(st["x"].dtype)


# ------------------------------------------------------------------------------------------- the kernels
def _own(st):
    from sgtapose_amd import ops_attn, ops_i8
    c = st["case"]
    if c["op"] == "i8":
        xq, xs = ops_i8.quantize_rows(st["x"])
        return ops_i8.linear_i8(xq, xs, st["wq"], st["ws"], st["bias"], relu=c["relu"], dtype=st["x"].dtype)
    seen = dict(causal=c["causal"], q_len=st["q_len"], kv_len=st["kv_len"], q_start=st["q_start"])
    train = c["mode"] == "train"
    if c["op"] == "rel":
        buckets = dict(max_distance=c["far"], bidirectional=not c["causal"])
        if not train:
            return ops_attn.rel_attention(st["q"], st["k"], st["v"], st["table"], **buckets, **seen)
        out, saved = ops_attn.rel_attention(st["q"], st["k"], st["v"], st["table"], **buckets, **seen, save=True)
        return (out, *ops_attn.rel_attention_bwd(st["dout"], st["q"], st["k"], st["v"], st["table"], out, saved, **buckets, **seen))
    if not train:
        return ops_attn.diff_attention(st["q"], st["k"], st["v"], st["lam"], lam_init=LAM_INIT, **seen)
    out, saved = ops_attn.diff_attention(st["q"], st["k"], st["v"], st["lam"], lam_init=LAM_INIT, **seen, save=True)
    return (out, *ops_attn.diff_attention_bwd(st["dout"], st["q"], st["k"], st["v"], st["lam"], out, saved, lam_init=LAM_INIT, **seen))


def run(state):
    if own:
        return _own(state)
    return {"rel": _plain_rel, "diff": _plain_diff, "i8": _plain_i8}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------- in 64 bits
def _exact_bucket(d, n, far, both):
    """One distance's bucket, from the definition: exact up to half the buckets, logarithmic from there to ``far``."""
    at = 0
    if both:
        n //= 2
        at, d = (n if d > 0 else 0), abs(d)
    else:
        d = max(-d, 0)
    e = n // 2
    if d < e:
        return at + d
    return at + min(n - 1, e + math.floor(math.log(d / e) / math.log(far / e) * (n - e) + 1e-9))


def _exact_map(q, k, bias, hidden):
    s = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(q.shape[-1])
    s = (s if bias is None else s + bias).masked_fill(hidden, -math.inf)
    return torch.nan_to_num(torch.softmax(s, -1), nan=0.0) if bool(hidden.all(-1).any()) else torch.softmax(s, -1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "i8":
        x, w = st["x"].double(), st["wq"].double() * st["ws"].double()[:, None]
        xs = (x.abs().amax(1, keepdim=True) / 127).float().double()
        xq = torch.nan_to_num(x / xs).round()
        y = torch.nn.functional.linear(xq * xs, w, None if st["bias"] is None else st["bias"].double())
        return torch.relu(y) if case["relu"] else y
    train, B, Lq, Lk = case["mode"] == "train", case["B"], case["Lq"], case["Lk"]
    G = case["H"] // case["Hkv"]
    names = ("q", "k", "v", "table" if case["op"] == "rel" else "lam")
    leaf = {n: st[n].double().requires_grad_(train) for n in names}
    zero = torch.zeros(B, dtype=torch.int64, device="cuda")
    first = zero if st["q_start"] is None else st["q_start"].long()
    nk = zero + Lk if st["kv_len"] is None else st["kv_len"].long()
    nq = zero + Lq if st["q_len"] is None else st["q_len"].long()
    jj, ii = torch.arange(Lk, device="cuda"), torch.arange(Lq, device="cuda")
    away = jj[None, None] - ii[None, :, None] - first[:, None, None]                # [B, Lq, Lk]
    hidden = (jj[None, None] >= nk[:, None, None]) | (ii[None, :, None] >= nq[:, None, None])
    if case["causal"]:
        hidden = hidden | (away > 0)
    if st["q_start"] is None:
        away = away[:1]
    if not case["ragged"] and st["q_start"] is None:
        hidden = hidden[:1]
    hidden = hidden[:, None]
    q, k = leaf["q"], leaf["k"].repeat_interleave(G, 2)
    v = leaf["v"].repeat_interleave(G, 2)
    if case["op"] == "rel":
        lo, hi = int(away.min()), int(away.max())
        of = torch.tensor([_exact_bucket(d, case["buckets"], case["far"], not case["causal"]) for d in range(lo, hi + 1)],
                          device="cuda")
        bias = _Gather.apply(leaf["table"], of[away - lo])
        y = torch.einsum("bhij,bjhd->bihd", _exact_map(q, k, bias, hidden), v)
    else:
        lam = leaf["lam"]
        size = torch.exp(lam[0].dot(lam[1])) - torch.exp(lam[2].dot(lam[3])) + LAM_INIT
        one, two = (_exact_map(q[:, :, :, m], k[:, :, :, m], None, hidden) for m in (0, 1))
        y = torch.einsum("bhij,bjhd->bihd", one - size * two, v)
    if not train:
        return y
    grads = torch.autograd.grad(y, [leaf[n] for n in names], st["dout"].double())
    return (y.detach(), *grads)


class _Gather(torch.autograd.Function):
    """table [buckets, H] by a bucket for each pair [B or 1, Lq, Lk] -> [B or 1, H, Lq, Lk]; the gradient is a product with the
    buckets' indicators."""

    @staticmethod
    def forward(ctx, table, bucket):
        ctx.save_for_backward(bucket)
        ctx.n = table.shape[0]
        return table.t()[:, bucket].transpose(0, 1)

    @staticmethod
    def backward(ctx, g):
        hit = torch.nn.functional.one_hot(ctx.saved_tensors[0].reshape(-1), ctx.n).double()
        return (g.transpose(0, 1).reshape(g.shape[1], -1) @ hit).t(), None
