"""Attention with a bucketed relative bias and differential attention (sgtapose_amd/ops_attn.py) against the formulas in 64 bits.

Tolerances are bounds, element by element, from the arithmetic of the kernels (u = eps / 2 of the element type, e = 2^-24):
  scores    D products summed in f32 (float operands as three bfloat16 numbers, whose smallest products, 3 e of |q||k|, are
            left out), times the scale, plus the bias, minus the reference: off by at most
            es = e ((D + 6) scale sum|q||k| + 4 |s| + 16), so a weight is off by a factor exp(2 es) (its own score and the sum's)
  weights   rounded to the element type before the product with v: u of each (IEEE half: 2^-25 at least, where it is subnormal)
  sums      Lk terms in f32: e (Lk + 3) of the sum of magnitudes
  output    rounded once more: u |o|
Gradients, with a = 4 es + e Lk for the relative error of a weight from the saved statistics:
  X = dO V^T   e (Dv + 5) |dO||V|^T;   delta: |dO| times the output's bound, and e (Dv + 2) |dO||O|
  dS           a |dS| + P (X's + delta's); rounded to the element type: u |dS| (IEEE half: scaled to |dO| next to one, so 2^-24 of it at least)
  dQ, dK, dV   the sums of those errors times the other operand's magnitude, e per term of the sum and 3 e, u of the result
"""
import math

import pytest
import torch

from sgtapose_amd import ops_attn
from sgtapose_amd._lib import SgtaHipError

gpu = pytest.mark.gpu
E = 2.0 ** -24
U = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
FLUSH = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
ALL = [torch.float32, torch.float16, torch.bfloat16]
NAMES = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}


# ---- the formulas, in 64 bits -----------------------------------------------------------------
def bucket_of(d, n, far, both):
    at = 0
    if both:
        n //= 2
        at, d = (n if d > 0 else 0), abs(d)
    else:
        d = max(-d, 0)
    if d < n // 2:
        return at + d
    return at + min(n - 1, n // 2 + math.floor(math.log(d / (n // 2)) / math.log(far / (n // 2)) * (n - n // 2) + 1e-9))


class Case:
    """Inputs of one call and everything a bound needs, in float64 on the CPU."""

    def __init__(self, maps, dtype, B, Lq, Lk, H, Hkv, D, Dv=None, causal=False, q_len=None, kv_len=None, q_start=None, buckets=32, far=40,
                 seed=0, scale=None, dout_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        Dv = D if Dv is None else Dv
        mp = (2,) if maps == 2 else ()
        rn = lambda *s: torch.randn(*s, generator=g)                                              # noqa: E731
        self.maps, self.dtype, self.causal, self.buckets, self.far = maps, dtype, causal, buckets, far
        self.dims = (B, Lq, Lk, H, Hkv, D, Dv)
        self.q, self.k, self.v = rn(B, Lq, H, *mp, D).to(dtype), rn(B, Lk, Hkv, *mp, D).to(dtype), rn(B, Lk, Hkv, Dv).to(dtype)
        self.w = (rn(buckets, H) if maps == 1 else 0.3 * rn(4, D)).to(dtype)
        self.dout = (dout_scale * rn(B, Lq, H, Dv)).to(dtype)
        self.lens = dict(q_len=q_len, kv_len=kv_len, q_start=q_start)
        self.scale = scale

    def kwargs(self, dev):
        kw = {n: None if t is None else torch.tensor(t, dtype=torch.int32, device=dev) for n, t in self.lens.items()}
        kw.update(causal=self.causal, scale=self.scale)
        if self.maps == 1:
            kw.update(max_distance=self.far, bidirectional=not self.causal)
        return kw

    def reference(self):
        """-> dict of float64 results and bounds."""
        B, Lq, Lk, H, Hkv, D, Dv = self.dims
        G, T = H // Hkv, self.dtype
        f = lambda t: t.double()                                                                  # noqa: E731
        nq = torch.tensor(self.lens["q_len"] or [Lq] * B).clamp(0, Lq)
        nk = torch.tensor(self.lens["kv_len"] or [Lk] * B).clamp(0, Lk)
        st = torch.tensor(self.lens["q_start"] or [0] * B)
        i, j = torch.arange(Lq), torch.arange(Lk)
        rel = j[None, None] - i[None, :, None] - st[:, None, None]
        seen = (j[None, None] < nk[:, None, None]) & (i[None, :, None] < nq[:, None, None])
        if self.causal:
            seen = seen & (rel <= 0)
        seen = seen[:, None]
        # what lies behind the lengths takes no part, whatever it is
        q, k, v, do = (torch.where((torch.arange(t.shape[1])[None] < n[:, None]).reshape(B, -1, *[1] * (t.dim() - 2)), f(t), 0.0)
                       for t, n in ((self.q, nq), (self.k, nk), (self.v, nk), (self.dout, nq)))
        q, do = q.transpose(1, 2), do.transpose(1, 2)
        k, v = k.transpose(1, 2).repeat_interleave(G, 1), v.transpose(1, 2).repeat_interleave(G, 1)
        c = D ** -0.5 if self.scale is None else self.scale
        bias = 0.0
        if self.maps == 1:
            rel = rel.clamp(-self.far, self.far)                    # the buckets stay the same from there on
            lo, hi = int(rel.min()), int(rel.max())
            of = torch.tensor([bucket_of(d, self.buckets, self.far, not self.causal) for d in range(lo, hi + 1)])[rel - lo]
            bias = f(self.w)[of].permute(0, 3, 1, 2)
        P, es, qs, ks, mags = [], [], [], [], []
        for p in range(self.maps):
            qp, kp = (q, k) if self.maps == 1 else (q[:, :, :, p], k[:, :, :, p])
            s = c * (qp @ kp.transpose(-1, -2)) + bias
            mag = c * (qp.abs() @ kp.abs().transpose(-1, -2))
            es.append(E * ((D + 6) * mag + 4 * s.abs().clamp(max=1e4) + 16).amax((-1, -2), keepdim=True))
            s = torch.where(seen, s, -math.inf)
            m = s.amax(-1, keepdim=True)
            e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
            t = e.sum(-1, keepdim=True)
            P.append(e / torch.where(t == 0, 1.0, t))
            qs.append(qp)
            ks.append(kp)
        u, tiny, sums = U[T], FLUSH[T], (Lk + 3) * E
        lam, lam_err = 0.0, 0.0
        if self.maps == 2:
            w = f(self.w)
            e1, e2 = torch.exp((w[0] * w[1]).sum()), torch.exp((w[2] * w[3]).sum())
            lam = e1 - e2 + 0.8
            lam_err = float(E * (D + 8) * (e1 * (1 + (w[0] * w[1]).abs().sum()) + e2 * (1 + (w[2] * w[3]).abs().sum()) + 2))
        sgn = (1.0, -lam)
        o = sum(sgn[p] * (P[p] @ v) for p in range(self.maps))
        va = v.abs()
        o_mid = sum(abs(sgn[p]) * ((u + 2 * es[p] + sums) * (P[p] @ va) + tiny * (seen.double() @ va)) for p in range(self.maps))
        if self.maps == 2:
            o_mid = o_mid + lam_err * (P[1] @ va)
        r = dict(out=o.transpose(1, 2), out_tol=(o_mid * 1.01 + u * o.abs() + 4 * E * o.abs() + 1e-30).transpose(1, 2), nq=nq, nk=nk, P=P)
        self.parts = dict(q=qs, k=ks, v=v, do=do, P=P, es=es, c=c, seen=seen, lam=lam, o_mid=o_mid, u=u, tiny=tiny, sums=sums,
                          of=of if self.maps == 1 else None, st=st, nq=nq, nk=nk)
        return r


def gradients(c):
    """-> {name: (gradient, bound)} in float64 for c.dout (after c.reference())."""
    r = c.reference()
    z = c.parts
    B, Lq, Lk, H, Hkv, D, Dv = c.dims
    G, u, P, v, do, lam = H // Hkv, z["u"], z["P"], z["v"], z["do"], z["lam"]
    X, Xe = do @ v.transpose(-1, -2), E * (Dv + 5) * (do.abs() @ v.abs().transpose(-1, -2))
    top = do.abs().amax() * 2
    tiny = 2.0 ** -24 * top if c.dtype == torch.float16 else 0.0
    sgn = (1.0, -lam)
    o = [P[p] @ v for p in range(c.maps)]
    out = sum(sgn[p] * o[p] for p in range(c.maps))
    a = [4 * e + z["sums"] + 16 * E for e in z["es"]]
    dsum = lambda t: (do.abs() * t).sum(-1, keepdim=True)                                         # noqa: E731
    d_err = dsum(z["o_mid"] + u * out.abs()) + E * (Dv + 2) * dsum(out.abs())
    res, dS, Se = {}, [], []
    d2 = d2_err = None
    if c.maps == 2:
        d2 = (do * o[1]).sum(-1, keepdim=True)
        d2_err = dsum((u + a[1]) * (P[1] @ v.abs()) + z["tiny"] * (z["seen"].double() @ v.abs()) + u * o[1].abs()) + E * (Dv + 2) * dsum(o[1].abs())
        d_err = d_err + abs(lam) * d2_err
    for p in range(c.maps):
        d = (do * o[p]).sum(-1, keepdim=True)
        t = sgn[p] * P[p] * (X - d)
        dS.append(t)
        Se.append(a[p] * t.abs() + abs(sgn[p]) * P[p] * (Xe + (d_err if p == 0 else d2_err)) + (8 * E * t.abs() if c.maps == 2 else 0.0))
    shared = lambda t: t.reshape(B, Hkv, G, *t.shape[2:]).sum(2)                                  # noqa: E731
    back = lambda t: t.transpose(1, 2)                                                            # noqa: E731

    def pack(name, parts):
        val, err = (torch.stack([x[i] for x in parts], 3) if c.maps == 2 and name != "dv" else parts[0][i] for i in (0, 1))
        # a half below 2^-14 has steps of 2^-24 whatever its size, so its rounding is off by up to 2^-25 rather than u of it
        res[name] = (val, err * 1.01 + u * val.abs() + 2 * E * val.abs() + FLUSH[c.dtype] + 1e-30)
    dq, dk = [], []
    for p in range(c.maps):
        k, q, m = z["k"][p], z["q"][p], dS[p].abs()
        e = Se[p] + (u + (Lk + 3) * E) * m + tiny
        dq.append((back(z["c"] * (dS[p] @ k)), back(z["c"] * (e @ k.abs()))))
        e = Se[p] + (u + (Lq * G + 3) * E) * m + tiny
        dk.append((back(shared(z["c"] * (dS[p].transpose(-1, -2) @ q))), back(shared(z["c"] * (e.transpose(-1, -2) @ q.abs())))))
    w = sum(sgn[p] * P[p] for p in range(c.maps))
    we = sum(abs(sgn[p]) * a[p] * P[p] for p in range(c.maps)) + (u + (Lq * G + 3) * E) * sum(abs(sgn[p]) * P[p] for p in range(c.maps)) + z["tiny"]
    if c.maps == 2:
        we = we + 1e-5 * P[1]
    pack("dq", dq)
    pack("dk", dk)
    pack("dv", [(back(shared(w.transpose(-1, -2) @ do)), back(shared(we.transpose(-1, -2) @ do.abs())))])
    if c.maps == 1:
        hit = torch.nn.functional.one_hot(z["of"], c.buckets).double()                            # [B, Lq, Lk, buckets]
        tot = lambda t: torch.einsum("bhij,bijn->nh", t, hit)                                     # noqa: E731
        val, err = tot(dS[0]), tot(Se[0] + (Lk + 200) * E * dS[0].abs())
    else:
        wt = c.w.double()
        e1, e2 = torch.exp((wt[0] * wt[1]).sum()), torch.exp((wt[2] * wt[3]).sum())
        dl, de = -d2.sum(), (d2_err + 300 * E * d2.abs()).sum()
        val = torch.stack([dl * e1 * wt[1], dl * e1 * wt[0], -dl * e2 * wt[3], -dl * e2 * wt[2]])
        err = (de + 1e-5 * dl.abs()) * torch.stack([e1 * wt[1].abs(), e1 * wt[0].abs(), e2 * wt[3].abs(), e2 * wt[2].abs()])
    res["dw"] = (val, err * 1.01 + u * val.abs() + 4 * E * val.abs() + FLUSH[c.dtype] + 1e-30)
    return r, res


def within(name, got, want, tol, rows=None):
    d = (got.double().cpu() - want).abs()
    tol_all = tol
    if rows is not None:
        keep = torch.arange(got.shape[1])[None] < rows[:, None]
        d, tol = d[keep], tol.expand(want.shape)[keep]
    bad = ~(d <= tol)
    # what exceeds the type's range becomes an infinity of its sign: right where the value, give or take its bound, does
    beyond = got.double().cpu().isinf() & (want * got.double().cpu().sign() + tol_all >= torch.finfo(got.dtype).max)
    bad &= ~(beyond if rows is None else beyond[keep])
    assert not bad.any(), "%s: %d of %d beyond the bound, worst %.3g against %.3g" % (
        name, int(bad.sum()), bad.numel(), float(d[bad].max()), float(tol.expand(d.shape)[bad].min()))


def forward(c, dev="cuda", **more):
    fn = ops_attn.rel_attention if c.maps == 1 else ops_attn.diff_attention
    return fn(c.q.to(dev), c.k.to(dev), c.v.to(dev), c.w.to(dev), **c.kwargs(dev), **more)


def check_forward(c):
    r = c.reference()
    got = forward(c)
    torch.cuda.synchronize()
    within("out", got, r["out"], r["out_tol"], r["nq"])
    return got


def both_ways(c, dev="cuda", **grads):
    t = [x.to(dev) for x in (c.q, c.k, c.v, c.w)]
    kw = c.kwargs(dev)
    fwd, bwd = ((ops_attn.rel_attention, ops_attn.rel_attention_bwd) if c.maps == 1 else (ops_attn.diff_attention, ops_attn.diff_attention_bwd))
    out, saved = fwd(*t, **kw, save=True)
    return out, bwd(c.dout.to(dev), *t, out, saved, **kw, **grads)


def check_both(c):
    r, want = gradients(c)
    out, got = both_ways(c)
    torch.cuda.synchronize()
    within("out", out, r["out"], r["out_tol"], r["nq"])
    rows = dict(dq=r["nq"], dk=r["nk"], dv=r["nk"])
    for name, g in zip(("dq", "dk", "dv", "dw"), got):
        within(name, g, *want[name], rows.get(name))
        if name in rows:
            behind = torch.arange(g.shape[1])[None] >= rows[name][:, None]
            assert bool((g.cpu()[behind] == 0).all()), name
    return out, got


# ---- host ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,far,both", [(32, 128, True), (32, 128, False), (16, 64, True), (64, 200, False), (4, 5, True), (2, 2, False),
                                        (6, 1024, True)])
def test_buckets_follow_the_definition(n, far, both):
    if both and n // 2 < 2:
        pytest.skip("one bucket a direction")
    got = ops_attn.relative_buckets(n, far, both)
    reach = ops_attn.bucket_reach(n, far, both)
    assert len(got) == 2 * reach + 1
    assert got == [bucket_of(d, n, far, both) for d in range(-reach, reach + 1)]
    assert bucket_of(-far - 7, n, far, both) == got[0] and bucket_of(far + 7, n, far, both) == got[-1]


def _cpu(maps=1, B=2, Lq=5, Lk=7, H=4, Hkv=2, D=16, Dv=None, dtype=torch.bfloat16):
    mp = (2,) if maps == 2 else ()
    z = lambda *s: torch.zeros(*s, dtype=dtype)                                                   # noqa: E731
    return [z(B, Lq, H, *mp, D), z(B, Lk, Hkv, *mp, D), z(B, Lk, Hkv, Dv or D), z(32, H) if maps == 1 else z(4, D)]


@pytest.mark.parametrize("what,change", [
    ("heads not shared evenly", dict(H=4, Hkv=3)), ("head size not a multiple of 8", dict(D=12)), ("head size too large", dict(D=136)),
    ("no keys", dict(Lk=0)), ("a type that has no kernel", dict(dtype=torch.float64)), ("different head sizes", dict(D=16, Dv=32))])
def test_rel_attention_refuses_shapes(what, change):
    with pytest.raises(SgtaHipError):
        ops_attn.rel_attention(*_cpu(**change))


@pytest.mark.parametrize("change", [dict(D=72), dict(D=64, Dv=136), dict(Hkv=3), dict(Lq=0), dict(D=20)])
def test_diff_attention_refuses_shapes(change):
    with pytest.raises(SgtaHipError):
        ops_attn.diff_attention(*_cpu(2, **change))


def test_refuses_what_is_not_on_the_gpu_and_bad_operands():
    for maps, fn in ((1, ops_attn.rel_attention), (2, ops_attn.diff_attention)):
        q, k, v, w = _cpu(maps)
        with pytest.raises(SgtaHipError, match="GPU"):
            fn(q, k, v, w)
        with pytest.raises(SgtaHipError):
            fn(q, k.float(), v, w)
        with pytest.raises(SgtaHipError):
            fn(q, k, v[:1], w)
        with pytest.raises(SgtaHipError):
            fn(q, k, v, w[:, :-1])
        with pytest.raises(SgtaHipError, match="contiguous"):
            fn(q.transpose(-1, -2).contiguous().transpose(-1, -2), k, v, w)
        with pytest.raises(SgtaHipError, match="kv_len"):
            fn(q, k, v, w, kv_len=torch.zeros(2, dtype=torch.int64))
        for bad in (0.0, -1.0, math.inf, math.nan):
            with pytest.raises(SgtaHipError, match="scale"):
                fn(q, k, v, w, scale=bad)
    q, k, v, w = _cpu()
    for kw in (dict(max_distance=8), dict(max_distance=2000), dict(bidirectional=False, max_distance=16)):
        with pytest.raises(SgtaHipError, match="max_distance"):
            ops_attn.rel_attention(q, k, v, w, **kw)
    with pytest.raises(SgtaHipError, match="buckets"):
        ops_attn.rel_attention(q, k, v, w[:3])


def test_c_entries_refuse_before_they_launch():
    import ctypes
    from sgtapose_amd import _lib
    lib = _lib.load()
    ok = dict(q=64, k=64, v=64, w=64, out=64, lut=64, B=1, Lq=4, Lk=4, H=2, Hkv=2, D=16, Dv=16, dtype=2, reach=8, num_buckets=8, scale=0.25)
    for change in (dict(q=None), dict(q=65), dict(H=3), dict(D=12), dict(Dv=24), dict(dtype=3), dict(scale=0.0), dict(reach=0), dict(reach=1025),
                   dict(lut=None), dict(Lk=0), dict(sq=(ctypes.c_long * 4)(16, 4, 16, 0)), dict(Lq=1 << 29), dict(out=None)):
        a = _lib.AttnArgs(**{**ok, **change})
        assert lib.sgta_rel_attn_fwd(ctypes.byref(a), None) < 0, change
        assert lib.sgta_attn_fwd_ws_floats(ctypes.byref(a), 1) == 0
    assert lib.sgta_rel_attn_fwd(None, None) < 0 and lib.sgta_diff_attn_fwd(None, None) < 0
    a = _lib.AttnArgs(**{**ok, "Lk": 1 << 20})                        # parts of the keys need a workspace
    assert lib.sgta_attn_fwd_ws_floats(ctypes.byref(a), 1) > 0 and lib.sgta_rel_attn_fwd(ctypes.byref(a), None) < 0


# ---- forward --------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1, 1, 1), (2, 1, 33, 2, 1), (1, 5, 64, 4, 4), (2, 33, 129, 4, 2), (1, 128, 128, 2, 2), (2, 129, 65, 3, 1), (1, 300, 517, 2, 1)]


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rel_forward(dtype, causal, shape):
    B, Lq, Lk, H, Hkv = shape
    for D in (16, 64, 128):
        check_forward(Case(1, dtype, B, Lq, Lk, H, Hkv, D, causal=causal, seed=D, q_start=[max(0, Lk - Lq)] * B if causal else None))


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_diff_forward(dtype, causal, shape):
    B, Lq, Lk, H, Hkv = shape
    for D, Dv in ((16, 32), (64, 128), (40, 24)):
        check_forward(Case(2, dtype, B, Lq, Lk, H, Hkv, D, Dv, causal=causal, seed=D, q_start=[max(0, Lk - Lq)] * B if causal else None))


@gpu
@pytest.mark.parametrize("D", [8, 24, 32, 40, 96, 104])
def test_rel_forward_head_sizes(D):
    for dtype in ALL:
        check_forward(Case(1, dtype, 2, 70, 90, 2, 2, D, seed=D))
        check_forward(Case(1, dtype, 2, 2, 90, 4, 2, D, seed=D))


@gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("Lq", [1, 3, 150])
def test_lengths_and_starts(maps, Lq):
    """Empty sequences, one key, all keys; starts before the first key (a causal query that sees nothing) and past the last;
    whatever lies behind the lengths (here NaN) takes no part, output rows behind the queries stay as they are."""
    for causal in (False, True):
        c = Case(maps, torch.bfloat16, 6, Lq, 200, 4, 2, 32, causal=causal, kv_len=[0, 1, 200, 77, 128, 500], seed=Lq,
                 q_len=[Lq, Lq, 0, max(1, Lq // 2), Lq, Lq + 9], q_start=[0, 0, 3, 76, -5, 2 ** 30 + 5])
        r = c.reference()
        for b in range(6):
            c.k[b, min(200, c.lens["kv_len"][b]):] = math.nan
            c.v[b, min(200, c.lens["kv_len"][b]):] = math.nan
            c.q[b, min(Lq, c.lens["q_len"][b]):] = math.nan
        out = torch.full((6, Lq, 4, 32), 7.0, dtype=torch.bfloat16, device="cuda")
        forward(c, out=out)
        within("out", out, r["out"], r["out_tol"], r["nq"])
        behind = torch.arange(Lq)[None] >= r["nq"][:, None]
        assert bool((out.cpu()[behind] == 7.0).all())
        assert bool((out[0].cpu()[: int(r["nq"][0])] == 0).all())
        fresh = forward(c)
        assert bool((fresh.cpu()[behind] == 0).all()) and torch.equal(fresh.cpu()[~behind], out.cpu()[~behind])


@gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_few_queries_against_long_caches(maps, dtype):
    """The split over the keys: lengths around the parts' ends, several rows a head, shared heads."""
    for Lq, H, Hkv, Lk in ((1, 8, 2, 2500), (4, 8, 1, 1025), (1, 1, 1, 5000), (8, 4, 1, 513)):
        n = [Lk, Lk - 1, 129]
        check_forward(Case(maps, dtype, 3, Lq, Lk, H, Hkv, 64, 64 if maps == 1 else 128, causal=True, kv_len=n, q_start=[x - Lq for x in n], seed=Lq))


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("Lq,Lk", [(1, 300), (200, 300)])
def test_rel_table_infinities_and_lowest_values(dtype, Lq, Lk):
    """-inf hides a bucket's keys, the type's lowest value weighs nothing beside others and evenly among its like."""
    for causal in (False, True):
        for value in (-math.inf, torch.finfo(dtype).min):
            c = Case(1, dtype, 1, Lq, Lk, 2, 2, 32, causal=causal, q_start=[Lk - Lq] if causal else None)
            c.w[::2] = value
            check_forward(c)
            if value == -math.inf:
                c.w[:] = value                                       # every row is empty: zeros
                assert bool((forward(c) == 0).all())
        c = Case(1, dtype, 1, Lq, Lk, 2, 2, 32, causal=causal, q_start=[Lk - Lq] if causal else None)
        c.w[:] = torch.finfo(dtype).min                              # all buckets at the lowest value: equal weights
        check_forward(c)


@gpu
def test_strided_operands_and_output():
    """Slices of one projection, a cache in another order, an output inside a wider buffer."""
    for maps in (1, 2):
        for Lq in (2, 150):
            c = Case(maps, torch.float16, 2, Lq, 150, 4, 2, 32, seed=5)
            r = c.reference()
            mp = (2,) if maps == 2 else ()
            wide = torch.randn(2, Lq, 4, 3, *mp, 32, device="cuda").half()
            q = wide[:, :, :, 1]
            q.copy_(c.q)
            k = c.k.cuda().transpose(1, 2).contiguous().transpose(1, 2)                   # [B, heads, L, D] in memory
            v = c.v.cuda().permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3)           # [L, B, heads, D]
            buf = torch.full((2, Lq, 4, 64), 5.0, device="cuda").half()
            fn = ops_attn.rel_attention if maps == 1 else ops_attn.diff_attention
            fn(q, k, v, c.w.cuda(), buf[..., 32:], **c.kwargs("cuda"))
            within("out", buf[..., 32:].contiguous(), r["out"], r["out_tol"])
            assert bool((buf[..., :32] == 5).all())
            one = c.k[:1].cuda().expand(2, -1, *[-1] * (c.k.dim() - 2))                   # one cache for both samples
            got = fn(c.q.cuda(), one, c.v.cuda(), c.w.cuda(), **c.kwargs("cuda"))
            c.k[1] = c.k[0]
            r = c.reference()
            within("out", got, r["out"], r["out_tol"])
            with pytest.raises(SgtaHipError, match="share memory"):
                fn(q, k, v, c.w.cuda(), buf[:1, ..., 32:].expand(2, -1, -1, -1), **c.kwargs("cuda"))


@gpu
def test_streams_and_graphs():
    """On a stream that is not the current device's default, and captured: every replay gives what the eager call gives."""
    for maps in (1, 2):
        for Lq, Lk in ((1, 1500), (140, 200)):
            c = Case(maps, torch.bfloat16, 2, Lq, Lk, 4, 2, 64, seed=9)
            t = [x.cuda() for x in (c.q, c.k, c.v, c.w)]
            kw = c.kwargs("cuda")
            fn = ops_attn.rel_attention if maps == 1 else ops_attn.diff_attention
            want = fn(*t, **kw)
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                other = fn(*t, **kw)
            s.synchronize()
            assert torch.equal(other, want)
            out = torch.empty_like(want)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                fn(*t, out, **kw)
            for n in range(3):
                t[0].copy_(c.q * (n + 1))
                want = fn(*t, **kw)
                out.zero_()
                g.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, want)


# ---- gradients ------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rel_gradients(dtype, causal, shape):
    B, Lq, Lk, H, Hkv = shape
    for D in (16, 64, 128):
        check_both(Case(1, dtype, B, Lq, Lk, H, Hkv, D, causal=causal, seed=D, q_start=[max(0, Lk - Lq)] * B if causal else None))


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_diff_gradients(dtype, causal, shape):
    B, Lq, Lk, H, Hkv = shape
    for D, Dv in ((16, 32), (64, 128), (40, 24)):
        check_both(Case(2, dtype, B, Lq, Lk, H, Hkv, D, Dv, causal=causal, seed=D, q_start=[max(0, Lk - Lq)] * B if causal else None))


@gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_gradients_lengths_and_starts(maps, dtype):
    for causal in (False, True):
        for Lq in (3, 150):
            c = Case(maps, dtype, 6, Lq, 200, 4, 2, 32, causal=causal, kv_len=[0, 1, 200, 77, 128, 500], seed=Lq,
                     q_len=[Lq, Lq, 0, max(1, Lq // 2), Lq, Lq + 9], q_start=[0, 0, 3, 76, -5, 2 ** 30 + 5])
            want_out, want = both_ways(c)
            for b in range(6):                                       # what lies behind the lengths takes no part
                for t in (c.k, c.v):
                    t[b, min(200, c.lens["kv_len"][b]):] = math.nan
                for t in (c.q, c.dout):
                    t[b, min(Lq, c.lens["q_len"][b]):] = math.nan
            out, got = check_both(c)
            assert torch.equal(out, want_out) and all(torch.equal(x, y) for x, y in zip(got, want))
            # gradients into the caller's tensors: rows behind the lengths stay as they are
            mine = [torch.full_like(x, 3.0) for x in got]
            names = ("dq", "dk", "dv", "dtable" if maps == 1 else "dlam")
            _, into = both_ways(c, **dict(zip(names, mine)))
            for name, x, y, n in zip(names, into, got, (c.parts["nq"], c.parts["nk"], c.parts["nk"], None)):
                if n is None:
                    assert torch.equal(x, y)
                    continue
                keep = (torch.arange(x.shape[1])[None] < n[:, None]).cuda()
                assert torch.equal(x[keep], y[keep]) and bool((x[~keep] == 3.0).all()), name


@gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("size", [1e-5, 1e4])
def test_half_gradients_of_any_magnitude(maps, size):
    """dO far from one: IEEE half keeps its relative accuracy (dV's operand is dO itself)."""
    check_both(Case(maps, torch.float16, 1, 200, 300, 2, 1, 32, seed=3, dout_scale=size))


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_rel_gradients_table_infinities_and_lowest_values(dtype):
    for causal in (False, True):
        for value in (-math.inf, torch.finfo(dtype).min):
            c = Case(1, dtype, 1, 200, 300, 2, 2, 32, causal=causal, q_start=[100] if causal else None)
            c.w[::2] = value
            check_both(c)
        c.w[:] = torch.finfo(dtype).min                              # equal weights everywhere
        check_both(c)


@gpu
@pytest.mark.parametrize("buckets,far", [(2, 2), (16, 64), (64, 1024), (128, 100)])
def test_rel_gradients_bucket_tables(buckets, far):
    for causal in (False, True):
        if not causal and buckets == 2:
            continue
        check_both(Case(1, torch.bfloat16, 2, 140, 260, 2, 1, 32, causal=causal, buckets=buckets, far=far, q_start=[120, 7] if causal else None))


@gpu
@pytest.mark.parametrize("maps", [1, 2])
def test_gradients_against_differences(maps):
    """Central differences of the 64-bit formula along random directions."""
    c = Case(maps, torch.float32, 2, 9, 40, 2, 1, 16, causal=True, q_start=[31, 20], kv_len=[40, 25], seed=4)
    r, want = gradients(c)
    _, got = both_ways(c)
    g = torch.Generator().manual_seed(1)
    h = 1e-4
    for name, at in (("dq", "q"), ("dk", "k"), ("dv", "v"), ("dw", "w")):
        base = getattr(c, at)
        d = torch.randn(base.shape, generator=g, dtype=torch.float64)
        side = []
        for sign in (1, -1):
            setattr(c, at, base.double() + sign * h * d)
            side.append((c.reference()["out"] * c.dout.double()).sum())
        setattr(c, at, base)
        slope = float((side[0] - side[1]) / (2 * h))
        mine = got[("dq", "dk", "dv", "dw").index(name)].double().cpu()
        rest = float((want[name][1] * d.abs()).sum()) + 1e-5 * float((mine * d).abs().sum())       # the bound; h^2 of the third derivative
        assert abs(slope - float((mine * d).sum())) <= rest, (name, slope, float((mine * d).sum()), rest)


@gpu
@pytest.mark.parametrize("maps", [1, 2])
def test_gradients_repeat_and_replay(maps):
    """The same inputs give the same bits, eager, on another stream, and from a graph replayed between eager work."""
    c = Case(maps, torch.bfloat16, 2, 300, 300, 4, 2, 64, causal=True, seed=8)
    want_out, want = both_ways(c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again_out, again = both_ways(c)
    s.synchronize()
    assert torch.equal(again_out, want_out) and all(torch.equal(x, y) for x, y in zip(again, want))
    t = [x.cuda() for x in (c.q, c.k, c.v, c.w)]
    do, kw = c.dout.cuda(), c.kwargs("cuda")
    fwd, bwd = ((ops_attn.rel_attention, ops_attn.rel_attention_bwd) if maps == 1 else (ops_attn.diff_attention, ops_attn.diff_attention_bwd))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, saved = fwd(*t, **kw, save=True)
        grads = bwd(do, *t, out, saved, **kw)
    for n in range(3):
        t[0].copy_(c.q * (1 + n))
        o, sv = fwd(*t, **kw, save=True)
        fresh = bwd(do, *t, o, sv, **kw)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, out) and all(torch.equal(x, y) for x, y in zip(fresh, grads))


def test_backward_refuses():
    z = _cpu()
    out = torch.zeros(2, 5, 4, 16, dtype=torch.bfloat16)
    with pytest.raises(SgtaHipError, match="GPU"):
        ops_attn.rel_attention_bwd(out, *z, out, (torch.zeros(1, 2, 4, 5, 2), None))
    import ctypes
    from sgtapose_amd import _lib
    lib = _lib.load()
    ok = dict(q=64, k=64, v=64, w=64, out=64, lut=64, B=1, Lq=4, Lk=4, H=2, Hkv=2, D=16, Dv=16, dtype=2, reach=8, num_buckets=8, scale=0.25,
              dout=64, dq=64, dk=64, dv=64, dw=64, stats=64, ws=64, ws_floats=1 << 20)
    for change in (dict(dout=None), dict(dq=None), dict(dw=None), dict(stats=None), dict(ws=None), dict(ws_floats=3), dict(dk=65), dict(D=12),
                   dict(sdv=(ctypes.c_long * 4)(16, 4, 16, 0))):
        a = _lib.AttnArgs(**{**ok, **change})
        assert lib.sgta_rel_attn_bwd(ctypes.byref(a), None) < 0, change
    assert lib.sgta_diff_attn_bwd(ctypes.byref(_lib.AttnArgs(**ok)), None) < 0      # no second map's product


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_widest_tables_and_heads(dtype):
    """The largest tables with the largest heads: what a work-group keeps still fits it."""
    for buckets, far in ((256, 1024), (64, 300)):
        check_both(Case(1, dtype, 1, 150, 200, 2, 1, 128, buckets=buckets, far=far, seed=5))
        check_both(Case(1, dtype, 1, 70, 180, 8, 1, 128, causal=True, buckets=buckets, far=far, q_start=[110], seed=6))
        check_forward(Case(1, dtype, 1, 1, 700, 16, 1, 128, causal=True, buckets=buckets, far=far, q_start=[699], seed=7))


@gpu
def test_first_call_with_a_table_is_not_captured():
    c = Case(1, torch.bfloat16, 1, 40, 50, 2, 2, 32, buckets=24, far=77)
    t = [x.cuda() for x in (c.q, c.k, c.v, c.w)]
    out = torch.empty_like(t[0])
    with pytest.raises(SgtaHipError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops_attn.rel_attention(*t, out, **c.kwargs("cpu"))
    want = ops_attn.rel_attention(*t, **c.kwargs("cpu"))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops_attn.rel_attention(*t, out, **c.kwargs("cpu"))
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@gpu
def test_saved_must_fit():
    c = Case(2, torch.bfloat16, 1, 20, 30, 2, 2, 32)
    t = [x.cuda() for x in (c.q, c.k, c.v, c.w)]
    out, (stats, out2) = ops_attn.diff_attention(*t, save=True)
    for saved in ((stats, None), (stats, out2.float()), (stats[:, :, :1], out2)):
        with pytest.raises(SgtaHipError, match="saved"):
            ops_attn.diff_attention_bwd(c.dout.cuda(), *t, out, saved)


@gpu
def test_positions_too_far_apart_are_refused():
    """Two rows of a tensor of 2^24 + 16 bytes a position (an untouched allocation; nothing is launched)."""
    wide = torch.empty(2, (1 << 23) + 8, dtype=torch.bfloat16, device="cuda")
    far = wide[:, :64].view(1, 2, 2, 32)
    near = torch.zeros(1, 2, 2, 32, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(32, 2, dtype=torch.bfloat16, device="cuda")
    for args in ((far, near, near), (near, far, near), (near, near, far)):
        with pytest.raises(SgtaHipError, match="bytes apart"):
            ops_attn.rel_attention(*args, table)


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_keys_beyond_the_reach_in_a_tile_that_is_not(dtype):
    """Few keys, all farther from the query than any bucket of its own, in a tile whose empty rest is nearer.  Calls with another table,
    whose values are large, come between, so that nothing left in LDS by an equal one helps."""
    other = Case(1, dtype, 8, 1, 40, 64, 8, 32, buckets=4, far=3, q_start=[20] * 8)
    other.w[:] = 100.0 * (1 + torch.arange(4)[:, None])
    for n, (Lq, kv_len, q_start) in enumerate([(1, 13, 30), (1, 1, 17), (2, 1, 9), (5, 1, 5), (1, 33, 50), (23, 1, 20), (2, 31, 36), (1, 130, 150)]):
        for causal in (False, True):
            forward(other)
            check_both(Case(1, dtype, 3, Lq, max(71, kv_len), 3, 3, 32, causal=causal, buckets=4, far=3, kv_len=[kv_len] * 3,
                            q_start=[q_start] * 3, seed=n))
