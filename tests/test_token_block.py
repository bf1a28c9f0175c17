"""Blocks of a token model as a user puts them together: 8-bit projections around attention with a cache, and a training step through
both kinds of attention.  Every stage is held to its own bound against the formula in 64 bits, on the inputs that the stage before
gave it (strided slices of a fused projection, a cache that is filled as it goes, a gradient that another kernel wrote).
"""
import pytest
import torch

from sgtapose_amd import ops_attn, ops_i8
from test_attention import ALL, FLUSH, NAMES, Case, gradients, within

gpu = pytest.mark.gpu
U = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def linear_bound(xq, xs, wq, ws, bias, relu, dtype):
    """-> value and bound of linear_i8: four roundings in f32 of the scaled sum and the bias, then the type's (u of the value; a half
    below 2^-14 has steps of 2^-24 whatever its size, so up to 2^-25 there)."""
    s = (xq.double() @ wq.double().t()) * (xs.double()[:, None] * ws.double())
    want = s + bias.double()
    tol = 4 * 2.0 ** -24 * (s.abs() + bias.double().abs()) + 1e-30
    want = want.clamp(min=0) if relu else want
    return want, tol + U[dtype] * (want.abs() + tol) + FLUSH[dtype]


class Block:
    """Self-attention with a cache and a feed-forward pair, weights in 8 bits."""

    def __init__(self, dtype, B, C, H, Hkv, D, room, hidden):
        g = torch.Generator().manual_seed(11)
        self.dtype, self.dims, self.room = dtype, (B, H, Hkv, D), room
        self.split = (H * D, Hkv * D, Hkv * D)

        def weight(n, k):
            w = (torch.randn(n, k, generator=g) * k ** -0.5).to(dtype).cuda()
            return (*ops_i8.quantize_rows(w), (0.1 * torch.randn(n, generator=g)).to(dtype).cuda())
        self.qkv, self.proj, self.up, self.down = weight(sum(self.split), C), weight(C, H * D), weight(hidden, C), weight(C, hidden)
        self.table = torch.randn(32, H, generator=g).to(dtype).cuda()
        self.kc, self.vc = (torch.zeros(B, room, Hkv, D, dtype=dtype, device="cuda") for _ in range(2))
        self.seen = []                                  # every stage's inputs and output

    def linear(self, x, w, relu=False):
        xq, xs = ops_i8.quantize_rows(x)
        y = ops_i8.linear_i8(xq, xs, *w[:2], w[2], relu=relu)
        self.seen.append(("linear", (xq, xs, *w, relu), y))
        return y

    def __call__(self, x, start, length):
        """x [B, L, C]: L new tokens a sequence at positions start[b] ...; length[b]: tokens in the cache with them."""
        B, H, Hkv, D = self.dims
        L, C = x.shape[1:]
        q, k, v = self.linear(x.view(B * L, C), self.qkv).view(B, L, -1).split(self.split, 2)
        q, k, v = q.view(B, L, H, D), k.view(B, L, Hkv, D), v.view(B, L, Hkv, D)      # slices: rows of the fused projection
        at = (start[:, None].long() + torch.arange(L, device=x.device)).clamp(max=self.room - 1)
        row = torch.arange(B, device=x.device)[:, None]
        self.kc[row, at], self.vc[row, at] = k, v
        o = ops_attn.rel_attention(q, self.kc, self.vc, self.table, causal=True, bidirectional=False, q_start=start, kv_len=length)
        self.seen.append(("attention", (q, self.kc.clone(), self.vc.clone(), start, length), o))
        x = x + self.linear(o.view(B * L, H * D), self.proj).view(B, L, C)
        y = self.linear(self.linear(x.view(B * L, C), self.up, relu=True), self.down)
        return x + y.view(B, L, C)

    def check(self):
        B, H, Hkv, D = self.dims
        for kind, args, got in self.seen:
            if kind == "linear":
                xq, xs, wq, ws, bias = (t.cpu() for t in args[:5])
                within(kind, got, *linear_bound(xq, xs, wq, ws, bias, args[5], self.dtype))
            else:
                q, k, v, start, length = (t.cpu() for t in args)
                c = Case(1, self.dtype, B, q.shape[1], self.room, H, Hkv, D, causal=True, buckets=32, far=128, q_start=start.tolist(),
                         kv_len=length.tolist())
                c.q, c.k, c.v, c.w = q, k, v, self.table.cpu()
                r = c.reference()
                within(kind, got, r["out"], r["out_tol"])
        self.seen.clear()


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_prompt_then_single_tokens(dtype):
    """A prompt of uneven lengths, then tokens one at a time, the last ones from a captured graph."""
    B, C = 3, 96
    block = Block(dtype, B, C, 4, 2, 24, room=300, hidden=200)
    g = torch.Generator().manual_seed(1)
    new = lambda L: torch.randn(B, L, C, generator=g).to(dtype).cuda()                            # noqa: E731
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")                           # noqa: E731
    x = new(270)
    y = block(x, ints(0, 0, 0), ints(270, 41, 1))      # the second and third prompts are shorter: what follows them is overwritten
    assert bool(torch.isfinite(y).all())
    block.check()
    start = ints(270, 41, 1)
    for _ in range(3):
        block(new(1), start, start + 1)
        block.check()
        start += 1
    x, length = new(1), start + 1
    out = torch.empty(B, 1, C, dtype=dtype, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out.copy_(block(x, start, length))
    block.seen.clear()
    for _ in range(3):
        x.copy_(new(1))
        kept = block.kc.clone(), block.vc.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        block.kc.copy_(kept[0])
        block.vc.copy_(kept[1])
        assert torch.equal(block(x, start, length), got)
        block.check()
        start += 1
        length += 1


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_training_step_through_both(dtype):
    """rel_attention's output is diff_attention's v; gradients go back through both, the first ones' into slices of one tensor."""
    B, L, H, D = 2, 150, 4, 32
    one = Case(1, dtype, B, L, L, H, H, D, causal=True, seed=2, kv_len=[L, 90])
    two = Case(2, dtype, B, L, L, H, H, D, D, causal=True, seed=3, kv_len=[L, 90])
    q, k, v, table = (t.cuda() for t in (one.q, one.k, one.v, one.w))
    q2, k2, lam, dout = (t.cuda() for t in (two.q, two.k, two.w, two.dout))
    kw1, kw2 = one.kwargs("cuda"), two.kwargs("cuda")
    dqkv = torch.zeros(B, L, 3, H, D, dtype=dtype, device="cuda")

    def step():
        o1, saved1 = ops_attn.rel_attention(q, k, v, table, **kw1, save=True)
        o2, saved2 = ops_attn.diff_attention(q2, k2, o1, lam, **kw2, save=True)
        g2 = ops_attn.diff_attention_bwd(dout, q2, k2, o1, lam, o2, saved2, **kw2)
        g1 = ops_attn.rel_attention_bwd(g2[2], q, k, v, table, o1, saved1, dqkv[:, :, 0], dqkv[:, :, 1], dqkv[:, :, 2], **kw1)
        return o1, o2, g1, g2
    o1, o2, g1, g2 = step()
    torch.cuda.synchronize()
    two.v, one.dout = o1.cpu(), g2[2].cpu()
    for c, out, got in ((one, o1, g1), (two, o2, g2)):
        r, want = gradients(c)
        within("out", out, r["out"], r["out_tol"])
        for name, t in zip(("dq", "dk", "dv", "dw"), got):
            within(name, t, *want[name], r["nk"] if name in ("dk", "dv") else None)
    assert bool((dqkv[1, 90:, 1:] == 0).all())
    want = [t.clone() for t in (*g1, *g2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o1, o2, g1, g2 = step()
    for _ in range(3):
        dqkv.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*g1, *g2), want))
