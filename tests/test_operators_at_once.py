"""The attention and 8-bit operators several at a time: calls on two streams, and two captured graphs replayed at once between eager work,
against the same calls one after another.  Workspaces are each call's own."""
import pytest
import torch

from sgtapose_amd import ops_attn, ops_i8
from test_attention import Case

gpu = pytest.mark.gpu


class Work:
    """One sample of everything: both attentions there and back, many keys split over the grid, the 8-bit pair."""

    def __init__(self, dtype, seed):
        self.cases = [Case(1, dtype, 2, 200, 300, 4, 2, 64, causal=True, q_start=[100, 0], kv_len=[300, 170], seed=seed),
                      Case(2, dtype, 2, 130, 200, 4, 2, 64, 128, q_len=[130, 60], seed=seed + 1)]
        self.step = Case(1, dtype, 2, 1, 3000, 4, 2, 64, causal=True, q_start=[2999, 1400], seed=seed + 2)
        g = torch.Generator().manual_seed(seed)
        self.x, self.w = (torch.randn(n, 320, generator=g).to(dtype).cuda() for n in (70, 96))
        self.t = [[x.cuda() for x in (c.q, c.k, c.v, c.w, c.dout)] for c in (*self.cases, self.step)]
        self.kw = [c.kwargs("cuda") for c in (*self.cases, self.step)]

    def run(self):
        out = []
        for (fwd, bwd), (*t, do), kw in zip(((ops_attn.rel_attention, ops_attn.rel_attention_bwd), (ops_attn.diff_attention, ops_attn.diff_attention_bwd)),
                                            self.t, self.kw):
            o, saved = fwd(*t, **kw, save=True)
            out += [o, *bwd(do, *t, o, saved, **kw)]
        out.append(ops_attn.rel_attention(*self.t[2][:4], **self.kw[2]))
        out.append(ops_i8.linear_i8(*ops_i8.quantize_rows(self.x), *ops_i8.quantize_rows(self.w)))
        return out


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
def test_two_streams_and_two_graphs(dtype):
    works = [Work(dtype, 3), Work(dtype, 40)]
    want = [[t.clone() for t in w.run()] for w in works]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in works]
    for _ in range(4):
        got = []
        for w, s in zip(works, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append([w.run() for _ in range(3)][-1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, v in zip(got, want) for a, b in zip(g, v))
    graphs, outs = [], []
    for w in works:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(w.run())
        graphs.append(g)
    for _ in range(4):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = works[0].run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o, v in zip(outs, want) for a, b in zip(o, v))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[0]))
