"""The attention operators record nothing for autograd: a call that would lose a gradient without a word is refused, and the documented
way, ``save=True`` with the backward operator inside an autograd.Function, gives the gradients of the formula."""
import pytest
import torch

from sgtapose_amd import ops_attn
from sgtapose_amd._lib import SgtaHipError
from test_attention import Case, gradients, within

gpu = pytest.mark.gpu
CALLS = [(1, ops_attn.rel_attention), (2, ops_attn.diff_attention)]


def operands(maps):
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)                                          # noqa: E731
    mp = (2,) if maps == 2 else ()
    return [z(2, 5, 4, *mp, 16), z(2, 7, 2, *mp, 16), z(2, 7, 2, 16), z(32, 4) if maps == 1 else z(4, 16)]


@pytest.mark.parametrize("maps,call", CALLS, ids=["rel", "diff"])
def test_refuses_to_lose_a_gradient(maps, call):
    for n in range(4):
        t = operands(maps)
        t[n].requires_grad_()
        with pytest.raises(SgtaHipError, match="no_grad"):
            call(*t)
        with torch.no_grad(), pytest.raises(SgtaHipError, match="on the GPU"):                    # past that check
            call(*t)
        with pytest.raises(SgtaHipError, match="on the GPU"):
            call(*t, save=True)


class Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, maps, kw, q, k, v, w):
        out, saved = CALLS[maps - 1][1](q, k, v, w, **kw, save=True)
        ctx.save_for_backward(q, k, v, w, out, *saved)
        ctx.maps, ctx.kw = maps, kw
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, w, out, stats, out2 = ctx.saved_tensors
        bwd = ops_attn.rel_attention_bwd if ctx.maps == 1 else ops_attn.diff_attention_bwd
        return None, None, *bwd(dout.contiguous(), q, k, v, w, out, (stats, out2), **ctx.kw)


@gpu
@pytest.mark.parametrize("maps", [1, 2])
def test_inside_a_function(maps):
    """One key / value sequence for both samples (its gradient is the sum of theirs), the sum of the outputs as the loss: its gradient
    comes expanded from one number."""
    c = Case(maps, torch.float32, 2, 40, 50, 4, 2, 32, causal=True, q_start=[10, 3], seed=6)
    c.k[1], c.v[1], c.dout[:] = c.k[0], c.v[0], 1.0
    _, want = gradients(c)
    leaf = [t.cuda().requires_grad_() for t in (c.q, c.k[:1].contiguous(), c.v[:1].contiguous(), c.w)]
    q, k, v, w = leaf
    out = Attention.apply(maps, c.kwargs("cuda"), q, k.expand(2, *k.shape[1:]), v.expand(2, *v.shape[1:]), w)
    out.sum().backward()
    within("dq", q.grad, *want["dq"])
    within("dw", w.grad, *want["dw"])
    for name, t in (("dk", k), ("dv", v)):
        value, bound = (x.sum(0, keepdim=True) for x in want[name])
        within(name, t.grad, value, bound + 2.0 ** -24 * value.abs())                             # and the sum of the two
