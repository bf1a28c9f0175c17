"""float32 products as three bfloat16 numbers an operand, at operands for which what is left out is largest: x = 2^n (1 + 2^-7 - 2^-23) has
parts 1, 2^-7 - 2^-15 and 2^-15 - 2^-23 (times 2^n), and the products mid lo + lo mid + lo lo are 7.9 * 2^-24 of x y.

test_attention.py counts 3 e for what is left out, e = 2^-24; 8 e at the most instead adds 5 to its constants, the least of which is Dv + 5
= 13 here (D + 6, Lk + 3 and Lq G + 3 are larger): 18 / 13 < 1.4 times its bounds.
"""
import pytest
import torch

from test_attention import Case, both_ways, gradients, within

gpu = pytest.mark.gpu


def parts(x):
    out = []
    for _ in range(3):
        p = (x.view(torch.int32) & -65536).view(torch.float32)          # the upper half
        out.append(p)
        x = x - p
    assert bool((x == 0).all())
    return [p.double() for p in out]


def test_what_is_left_out():
    x = torch.tensor([1 + 2.0 ** -7 - 2.0 ** -23])
    hi, mid, lo = parts(x)
    left = float((2 * mid * lo + lo * lo) / (x.double() * x.double()))
    assert 7.8 * 2.0 ** -24 < left < 8 * 2.0 ** -24
    g = torch.Generator().manual_seed(1)
    x, y = torch.randn(100000, generator=g), torch.randn(100000, generator=g)
    (_, m1, l1), (_, m2, l2) = parts(x), parts(y)
    left = (m1 * l2 + l1 * m2 + l1 * l2) / (x.double() * y.double())
    assert float(left.min()) >= 0 and float(left.max()) < 8 * 2.0 ** -24 and float(left.mean()) < 2.1 * 2.0 ** -24


@gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("same_sign", [True, False])
def test_largest_rest(maps, same_sign):
    for Lq, Lk, D, Dv in ((40, 70, 8, 8), (150, 130, 32, 32), (33, 90, 64, 64), (2, 60, 16, 16)):
        c = Case(maps, torch.float32, 2, Lq, Lk, 4, 2, D, Dv, seed=D)
        for t in (c.q, c.k, c.v, c.dout):
            sign = 1.0 if same_sign else t.sign()
            t.copy_(sign * (1 + 2.0 ** -7 - 2.0 ** -23) * 2.0 ** t.abs().log2().round().clamp(-2, 1))
        r, want = gradients(c)
        out, got = both_ways(c)
        within("out", out, r["out"], 1.4 * r["out_tol"])
        for name, t in zip(("dq", "dk", "dv", "dw"), got):
            within(name, t, want[name][0], 1.4 * want[name][1])


@gpu
def test_floats_next_to_the_largest():
    """A split to the nearest would make infinities of them, and not-a-numbers where a mask weighs them with zero.  (Forward: dO V^T of such
    values is itself infinite, which the documentation lets through a mask, 0 times infinity.  The gradients take 1e30.)"""
    c = Case(1, torch.float32, 1, 40, 70, 2, 2, 16, causal=True, q_start=[0], seed=3)
    want_out, want = both_ways(c)
    for size in (torch.finfo(torch.float32).max, 1e30):
        c.v[:, 40:] = size                               # no query sees them
        c.k[:, 50:] = -size
        out, got = both_ways(c)
        assert torch.equal(out, want_out)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
