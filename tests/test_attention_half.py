"""IEEE half gradients whose values are far from one: what is formed on the way, P (dO V^T - delta), may lie beyond the half range where every
operand and every result lies in it.  Bounds as in test_attention.py."""
import pytest
import torch

from test_attention import Case, check_both

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("size,dout", [(2e3, 1e-1), (5e3, 1e-3), (1e-3, 1.0), (1e-3, 1e3)])
def test_values_of_any_magnitude(maps, size, dout):
    for D, Dv in ((16, 16), (64, 64 if maps == 1 else 128)):
        for Lq, Lk in ((40, 60), (200, 300)):
            c = Case(maps, torch.float16, 2, Lq, Lk, 4, 2, D, Dv, causal=Lk == 300, q_start=[100, 0] if Lk == 300 else None, seed=D, dout_scale=dout)
            c.v = (c.v.float().clamp(-4, 4) * size).half()
            check_both(c)


@gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("size", [500.0, 4e3, 2.5e4])
def test_gradients_along_the_values(maps, size):
    """dO in the direction of some keys' values, every element of the same size: dO V^T is Dv |dO||v|, far beyond a half where |dO| is brought
    next to one, while out (at most 2.2 |v|), dQ and dK are halves."""
    for Lq, Lk, D in ((40, 6, 64), (200, 300, 64), (3, 40, 64)):
        c = Case(maps, torch.float16, 2, Lq, Lk, 4, 2, D, 64 if maps == 1 else 128, seed=9)
        way = torch.randn(c.v.shape[-1], generator=torch.Generator().manual_seed(2)).sign()
        c.v[:] = (size * way * torch.where(torch.arange(Lk) % 3 == 0, 1.0, -0.5)[None, :, None, None]).half()
        c.v += (0.01 * size * torch.randn(c.v.shape, generator=torch.Generator().manual_seed(3))).half()
        c.dout[:] = (1e-3 * way).half()
        check_both(c)


@gpu
@pytest.mark.parametrize("maps", [1, 2])
def test_few_large_values(maps):
    """Most keys have values near one, a few have large ones: those tiles must not cost the others their accuracy."""
    for Lq, Lk in ((40, 90), (200, 300)):
        c = Case(maps, torch.float16, 2, Lq, Lk, 4, 2, 64, 64, seed=7, dout_scale=1e-2)
        c.v[:, 70] = 3e4 * c.v[:, 70].sign()
        c.v[:, 3] = -2e4 * c.v[:, 3].sign()
        check_both(c)


@gpu
@pytest.mark.parametrize("Lq,Lk,Hkv,D", [(8, 130, 2, 64), (1, 63, 8, 24), (64, 200, 2, 96)])
def test_small_weights_beside_large_values(Lq, Lk, Hkv, D):
    """Values of some thousand alone leave the scale where it is: keys of small weights keep what |dO| next to one gives them."""
    for seed in range(4):
        c = Case(1, torch.float16, 2, Lq, Lk, 4 if Hkv == 2 else 8, Hkv, D, buckets=16, far=40, seed=seed)
        c.w = (c.w.float() * 30).half()
        c.v = (c.v.float() * 3000).half()
        check_both(c)
