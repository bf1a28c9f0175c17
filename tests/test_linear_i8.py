"""Quantisation of rows and 8-bit token products (sgtapose_amd/ops_i8.py): whole numbers exactly, the epilogue to its roundings.

out = fl(fl(sum) fl(xs ws) (+ bias)) in f32, then the type's rounding: each f32 operation is off by 2^-24 of its result, so
|out - exact| <= (4 * 2^-24)(|sum xs ws| + |bias|) + u |out|, u = eps / 2 of the output type (0 for f32, counted in the 4).
"""
import pytest
import torch

from sgtapose_amd import ops_i8
from sgtapose_amd._lib import SgtaHipError

gpu = pytest.mark.gpu
U = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
ALL = [torch.float32, torch.float16, torch.bfloat16]
IDS = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}


def quant_ref(x):
    """Scales in f32, bytes from the quotient in 64 bits."""
    top = x.float().abs().amax(1)
    xs = (top / 127).float()
    q = torch.where(xs[:, None] > 0, (x.double() / xs.double()[:, None]).round(), 0.0)
    return q.clamp(-127, 127).to(torch.int8), xs


def check_linear(M, N, K, dtype, relu, with_bias, seed=0, pad_x=0, pad_w=0, shift=0):
    g = torch.Generator().manual_seed(seed)
    xq = torch.randint(-128, 128, (M, K + pad_x), generator=g, dtype=torch.int8)[:, :K]
    wq = torch.randint(-128, 128, (N, K + pad_w), generator=g, dtype=torch.int8)[:, :K]
    xs, ws = torch.rand(M, generator=g) + 0.01, (torch.rand(N, generator=g) + 0.01) * 1e-3
    bias = torch.randn(N, generator=g).to(dtype) if with_bias else None
    s = (xq.double() @ wq.double().t()) * (xs.double()[:, None] * ws.double())
    want = s + (bias.double() if with_bias else 0.0)
    tol = 4 * 2.0 ** -24 * (s.abs() + (bias.double().abs() if with_bias else 0.0)) + 1e-30
    if relu:
        want = want.clamp(min=0)
    tol = tol + U[dtype] * (want.abs() + tol)

    def dev(t, pad):                                    # the same strides, and ``shift`` bytes off a 16-byte border
        whole = torch.zeros(t.shape[0] * (t.shape[1] + pad) + shift, dtype=torch.int8, device="cuda")[shift:].view(t.shape[0], -1)
        whole[:, :t.shape[1]] = t.cuda()
        return whole[:, :t.shape[1]]
    out = torch.full((M, N + 3), 9.0, dtype=dtype, device="cuda")
    ops_i8.linear_i8(dev(xq, pad_x), xs.cuda(), dev(wq, pad_w), ws.cuda(), None if bias is None else bias.cuda(), out[:, :N], relu=relu)
    d = (out[:, :N].double().cpu() - want).abs()
    assert bool((d <= tol).all()), (M, N, K, float((d - tol).max()))
    assert bool((out[:, N:] == 9).all())
    plain = ops_i8.linear_i8(dev(xq, pad_x), xs.cuda(), dev(wq, pad_w), ws.cuda(), None if bias is None else bias.cuda(), relu=relu, dtype=dtype)
    assert torch.equal(plain, out[:, :N])


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=IDS.get)
@pytest.mark.parametrize("M", [1, 2, 16, 17, 33, 64, 65, 130, 300])
def test_linear_sizes(dtype, M):
    for N, K in ((1, 1), (16, 64), (37, 80), (65, 144), (130, 1040), (256, 4096)):
        check_linear(M, N, K, dtype, relu=M % 2 == 0, with_bias=N % 2 == 1, seed=M + N)


@gpu
@pytest.mark.parametrize("M", [1, 40, 70, 200])
def test_linear_any_alignment(M):
    for N, K, pad_x, pad_w, shift in ((33, 15, 0, 0, 0), (33, 17, 0, 0, 1), (50, 129, 3, 0, 5), (64, 255, 1, 17, 0), (64, 256, 0, 3, 8), (20, 1000, 0, 0, 0)):
        check_linear(M, N, K, torch.bfloat16, False, True, pad_x=pad_x, pad_w=pad_w, shift=shift)


@gpu
@pytest.mark.parametrize("M,N,K", [(3600, 3500, 200), (3600, 3500, 129), (1700, 1800, 4096), (1700, 1801, 640), (4096, 4096, 128)])
def test_linear_every_tile(M, N, K):
    """Sizes that take the largest tile, the middle one and the smallest, aligned and not; on the GPU in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(1)
    xq = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8, device="cuda")
    wq = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8, device="cuda")
    xs, ws = torch.ones(M, device="cuda"), torch.ones(N, device="cuda")
    got = ops_i8.linear_i8(xq, xs, wq, ws)
    assert torch.equal(got, (xq.double() @ wq.double().t()).float())


@gpu
def test_longest_sum_is_exact():
    K = ops_i8.MAX_K
    for M in (1, 70):
        xq, wq = (torch.full((n, K), -128, dtype=torch.int8, device="cuda") for n in (M, 5))
        got = ops_i8.linear_i8(xq, torch.ones(M, device="cuda"), wq, torch.ones(5, device="cuda"))
        assert bool((got.double() == torch.tensor(float(128 * 128 * K)).float().double().cuda()).all())


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=IDS.get)
def test_quantize_rows(dtype):
    for M, K in ((1, 1), (3, 7), (5, 64), (130, 343), (4, 4096), (3, 8200), (2, 20001), (4097, 40), (4100, 4105)):
        g = torch.Generator().manual_seed(K)
        x = (torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g) * 4)).to(dtype)
        if M > 2:
            x[0] = 0
        q, s = quant_ref(x)
        xq, xs = ops_i8.quantize_rows(x.cuda())
        assert torch.equal(xq.cpu(), q) and torch.equal(xs.cpu(), s)
        wide = torch.zeros(M, K + 5, dtype=dtype, device="cuda")[:, 3:K + 3]              # rows off a 16-byte border
        wide.copy_(x)
        into = torch.full((M, K + 9), 77, dtype=torch.int8, device="cuda")
        ops_i8.quantize_rows(wide, into[:, 1:K + 1])
        assert torch.equal(into[:, 1:K + 1].cpu(), q) and bool((into[:, 0] == 77).all()) and bool((into[:, K + 1:] == 77).all())


@gpu
def test_quantize_next_to_a_half():
    """Quotients at and next to k + 1/2, where a quotient rounded in f32 would fall to the other side."""
    xs = torch.rand(200, generator=torch.Generator().manual_seed(3)) + 0.5
    half = (torch.arange(-126, 126) + 0.5)
    x = (xs[:, None] * half).float()
    x = torch.cat([x, x.nextafter(torch.tensor(9e9)), x.nextafter(torch.tensor(-9e9)), (xs * 127)[:, None]], 1)
    q, s = quant_ref(x)
    xq, got = ops_i8.quantize_rows(x.cuda())
    assert torch.equal(got.cpu(), s) and torch.equal(xq.cpu(), q)


@gpu
def test_quantize_extremes():
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[1e-45, 3e-45, -1.4e-43, 0.0], [3e38, -3e38, 1.0, 0.0], [inf, 1.0, -2.0, 0.0], [nan, 1.0, 2.0, 3.0], [0.0, -0.0, 0.0, 0.0],
                      [1e-38, -1e-38, 5e-39, 1e-40]])
    xq, xs = ops_i8.quantize_rows(x.cuda())
    q, s = quant_ref(x[[0, 1, 4, 5]])
    assert torch.equal(xs.cpu()[[0, 1, 4, 5]], s) and torch.equal(xq.cpu()[[0, 1, 4, 5]], q)
    assert xs[2] == inf and bool(xs[3].isnan())
    wq, ws = ops_i8.quantize_rows(torch.eye(4, device="cuda"))
    y = ops_i8.linear_i8(xq, xs, wq, ws)
    assert not bool(y[2:4].isfinite().any()) and bool((y[4] == 0).all())


@gpu
def test_graph_replays():
    x, w = torch.randn(70, 320, device="cuda").half(), torch.randn(96, 320, device="cuda").half()
    wq, ws = ops_i8.quantize_rows(w)
    out, xq, xs = torch.empty(70, 96, device="cuda").half(), torch.empty(70, 320, dtype=torch.int8, device="cuda"), torch.empty(70, device="cuda")
    ops_i8.linear_i8(*ops_i8.quantize_rows(x, xq, xs), wq, ws, None, out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops_i8.linear_i8(*ops_i8.quantize_rows(x, xq, xs), wq, ws, None, out)
    for n in range(3):
        x.copy_(torch.randn(70, 320))
        want = ops_i8.linear_i8(*ops_i8.quantize_rows(x), wq, ws, dtype=torch.float16)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals():
    i8 = lambda *s: torch.zeros(*s, dtype=torch.int8)                                             # noqa: E731
    x, xs, w, ws = i8(3, 32), torch.zeros(3), i8(5, 32), torch.zeros(5)
    ok = dict(xq=x, xs=xs, wq=w, ws=ws)
    with pytest.raises(SgtaHipError, match="GPU"):
        ops_i8.linear_i8(**ok)
    for change in (dict(xq=x.float()), dict(wq=i8(5, 31)), dict(xs=torch.zeros(4)), dict(ws=ws.double()), dict(bias=torch.zeros(4)),
                   dict(bias=ws.half(), dtype=torch.float32), dict(out=torch.zeros(3, 6)), dict(dtype=torch.float64), dict(xq=i8(0, 32), xs=torch.zeros(0)),
                   dict(xq=i8(32, 3).t()), dict(xq=i8(1, 32).expand(3, 32)), dict(xq=i8(3, 131072), wq=i8(5, 131072))):
        with pytest.raises(SgtaHipError):
            ops_i8.linear_i8(**{**ok, **change})
    with pytest.raises(SgtaHipError, match="GPU"):
        ops_i8.quantize_rows(torch.zeros(3, 4))
    for bad in (torch.zeros(3), torch.zeros(3, 4).double(), torch.zeros(4, 3).t(), torch.zeros(0, 4)):
        with pytest.raises(SgtaHipError):
            ops_i8.quantize_rows(bad)
    with pytest.raises(SgtaHipError):
        ops_i8.quantize_rows(torch.zeros(3, 4), i8(3, 5))


def test_c_entries_refuse_before_they_launch():
    from sgtapose_amd import _lib
    lib = _lib.load()
    ok = [64, 32, 64, 64, 32, 64, None, 64, 8, 4, 8, 32, 0, 0, None]
    for at, v in ((0, None), (1, 31), (3, None), (4, 16), (7, None), (8, 7), (9, 0), (10, 0), (11, 0), (13, 3), (7, 65), (1, (1 << 22) + 1)):
        a = list(ok)
        a[at] = v
        assert lib.sgta_linear_i8(*a) < 0, (at, v)
    a = list(ok)
    a[1], a[4], a[11] = 131072, 131072, 131072
    assert lib.sgta_linear_i8(*a) == -2
    ok = [64, 32, 0, 64, 32, 64, 4, 32, None]
    for at, v in ((0, None), (1, 31), (2, 3), (3, None), (4, 31), (5, None), (6, 0), (7, 0)):
        a = list(ok)
        a[at] = v
        assert lib.sgta_quant_rows_i8(*a) < 0, (at, v)


@gpu
def test_more_rows_than_a_launch_takes():
    """2^23 rows a launch: the rows on both sides of each border, and the last."""
    M = (1 << 24) + 3
    x = torch.zeros(M, 16, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, (1 << 23) - 1, 1 << 23, (1 << 24) - 1, 1 << 24, M - 1], device="cuda")
    x[at] = torch.randn(6, 16, device="cuda").to(torch.bfloat16)
    xq, xs = ops_i8.quantize_rows(x)
    few, fews = ops_i8.quantize_rows(x[at].contiguous())
    assert torch.equal(xq[at], few) and torch.equal(xs[at], fews)
    assert int(xs.count_nonzero()) == 6 and int((xq != 0).any(1).sum()) == 6
