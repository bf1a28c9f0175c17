"""The live profile's work of the attention calls against the tensors and products of the formulas, counted one by one."""
import pytest

from sgtapose_amd import _lib, ops_attn


@pytest.mark.parametrize("maps,dtype,size", [(1, 0, 4), (1, 2, 2), (2, 1, 2)])
def test_work(monkeypatch, maps, dtype, size):
    B, Lq, Lk, H, Hkv, D, Dv = 2, 30, 50, 6, 3, 16, 16 * maps
    a = _lib.AttnArgs(B=B, Lq=Lq, Lk=Lk, H=H, Hkv=Hkv, D=D, Dv=Dv, dtype=dtype)
    assert ops_attn._meta("x", a, maps) is None
    monkeypatch.setattr(_lib, "PROFILE", [])
    pairs = B * H * Lq * Lk
    scores, values = 2 * pairs * D, 2 * pairs * Dv           # one product over all pairs
    q = dq = B * Lq * H * maps * D
    k = dk = B * Lk * Hkv * maps * D
    v = dv = B * Lk * Hkv * Dv
    out = dout = B * Lq * H * Dv
    m = ops_attn._meta("x", a, maps)
    assert m["flops"] == m["exec_flops"] == maps * (scores + values)
    assert m["bytes"] == size * (q + k + v + out)
    m = ops_attn._meta("x", a, maps, backward=True)
    # of each map the scores, dQ, dK; dO V^T and dV once; the two kernels compute the scores and dO V^T each
    assert m["flops"] == maps * 3 * scores + 2 * values
    assert m["exec_flops"] == m["flops"] + maps * scores + values
    second = out if maps == 2 else 0
    assert m["bytes"] == size * (q + k + v + out + second + dout + dq + dk + dv)
