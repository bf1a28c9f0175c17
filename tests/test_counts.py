"""Counts that do not fit the kernels' 32 bits are refused before anything is cut (tensors without memory: nothing is launched)."""
import ctypes

import pytest
import torch

from sgtapose_amd import _lib, ops_attn, ops_i8
from sgtapose_amd._lib import SgtaHipError


def empty(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("M,K", [((1 << 32) + 5, 1), (1 << 31, 4), (3, 1 << 31)])
def test_quantize_rows(M, K):
    with pytest.raises(SgtaHipError, match="32 bits"):
        ops_i8.quantize_rows(empty(M, K))


@pytest.mark.parametrize("M,N", [((1 << 32) + 5, 8), (1 << 31, 8), (8, 1 << 31), (8, (1 << 32) + 8)])
def test_linear_i8(M, N):
    i8 = torch.int8
    with pytest.raises(SgtaHipError, match="32 bits"):
        ops_i8.linear_i8(empty(M, 16, dtype=i8), empty(M, dtype=torch.float32), empty(N, 16, dtype=i8), empty(N, dtype=torch.float32))


def test_the_largest_count_is_not_refused_for_its_size():
    with pytest.raises(SgtaHipError, match="GPU"):
        ops_i8.quantize_rows(empty((1 << 31) - 1, 1))


@pytest.mark.parametrize("B,L,H", [((1 << 32) + 1, 4, 1), (1 << 24, 4, 1), (3, 4, 1 << 23), (1 << 10, (1 << 21) + 1, 1)])
def test_attention(B, L, H):
    q, k, v = (empty(B, L, H, 16) for _ in range(3))
    for call in (lambda: ops_attn.rel_attention(q, k, v, empty(32, H)),
                 lambda: ops_attn.diff_attention(empty(B, L, H, 2, 16), empty(B, L, H, 2, 16), v, empty(4, 16))):
        with pytest.raises(SgtaHipError, match="2\\^24"):
            call()


def test_table_gradient_grid():
    """A work-group a head and bucket."""
    lib = _lib.load()
    a = _lib.AttnArgs(q=64, k=64, v=64, w=64, out=64, lut=64, B=1, Lq=4, Lk=4, H=1 << 20, Hkv=1 << 20, D=16, Dv=16, dtype=2, reach=8,
                      num_buckets=16, scale=0.25, dout=64, dq=64, dk=64, dv=64, dw=64, stats=64, ws=64, ws_floats=1 << 40)
    assert lib.sgta_rel_attn_bwd(ctypes.byref(a), None) == -2
