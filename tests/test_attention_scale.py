"""Scales far from one: the kernels work in units of log2, with the scale times log2 e and, for dK and dV, its inverse, both in float32."""
import ctypes

import pytest
import torch

from sgtapose_amd import _lib, ops_attn
from sgtapose_amd._lib import SgtaHipError
from test_attention import ALL, NAMES, Case, check_both

gpu = pytest.mark.gpu


@pytest.mark.parametrize("scale", [3e38, 1e37, 1e-37, 1e-40, 1e-300, 1e300])
def test_refuses_what_has_no_inverse(scale):
    q = torch.empty(2, 5, 4, 16, device="meta")
    with pytest.raises(SgtaHipError, match="scale"):
        ops_attn.rel_attention(q, q, q, torch.empty(32, 4, device="meta"), scale=scale)
    a = _lib.AttnArgs(q=64, k=64, v=64, w=64, out=64, lut=64, B=1, Lq=4, Lk=4, H=2, Hkv=2, D=16, Dv=16, dtype=2, reach=8, num_buckets=8, scale=scale)
    assert _lib.load().sgta_rel_attn_fwd(ctypes.byref(a), None) == -1


@gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("scale", [1e-36, 1e-12, 30.0])
def test_far_from_one(maps, dtype, scale):
    """1e-36 weighs all keys alike but for the bias; 30 leaves one or two keys of a row.  dQ and dK carry the scale."""
    for Lq, Lk in ((150, 200), (3, 90)):
        check_both(Case(maps, dtype, 2, Lq, Lk, 4, 2, 32, causal=maps == 1, q_start=[50, 0] if maps == 1 else None, scale=scale, seed=4))
