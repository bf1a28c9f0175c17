"""The attention kernels' forms for large grids (a wave for every 32 rows, from 416 work-groups of 128 rows on, in the forward pass with
lengths from 832 on) and the orders in which work-groups take heads, at sizes that a 64-bit reference can hold: many heads of short sequences.  Bounds as in test_attention.py.

Work-groups: B H ceil(Lq / 128) forward and for dQ, B Hkv ceil(Lk / 128) for dK and dV.
"""
import pytest
import torch

from test_attention import ALL, NAMES, Case, check_both, check_forward

gpu = pytest.mark.gpu

# B, Lq, Lk, H, Hkv: work-groups forward / dK dV, and what B Hkv (B H) is a multiple of
GRIDS = [(1, 33, 33, 704, 704),        # 704 / 704; 8
         (2, 130, 140, 176, 176),      # 704 / 704, two blocks a head; 8, lengths that end inside a tile
         (1, 50, 70, 704, 176),        # 704 / 176, shared heads; 8
         (1, 40, 33, 704, 44),         # 704 / 44; heads by 8, key heads not
         (1, 33, 45, 705, 705),        # 705 / 705; neither
         (1, 36, 35, 703, 703),        # 703 / 703; neither
         (1, 200, 131, 352, 176),      # 704 / 352, two blocks a head
         (1, 33, 36, 416, 416),        # 416 / 416: the first of the large ones; 8
         (1, 36, 33, 415, 415),        # 415 / 415: the last of the small ones; neither
         (2, 130, 40, 208, 208)]       # 832 / 416 with lengths: the first of the large ones of either pass
EVERY_TYPE = GRIDS[:2]


def lengths(B, Lq, Lk, causal):
    kw = dict(q_start=[max(0, Lk - Lq)] * B if causal else None)
    if B == 2:
        kw.update(kv_len=[Lk, 77], q_len=[Lq, 90])
    return kw


def cases():
    for n, grid in enumerate(GRIDS):
        for causal in (False, True):
            for t in ALL if grid in EVERY_TYPE else [ALL[(n + causal) % 3]]:
                yield pytest.param(grid, causal, t, n, id="%s %s %s" % (NAMES[t], "causal" if causal else "full", "x".join(map(str, grid))))


@gpu
@pytest.mark.parametrize("grid,causal,dtype,n", cases())
def test_rel_large_grids(grid, causal, dtype, n):
    B, Lq, Lk, H, Hkv = grid
    for D in {0: (64, 128), 1: (16, 40)}.get(n, ((32, 64, 96, 128, 24, 128, 40, 64)[n - 2],)):
        check_both(Case(1, dtype, B, Lq, Lk, H, Hkv, D, causal=causal, seed=D, **lengths(B, Lq, Lk, causal)))


@gpu
@pytest.mark.parametrize("grid,causal,dtype,n", cases())
def test_diff_large_grids(grid, causal, dtype, n):
    B, Lq, Lk, H, Hkv = grid
    for D, Dv in {0: ((64, 128),), 1: ((32, 64),)}.get(n, (((16, 32), (64, 128), (40, 24), (32, 64), (48, 96), (64, 128), (32, 64), (40, 128))[n - 2],)):
        check_both(Case(2, dtype, B, Lq, Lk, H, Hkv, D, Dv, causal=causal, seed=D, **lengths(B, Lq, Lk, causal)))


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("causal", [False, True])
def test_longer_sequences_on_large_grids(causal, dtype):
    """Four blocks a head and several tiles before, within and behind the reach."""
    for maps, D, Dv in ((1, 64, 64), (2, 32, 64)):
        check_forward(Case(maps, dtype, 1, 400, 400, 176, 44, D, Dv, causal=causal, far=60, seed=1))
    check_both(Case(1, dtype, 1, 270, 270, 240, 240, 32, causal=causal, far=60, seed=2))


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_rel_gradients_padded_heads(dtype):
    for D in (8, 24, 40, 96, 104):
        check_both(Case(1, dtype, 2, 70, 90, 2, 1, D, seed=D, kv_len=[90, 50]))


@gpu
@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
def test_wide_tables_on_large_grids(dtype):
    """Float heads beyond 64 with a reach beyond 256 take the same form whatever the grid."""
    check_both(Case(1, dtype, 1, 33, 40, 704, 704, 96, buckets=64, far=300, seed=5))
