"""Large finite values in the table of ``rel_attention``: a softmax does not see a constant, so keys that all lie in buckets of one value
weigh the same whatever the value is, and keys of a far lower value than others weigh nothing.  The references and bounds are those of a
moderate value in its place (test_attention.py): they do not grow with the value.

What a value adds to a bound: a row's reference (its maximum in units of log2, in f32) is off the true one by half a step of it, 64 for
values below 2^31 in those units, so the terms of a weight's exponent are up to 64 + |s| and its three roundings 3 * 2^-24 * 80 * ln 2 =
166 * 2^-24 of the weight.  The moderate value is 40 or more in magnitude: the bound's 2 es holds 8 * 2^-24 * 40 for it.
"""
import pytest
import torch

from test_attention import NAMES, Case, both_ways, forward, gradients, within

gpu = pytest.mark.gpu
VALUES = [(torch.float32, v) for v in (-1e4, -1e6, -1e9, 1e9)] + [(torch.bfloat16, v) for v in (-1e4, -1e9, 1e6)] + [(torch.float16, v) for v in (-1e4, -65504.0)]
IDS = ["%s %g" % (NAMES[t], v) for t, v in VALUES]


def check(c, buckets, value, moderate):
    """Table entries ``buckets`` hold ``value``; reference and bounds with ``moderate`` there.

    Where other keys are seen beside them, a value of -1e4 or less leaves weights of zero, a moderate one of -60 in the reference
    weights of up to exp(-60 + 15): the other scores, normal numbers and a normal bias, lie within 15 of each other.  3e-20 a weight, 600 pairs
    at most in a sum, values, queries, gradients and their products (D <= 64) below 1000: within 1e-13 of any result."""
    gone = 1e-13 if moderate < 0 else 0.0
    c.w[buckets] = moderate
    r, want = gradients(c)
    c.w[buckets] = value
    out, got = both_ways(c)
    alone = forward(c)
    torch.cuda.synchronize()
    rows = dict(dq=r["nq"], dk=r["nk"], dv=r["nk"])
    within("out", out, r["out"], r["out_tol"] + gone, r["nq"])
    within("out without save", alone, r["out"], r["out_tol"] + gone, r["nq"])
    for name, g in zip(("dq", "dk", "dv", "dw"), got):
        within(name, g, want[name][0], want[name][1] + gone, rows.get(name))


@gpu
@pytest.mark.parametrize("dtype,value", VALUES, ids=IDS)
def test_a_table_of_one_value(dtype, value):
    """Near, far and masked tiles, few queries and many, every head size."""
    every = slice(None)
    for Lq, Lk, H, Hkv, D, far in ((200, 300, 2, 2, 32, 40), (150, 260, 4, 2, 64, 128), (130, 190, 2, 1, 128, 40), (1, 700, 4, 1, 64, 128), (5, 90, 2, 2, 16, 40)):
        for causal in (False, True):
            check(Case(1, dtype, 2, Lq, Lk, H, Hkv, D, causal=causal, far=far, kv_len=[Lk, Lk - 37], q_start=[Lk - Lq, Lk - Lq - 30] if causal else None,
                       seed=D), every, value, 40.0)


@gpu
@pytest.mark.parametrize("dtype,value", VALUES, ids=IDS)
def test_rows_that_see_only_far_keys(dtype, value):
    """Every key farther than the last bucket of its own; whole tiles and tiles that the lengths cut."""
    for D in (32, 64, 96):
        for Lq in (1, 150):
            for causal in (False, True):
                c = Case(1, dtype, 4, Lq, 130, 2, 1, D, causal=causal, buckets=16, far=16, kv_len=[100, 128, 37, 64], q_start=[400, 150, 200, 333], seed=D)
                check(c, 15 if causal else 7, value, 40.0)


@gpu
@pytest.mark.parametrize("dtype,value", [x for x in VALUES if x[1] < 0], ids=[i for i, x in zip(IDS, VALUES) if x[1] < 0])
def test_rows_that_see_far_keys_beside_rows_that_see_near_ones(dtype, value):
    """The far buckets hide their keys from rows that see others, and from no one in rows that see nothing else."""
    for D in (32, 64):
        c = Case(1, dtype, 2, 300, 300, 2, 1, D, buckets=16, far=16, kv_len=[70, 33], seed=D)
        check(c, [7, 15], value, -60.0)
        c = Case(1, dtype, 2, 300, 300, 2, 1, D, buckets=16, far=16, seed=D)
        check(c, [3, 4, 5, 11, 12], value, -60.0)
