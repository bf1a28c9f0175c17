"""What ``save=True`` returns is read by the backward kernels as it was written: anything else is refused (on the CPU: nothing is launched)."""
import pytest
import torch

from sgtapose_amd import ops_attn
from sgtapose_amd._lib import SgtaHipError

SHAPE = (2, 5, 4, 16)                                    # B, Lq, H, Dv
like = torch.zeros(1, dtype=torch.bfloat16)


def stats(maps):
    return torch.zeros(maps, 2, 4, 5, 2)


def out2():
    return torch.zeros(SHAPE, dtype=torch.bfloat16)


def test_accepts_its_own():
    ops_attn._saved(stats(1), None, 1, SHAPE, like)
    ops_attn._saved(stats(2), out2(), 2, SHAPE, like)


@pytest.mark.parametrize("what,bad", [
    ("half the bytes", stats(1).half()), ("twice the bytes", stats(1).double()), ("another order", stats(1).transpose(1, 2).contiguous().transpose(1, 2)),
    ("expanded", torch.zeros(1, 1, 1, 1, 1).expand(1, 2, 4, 5, 2)), ("two maps", stats(2)), ("another device", stats(1).to("meta")), ("nothing", None)])
def test_statistics(what, bad):
    with pytest.raises(SgtaHipError, match="saved"):
        ops_attn._saved(bad, None, 1, SHAPE, like)


@pytest.mark.parametrize("what,bad", [
    ("none", None), ("another type", out2().float()), ("expanded", torch.zeros(1, 1, 1, 1, dtype=torch.bfloat16).expand(SHAPE)),
    ("another order", out2().transpose(1, 2).contiguous().transpose(1, 2)), ("another device", out2().to("meta")),
    ("two bytes off", torch.zeros(641, dtype=torch.bfloat16)[1:].view(SHAPE))])
def test_second_map(what, bad):
    with pytest.raises(SgtaHipError, match="saved"):
        ops_attn._saved(stats(2), bad, 2, SHAPE, like)
    with pytest.raises(SgtaHipError, match="saved"):
        ops_attn._saved(stats(1), out2(), 1, SHAPE, like)
