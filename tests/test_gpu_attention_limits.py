"""Attention over the cache at the limits of its inputs, on the GPU.  Bounds and the
plain form in 64 bits are those of test_gpu_attention.py."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tests.test_gpu_attention import DEV, Case  # noqa: E402


I32 = torch.iinfo(torch.int32)


@pytest.mark.parametrize("held,t", [("bf16", None), ("int8", "bf16")])
@pytest.mark.parametrize("width", [8, 200])   # segments whole, and split and joined
@pytest.mark.parametrize("copies", [1, 40])   # with 40, 200 sequences: the join reads what the main kernel left
def test_the_smallest_lengths_with_positive_starts(copies, width, held, t):
    """lens - starts passes the ends of int32: nothing to attend to, and the others' bits as beside lengths of 0."""
    lens = [100, I32.min, 128, I32.min + 3, -1] * copies
    starts = [0, 5, 3, I32.max, I32.max] * copies
    c = Case(lens=lens, starts=starts, q_heads=6, k_heads=2, dim=64, page=16, held=held, t=t, width=width)
    got, lse = c.check()
    empty = torch.tensor(lens, device=DEV) < 0
    assert bool((got[empty] == 0).all() & (lse[empty] == -math.inf).all())
    c.l.clamp_(min=0)
    c.s[empty] = 0
    plain, plse = c.run()
    assert torch.equal(got, plain) and torch.equal(lse, plse)


@pytest.mark.parametrize("start", [1, 5, 1 << 30, I32.max])
@pytest.mark.parametrize("length", [I32.min, I32.min + 1, -(1 << 30) - 1, -1, 0])
def test_one_sequence_of_no_length_with_a_start(length, start):
    for width in (4, 4000):
        c = Case(lens=[length], starts=[start], q_heads=4, k_heads=2, dim=64, page=16, held="fp16", width=width)
        got, lse = c.run()
        assert bool((got == 0).all() & (lse == -math.inf).all())
