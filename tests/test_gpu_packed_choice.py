"""Packed prompts of up to 160 tokens on both sides of the rule that chooses between the kernel for short sequences and the tiles: the same call
with a larger bound on the lengths always takes the tiles."""
import pytest
import torch

from test_gpu_packed_prefill import call, check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def d():
    import puter_b200

    return puter_b200.Device()


@pytest.mark.parametrize("fmt", [2, 1])
@pytest.mark.parametrize("batch,longest,heads,kv,dim", [(300, 128, 16, 1, 64), (130, 160, 32, 2, 64), (300, 95, 16, 1, 64), (300, 96, 16, 1, 64), (300, 112, 16, 2, 64),
                                                        (200, 130, 28, 4, 64), (100, 128, 32, 1, 40), (40, 160, 16, 2, 128), (300, 24, 8, 1, 128)])
def test_both_sides_of_the_choice(d, fmt, batch, longest, heads, kv, dim):
    lens = [(37 * i) % (longest + 1) for i in range(batch - 1)] + [longest]
    q, k, v, starts = make(fmt, lens, heads, kv, dim, batch + heads)
    outs = [call(d, q, k, v, starts, heads, kv, dim, fmt, longest=n) for n in (longest, 161)]
    for out in outs:
        check(out, q, k, v, starts, heads, kv, dim, fmt, True, None)
    assert d.take_error() == 0
