"""ops.group_norm at the ends of what its values may be."""
import math

import pytest
import torch

from test_cross_attention import HALF, check
from test_group_norm import ACTS, NAMES, make, reference, run


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape,groups", [((296, 4, 1000), 1000), ((300, 2, 96), 96), ((64, 1, 24), 3), ((2, 30, 64), 64), ((3, 1000, 40), 10), ((1, 90000, 8), 8),
                                          ((2, 50000, 32), 2), ((4, 3, 20), 20)])
def test_a_group_with_an_infinity_is_not_a_number(shape, groups, dtype):
    """However its values are dealt out to threads: one that holds all of them, one value each, first and last ones."""
    x, w, b, dy = make(shape, dtype, seed=30)
    N, S, C = shape
    width = C // groups
    for kind in ACTS:
        clean = run(x, groups, w, b, dy, kind)
        for row in sorted({0, S // 2, S - 1}):
            for bad in (math.inf, -math.inf):
                y, channel = x.clone(), (5 * width) % C + width - 1
                y[N - 1, row, channel] = bad
                spoilt = torch.zeros(shape, dtype=torch.bool)
                spoilt[N - 1, :, channel - width + 1:channel + 1] = True
                got = run(y, groups, w, b, dy, kind)
                for i in (0, 1):
                    assert bool(got[i].cpu()[spoilt].isnan().all()) and torch.equal(got[i].cpu()[~spoilt], clean[i].cpu()[~spoilt])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [None, "silu"])
@pytest.mark.parametrize("shape,groups", [((2, 500, 32), 4), ((1, 100000, 12), 3), ((3, 49, 256), 32), ((2, 3001, 33), 11), ((1, 60000, 64), 1), ((2, 7, 5000), 1),
                                          ((1, 20000, 7), 7), ((2, 40, 2056), 257)])
def test_the_mean_keeps_its_bits_far_from_zero(shape, groups, kind):
    """Values about 1e5 or -2^20 with deviations near 2, against the formula and the bounds of the same values about 0: their differences from
    the offset are floats, and neither result nor gradients depend on it.  The means' rounding alone would be 4e-3 or 3e-2."""
    for offset in (1e5, -2.0 ** 20):
        x, w, b, dy = make(shape, torch.float32, seed=31, offset=offset, spread=2.0)
        near = x - offset
        assert torch.equal(near.double(), x.double() - offset)
        want, bound = reference(near, groups, w, b, dy, kind)
        for name, a, c, e in zip(NAMES, run(x, groups, w, b, dy, kind), want, bound):
            check(a, c, e, name)
