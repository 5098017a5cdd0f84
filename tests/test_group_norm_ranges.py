"""ops.group_norm at the ends of what its values may be."""
import math

import pytest
import torch

from test_cross_attention import HALF
from test_group_norm import ACTS, make, run


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
