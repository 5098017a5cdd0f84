"""The angles of ops.rotary_positions: places that lie next to whole turns, whose sines show the angle itself."""
import math

import pytest
import torch

from medvision_b200.ops import rotary_positions

from test_cross_attention import E


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_angles_are_rounded_to_the_nearest(kind):
    """An angle is a whole number of 2^-32 turns, off by half of one (a place's turns are off by less than 2^-64 a position); the sine by 4 e of
    itself more.  Cut off instead of rounded, a place in two would be off by more, always the same way."""
    places = [p for k in range(1, 400) for p in (710 * k, -710 * k)]
    places = [p for p in places if abs(math.remainder(p, 2 * math.pi)) < 1e-3 * 25]
    assert len(places) > 700
    x = torch.zeros(1, len(places), 1, 2)
    x[..., 0] = 1.0
    at = torch.tensor(places, dtype=kind).view(1, -1, 1)
    sines = rotary_positions(x.cuda(), at.cuda())[0, :, 0, 1].cpu().double()
    angles = torch.tensor([math.remainder(p, 2 * math.pi) - (p - math.remainder(p, 2 * math.pi)) / (2 * math.pi) * 2.4492935982947064e-16 for p in places],
                          dtype=torch.float64)  # (math.pi is 1.22e-16 less than pi)
    off = sines - angles.sin()
    half = 2 * math.pi * (2.0 ** -33 + 3e5 * 2.0 ** -64)
    assert bool((off.abs() <= half + 4 * E * angles.abs()).all()), "worst %g of %g" % (float(off.abs().max()), half)
    # ... and the mean of n errors of random signs within five standard deviations of 0
    assert abs(float(off.mean())) <= 5 * half / math.sqrt(3 * len(places)) + 4 * E * float(angles.abs().max()) / math.sqrt(len(places))
