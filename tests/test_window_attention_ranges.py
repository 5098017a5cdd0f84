"""ops.window_attention at the ends of what its arguments may be: places and reaches beyond 32 bits."""
import pytest
import torch

from medvision_b200.ops import window_attention

from test_cross_attention import HALF, NAMES, check
from test_window_attention import compare, make, reference, run


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", [(3, 1, 2, 2, 64, 300), (3, 150, 4, 2, 64, 300), (3, 200, 2, 1, 128, 200), (3, 40, 2, 2, 20, 70), (3, 33, 1, 1, 200, 50)])
def test_places_and_reaches_beyond_32_bits(shape, dtype):
    """Tokens far behind their states and far before them, that read all, some or none of them."""
    far = 2 ** 33
    T, L = shape[1], shape[5]
    for window in ((10 ** 12, 0, 0), (10 ** 12, 10 ** 12, 3), (far - L // 2, 0, 0), (0, far + T, 1), (far, far - 5, 0)):
        compare(shape, window, dtype, offsets=[far, -far, far + T + L], seed=20)


@pytest.mark.gpu
def test_one_far_place_for_all_sequences():
    q, k, v, g = make(2, 90, 2, 1, 32, 120, torch.float32, seed=21)
    most = 2 ** 63 - 1
    # the same windows in small numbers: all states, but for the last two, where token t's window begins at most + t - most = t and ends at
    # -2^63 + t + most = t - 1
    for offset, small, place in ((3 * 10 ** 9, (200, 200), 0), (-3 * 10 ** 9, (200, 200), 0), (2 ** 62, (200, 200), 0), (-2 ** 62, (200, 200), 0),
                                 (most, (0, 200), 0), (-2 ** 63, (200, 0), -1)):
        res, bound = reference(q, k, v, g, *small, 0, [place] * 2, [120] * 2, 32 ** -0.5, torch.float32)
        for name, a, b, c in zip(NAMES, run(q, k, v, g, most, most, offsets=offset), res, bound):
            check(a, b, c, name)
    none = window_attention(q.cuda(), k.cuda(), v.cuda(), 10 ** 9, 10 ** 9, offsets=3 * 10 ** 9)
    assert not bool(none.any())
