"""ops.window_attention at the ends of what its arguments may be: places and reaches beyond 32 bits, and tokens
that read nothing, whatever they hold."""
import math

import pytest
import torch

from medvision_b200.ops import window_attention

from test_cross_attention import HALF, NAMES, check
from test_window_attention import allowed_states, compare, make, reference, run


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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("heads,dim", [((4, 2), 64), ((2, 2), 128), ((6, 2), 64), ((3, 1), 128), ((8, 1), 32), ((2, 1), 20), ((2, 2), 200), ((1, 1), 96)])
def test_tokens_that_read_nothing_may_hold_anything(heads, dim, dtype):
    """Padded tokens behind short sequences, tokens before all states, sequences without states: their queries and incoming gradients come
    near no sum of another token's or state's, in no bit."""
    N, T, L, window = 5, 400, 400, (30, 0)
    offsets, lengths = [0, 0, -150, 37, 0], [150, 277, 400, 100, 0]
    q, k, v, g = make(N, T, *heads, dim, L, dtype, seed=22)
    kw = dict(offsets=torch.tensor(offsets, device="cuda"), lengths=torch.tensor(lengths, device="cuda"))
    clean = run(q, k, v, g, *window, **kw)
    nothing = torch.stack([~allowed_states(T, L, *window, 0, o, n).any(1) for o, n in zip(offsets, lengths)])
    assert bool(nothing.any(1).all()) and not bool(nothing[:4].all(1).any())
    for bad_q, bad_g in ((math.nan, math.nan), (math.inf, -math.inf), (0.5, math.nan), (math.nan, 0.5)):
        x, y = q.clone(), g.clone()
        x[nothing], y[nothing] = bad_q, bad_g
        got = run(x, k, v, y, *window, **kw)
        for a, b in zip(got, clean):
            assert torch.equal(a, b)
        assert not bool(got[0][nothing].any()) and not bool(got[1][nothing].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("heads", [(2, 2), (6, 2)])
@pytest.mark.parametrize("loud", ["query", "key"])
def test_float16_ranges_go_by_what_is_read(loud, heads, dim):
    """Slopes of weights are brought to float16's range by bounds of the values and of the incoming gradients: not by those of states and
    tokens that have no part in them, however large.  Here the slopes are as small as the largest factor leaves them; queries (or keys) of
    2^12 bring their gradients' products back to float16's normal numbers."""
    N, T, L, window = 3, 128, 400, (63, 0)
    offsets, lengths = [100, 0, 270], [400, 60, 330]
    q, k, v, g = make(N, T, *heads, dim, L, torch.float32, seed=23)
    up, down = (q, k) if loud == "query" else (k, q)
    up *= 2.0 ** 12
    down *= 2.0 ** -12
    q, k, v, g = q.half(), k.half(), (v / 64).half(), (g * 2.0 ** -14).half()
    read = torch.stack([allowed_states(T, L, *window, 0, o, n) for o, n in zip(offsets, lengths)])
    v[~read.any(1)], g[~read.any(2)] = 0.0, 0.0
    kw = dict(offsets=torch.tensor(offsets, device="cuda"), lengths=torch.tensor(lengths, device="cuda"))
    clean = run(q, k, v, g, *window, **kw)
    assert bool(clean[1 + (loud == "query")].any())
    for in_v, in_g in ((6e4, 0.0), (0.0, -6e4), (-6e4, 6e4)):
        x, y = v.clone(), g.clone()
        x[~read.any(1)], y[~read.any(2)] = in_v, in_g
        for a, b in zip(run(q, k, x, y, *window, **kw), clean):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape,window", [((1, 1500, 8, 1, 64, 1500), (400, 0, 5)), ((2, 900, 8, 1, 128, 900), (300, 10, 130)), ((1, 700, 6, 1, 64, 700), (200, 200, 130)),
                                          ((2, 500, 8, 1, 96, 500), (300, 0, 40)), ((1, 600, 4, 1, 200, 600), (250, 0, 40))])
def test_rows_and_first_states_in_parts_together(shape, window, dtype):
    """Few sequences and key heads: the rows of the first states' tiles and those of the others are both cut into parts, on the tensor cores and in
    float arithmetic, and the states of the queries' gradients too."""
    N, T, L = shape[0], shape[1], shape[5]
    compare(shape, window, dtype, seed=24)
    if N > 1:
        compare(shape, window, dtype, offsets=[-T // 3, 40], lengths=[L, L // 2 + 3], seed=25)


PRECISE = [((2, 257, 4, 2, 64, 257), (90, 0, 3)), ((1, 600, 2, 2, 128, 600), (40, 40, 0)), ((3, 1, 16, 4, 128, 700), (500, 0, 4)), ((2, 130, 3, 1, 32, 130), (2, 0, 0)),
           ((1, 1100, 2, 2, 40, 1100), (10 ** 9, 0, 0)), ((2, 300, 8, 1, 96, 300), (33, 7, 130)), ((1, 70, 2, 2, 33, 70), (9, 0, 1))]


def fine(q, k, v, g, window, offsets, lengths, scale, dtype):
    """What test_window_attention.reference gives for out and dv, with bounds in which a weight is a number of two pieces: off by the square of
    half a step, 3e-6 where its exponential is a polynomial, and in float16 2^-35 (the second piece's smallest step, weights being scaled by
    2^10 at least)."""
    u, few = HALF[dtype], 2.0 ** -35 if dtype == torch.float16 else 0.0
    rest, tiny = u * u + 3e-6, 2.0 ** -25 if dtype == torch.float16 else 0.0
    at = (offsets, lengths, scale, torch.float32)
    res, bound = reference(q, k, v, g, *window, *at)
    size = reference(q, k, v.abs(), g.abs(), *window, *at)[0]
    read = torch.stack([allowed_states(q.shape[1], k.shape[1], *window, o, n).double() for o, n in zip(offsets, lengths)])
    group = q.shape[2] // k.shape[2]
    every = {0: torch.einsum("ntj,njhd->nthd", read, v.abs().double()).repeat_interleave(group, 2),
             3: torch.einsum("ntj,nthd->njhd", read, g.abs().double()).unflatten(2, (-1, group)).sum(3)}
    for i in (0, 3):
        bound[i] += u * res[i].abs() + 2 * rest * size[i] + few * every[i] + tiny
    return [(res[i], bound[i]) for i in (0, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape,window", PRECISE)
def test_weights_keep_their_bits(shape, window, dtype):
    """Results and values' gradients are as far off as their own rounding, and the sums in float, put them: no weight is rounded to the type."""
    N, T, H, Hk, D, L = shape
    q, k, v, g = make(*shape, dtype, seed=26)
    offsets = [L - T - 3 * n for n in range(N)]
    lengths = [max(0, L - 5 * n) for n in range(N)]
    for alike in (False, True):  # (True: all weights of a row are 1 / n)
        if alike:
            q = torch.zeros_like(q)
        out, dv = fine(q, k, v, g, window, offsets, lengths, D ** -0.5, dtype)
        got = run(q, k, v, g, *window, offsets=torch.tensor(offsets, device="cuda"), lengths=torch.tensor(lengths, device="cuda"))
        check(got[0], *out, "out")
        check(got[3], *dv, "dv")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape,window", PRECISE)
def test_rounded_weights(shape, window, dtype):
    """The caller's choice: the bounds of attention whose weights are rounded once.  Without half types, or without tensor cores, it changes nothing."""
    q, k, v, g = make(*shape, dtype, seed=27)
    N, T, H, Hk, D, L = shape
    res, bound = reference(q, k, v, g, *window, [L - T] * N, [L] * N, D ** -0.5, dtype)
    got = run(q, k, v, g, *window, offsets=L - T, rounded_weights=True)
    for name, a, b, c in zip(NAMES, got, res, bound):
        check(a, b, c, name)
    if dtype == torch.float32:
        for a, b in zip(got, run(q, k, v, g, *window, offsets=L - T)):
            assert torch.equal(a, b)
