"""ops.cross_attention where operands of one call differ in size by many powers of two: float16 has few bits for small numbers.

Tolerances are those of test_cross_attention, and for what float16 rounds on its way into a product:
  slopes   dS is rounded after a power of two that brings a bound B of |dS| to at least 2^14; a half's smallest step there is 2^-24, so
           an element is off by at most 2^-25 2^-14 B = 2^-39 B beside its relative rounding.  B: 2 D max|g| max|v|.
  weights  the largest is at least 2^11 before it is rounded: an element is off by at most 2^-25 2^-11 = 2^-36 of the largest, and 2^21
           states, the most that a call takes, by at most 2^-15 of it together, whatever their number.
"""
import math

import pytest
import torch

from medvision_b200.ops import cross_attention

from test_cross_attention import E, HALF, NAMES, check, make, reference, run


def slopes(q, k, v, g, image, allowed, scale):
    """What 2^-39 B per element of dS comes to in dq and dk, with B of the whole call."""
    q, k, v, g = (t.double() for t in (q, k, v, g))
    H, Hk, D = q.shape[2], k.shape[2], q.shape[3]
    dq, dk = torch.zeros_like(q), torch.zeros_like(k)
    most = 2 * D * float(g.abs().max()) * float(v[allowed].abs().max())
    for r, n in enumerate(image):
        for h in range(H if 0 <= n < k.shape[0] else 0):
            dq[r, :, h] = abs(scale) * 2.0 ** -39 * most * k[n, allowed[n], h * Hk // H].abs().sum(0)
            dk[n, allowed[n], h * Hk // H] += abs(scale) * 2.0 ** -39 * most * q[r, :, h].abs().sum(0)
    return dq, dk


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("indexed", [False, True])
@pytest.mark.parametrize("size", [1.0, 1e-4])
def test_half_gradients_where_values_of_some_states_are_small_or_zero(dim, indexed, size):
    """Background, padding: 128 states of 1e-6, 128 of 0, 128 of 1e-3, the rest ordinary.  delta averages over all of them, so that dS of a
    small state is as large as that of any other."""
    R, T, H, Hk, N, L = 3, 70, 2, 1, 3, 700
    q, k, v, g = make(R, T, H, Hk, dim, N, L, torch.float32, seed=21)
    q, g = (q * 4).half(), (g * size).half()
    v[:, :128] *= 1e-6
    v[:, 128:256] = 0
    v[:, 256:384] *= 1e-3
    k, v = k.half(), v.half()
    image = [2, 0, 0] if indexed else [0, 1, 2]
    kw = dict(batch_index=torch.tensor(image).cuda()) if indexed else {}
    allowed = torch.ones(N, L, dtype=torch.bool)
    res, bound = reference(q, k, v, g, image, allowed, dim ** -0.5, torch.float16)
    more = slopes(q, k, v, g, image, allowed, dim ** -0.5)
    bound[1] += more[0]
    bound[2] += more[1]
    for name, a, b, c in zip(NAMES, run(q, k, v, g, **kw), res, bound):
        check(a, b, c, name)



@pytest.mark.gpu
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("states", [2 ** 15, 2 ** 18])
@pytest.mark.parametrize("masked", [False, True])
def test_half_weights_of_many_states_far_below_the_largest(dim, states, masked):
    """One score of 8192 lies some 2^25.2 above the others, whose values alone are not 0: their weights are below a half's smallest step."""
    T, H, every = 2048, 8, 8192
    gen = torch.Generator().manual_seed(23)
    q = torch.zeros(1, T, H, dim, dtype=torch.float16)
    q[..., 3] = 1 + torch.randint(0, 10, (1, T, H), generator=gen) / 1024
    k = torch.zeros(1, states, 1, dim, dtype=torch.float16)
    k[:, ::every, :, 3] = 17.5
    v = torch.ones(1, states, 1, dim, dtype=torch.float16)
    v[:, 1::2, :, 1] = 0.5
    v[:, ::every] = 0
    mask = torch.ones(1, states, dtype=torch.bool)
    if masked:
        mask[:, 5::7] = False
    with torch.no_grad():
        out = cross_attention(q.cuda(), k.cuda().expand(1, states, H, dim), v.cuda().expand(1, states, H, dim), scale=1.0,
                              mask=mask.cuda() if masked else None)
    score = (q[..., 3].double() * 17.5).unsqueeze(-1)                       # of the far states; the others have 0
    some = mask[0].double()
    far = float(some[::every].sum())
    others = some.clone()
    others[::every] = 0
    values = (others @ v[0, :, 0].double()).view(1, 1, 1, dim)
    want = values * (-score).exp() / (far + others.sum() * (-score).exp())
    w = HALF[torch.float16] + 8 * math.sqrt(dim + states) * E + 8 * math.sqrt(dim) * E * 18
    bound = (2 * w + HALF[torch.float16]) * want + 2.0 ** -15 + 2.0 ** -25
    assert float(want.min()) > 3 * 2.0 ** -15  # (0 in its place would not pass)
    check(out, want, bound, "out")
