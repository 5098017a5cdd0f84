"""ops.cross_attention where operands of one call differ in size by many powers of two, where float16 has few bits for small
numbers, and where float32 operands are infinite, which the tensor cores take in pieces.

Tolerances are those of test_cross_attention, and for what float16 rounds on its way into a product:
  slopes   dS is rounded after a power of two that brings a bound B of |dS| to at least 2^14; a half's smallest step there is 2^-24, so
           an element is off by at most 2^-25 2^-14 B = 2^-39 B beside its relative rounding.  B: |g| times the largest |v| (2-norms) plus
           |delta|, of the row (dq) or the largest of the rows that read the state (dk).
  weights  the largest is at least 2^11 before it is rounded: an element is off by at most 2^-25 2^-11 = 2^-36 of the largest, and 2^21
           states, the most that a call takes, by at most 2^-15 of it together, whatever their number.
"""
import math

import pytest
import torch

from medvision_b200.ops import cross_attention

from test_cross_attention import E, HALF, NAMES, check, make, reference, run


def slopes(q, k, v, g, image, allowed, scale):
    """What 2^-39 B per element of dS comes to in dq (B of the row) and dk (B of all rows of the state's image and key head)."""
    q, k, v, g = (t.double() for t in (q, k, v, g))
    H, Hk = q.shape[2], k.shape[2]
    dq, dk = torch.zeros_like(q), torch.zeros_like(k)
    largest = torch.zeros(2, k.shape[0], Hk, dtype=torch.float64)  # of |g||v| and of |delta|
    rows = []
    for r, n in enumerate(image):
        for h in range(H if 0 <= n < k.shape[0] and bool(allowed[n].any()) else 0):
            kh = h * Hk // H
            a, b = k[n, allowed[n], kh], v[n, allowed[n], kh]
            delta = (g[r, :, h] * (torch.softmax(scale * q[r, :, h] @ a.T, 1) @ b)).sum(1).abs()
            gv = g[r, :, h].norm(dim=1) * b.norm(dim=1).max()
            dq[r, :, h] = abs(scale) * 2.0 ** -39 * (gv + delta)[:, None] * a.abs().sum(0)
            largest[:, n, kh] = torch.maximum(largest[:, n, kh], torch.stack([gv.max(), delta.max()]))
            rows.append((r, n, h, kh))
    for r, n, h, kh in rows:
        dk[n, allowed[n], kh] += abs(scale) * 2.0 ** -39 * largest[:, n, kh].sum() * q[r, :, h].abs().sum(0)
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
@pytest.mark.parametrize("tokens", [1, 70])
def test_half_gradients_of_quiet_rows_beside_loud_ones(dim, tokens):
    """Gradients that differ by 2^17 between regions: those of the quiet ones keep their bits, and do not depend on the others."""
    R, H, Hk, N, L = 6, 4, 2, 3, 500
    q, k, v, g = make(R, tokens, H, Hk, dim, N, L, torch.float32, seed=22)
    image = [0, 1, 1, -1, 2, 2]
    size = torch.tensor([2.0 ** 11, 2.0 ** -6, 2.0 ** -6, 2.0 ** 13, 2.0 ** 11, 2.0 ** -6])
    g = g * size.view(R, 1, 1, 1)
    q, k, v, g = (t.half() for t in (q, k, v, g))
    allowed = torch.ones(N, L, dtype=torch.bool)
    index = torch.tensor(image).cuda()
    res, bound = reference(q, k, v, g, image, allowed, dim ** -0.5, torch.float16)
    more = slopes(q, k, v, g, image, allowed, dim ** -0.5)
    bound[1] += more[0]
    bound[2] += more[1]
    got = run(q, k, v, g, batch_index=index)
    for name, a, b, c in zip(NAMES, got, res, bound):
        check(a, b, c, name)
    quiet = g.clone()
    quiet[size > 1] = 0
    alone = run(q, k, v, quiet, batch_index=index)
    assert torch.equal(got[1][size < 1], alone[1][size < 1])            # dq of the quiet regions
    assert torch.equal(got[2][1], alone[2][1]) and torch.equal(got[3][1], alone[3][1])  # dk, dv of an image that only they read
    assert not bool(got[1][3].any())


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


def _float_bits(pattern):
    return torch.tensor([pattern], dtype=torch.int32).view(torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,states", [(3, 40), (70, 8192)])  # float arithmetic, and pieces on the tensor cores
@pytest.mark.parametrize("dim", [20, 64])
def test_infinite_float_operands(tokens, states, dim):
    """An infinite value makes its column infinite; a key whose product with the query is -inf has no weight; NaN stays."""
    H, inf = 2, float("inf")
    q, k, v, g = make(1, tokens, H, H, dim, 1, states, torch.float32, seed=24)
    q[..., 0] = q[..., 0].abs() + 0.5
    allowed = torch.ones(1, states, dtype=torch.bool)
    res, bound = reference(q, k, v, g, [0], allowed, dim ** -0.5, torch.float32)
    dirty = v.clone()
    dirty[0, 5, 0, 3], dirty[0, 9, 1, 4], dirty[0, 7, 1, 6], dirty[0, 11, 1, 6] = inf, -inf, inf, -inf
    dirty[0, 12, 0, 8] = _float_bits(0x7f800001)                            # NaN whose upper half alone reads as infinity
    with torch.no_grad():
        out = cross_attention(q.cuda(), k.cuda(), dirty.cuda()).cpu()
    assert bool((out[..., 0, 3] == inf).all()) and bool((out[..., 1, 4] == -inf).all())
    assert bool(out[..., 1, 6].isnan().all()) and bool(out[..., 0, 8].isnan().all())
    special = torch.zeros(H, dim, dtype=torch.bool)
    for place in ((0, 3), (1, 4), (1, 6), (0, 8)):
        special[place] = True
    check(torch.where(special, res[0].float(), out), res[0], bound[0], "out")
    # keys that are infinitely far: as if they were left out
    dirty, gone = k.clone(), torch.zeros(1, states, dtype=torch.bool)
    gone[0, [0, 17, 33]] = True
    dirty[0, [0, 17, 33], :, 0] = -inf
    with torch.no_grad():
        out = cross_attention(q.cuda(), dirty.cuda(), v.cuda())
    res, bound = reference(q, k, v, g, [0], ~gone, dim ** -0.5, torch.float32)
    check(out, res[0], bound[0], "out")
    # an infinite query has no softmax; the other rows do not see it
    dirty = q.clone()
    dirty[0, 1, 0, 2] = inf
    with torch.no_grad():
        out = cross_attention(dirty.cuda(), k.cuda(), v.cuda()).cpu()
    res, bound = reference(q, k, v, g, [0], allowed, dim ** -0.5, torch.float32)
    assert bool(out[0, 1, 0].isnan().all())
    out[0, 1, 0] = res[0][0, 1, 0].float()
    check(out, res[0], bound[0], "out")
    # an infinite gradient reaches the values' gradients as it is
    dirty = g.clone()
    dirty[0, 2, 1, 7] = -inf
    dv = run(q, k, v, dirty)[3].cpu()
    assert bool((dv[0, :, 1, 7] == -inf).all())
    dv[0, :, 1, 7] = res[3][0, :, 1, 7].float()
    check(dv, res[3], bound[3], "dv")
