"""ops.cross_attention against its formula in float64: forward, gradients, masks that leave nothing, odd sizes and strides, what
states that are left out may hold, other streams and graphs, and what it refuses.

Tolerances.  u: half a step of the type (weights of half types are rounded to it once, so is every result); e = 2^-24.  With
products of D terms and sums of n terms in float, errors of random signs grow with the square root; 8 sqrt(n) e covers six standard
deviations and the functions' own few ulps.
  score:   relative error of a weight  w = u + 8 sqrt(D + n) e + |scale| max|q||k| 8 sqrt(D) e          (u: half types only)
  out:     u |out| + 2 w sum p |v|                                      (numerator and normaliser)
  dv:      u |dv| + 2 w sum p |g|
  ds:      error  2 w |ds| + p (u sum|g||o| + 8 sqrt(D) e (sum|g||v| + sum|g||o|))      (delta is formed with the rounded output)
  dq, dk:  u |d| + scale sum err(ds) |k| or |q|
float16 adds its smallest step 2^-25 per result, and per weight (p below 2^-14 has fewer bits) 2^-25 of the values it meets.
"""
import ctypes
import math

import pytest
import torch

from medvision_b200.ops import cross_attention

E = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def reference(q, k, v, g, image, allowed, scale, dtype):
    """(value, bound) of out, dq, dk, dv, all float64 on the CPU.  image: list of ints (outside: none); allowed: (N, L) bool."""
    q, k, v, g = (t.detach().cpu().double() for t in (q, k, v, g))
    R, T, H, D = q.shape
    N, L, Hk, _ = k.shape
    u = HALF[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    res = [torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k)]
    bound, size = [torch.zeros_like(t) for t in res], [torch.zeros_like(t) for t in res]
    for r in range(R):
        n = image[r]
        if not 0 <= n < N or not bool(allowed[n].any()):
            continue
        J = allowed[n].nonzero().squeeze(1)
        for h in range(H):
            a, b = k[n, J, h * Hk // H], v[n, J, h * Hk // H]
            x, gr = q[r, :, h], g[r, :, h]
            s = scale * x @ a.T
            p = torch.softmax(s, 1)
            o = p @ b
            dp = gr @ b.T
            delta = (gr * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            big = float((abs(scale) * x.abs() @ a.abs().T).max())
            w = (0 if dtype == torch.float32 else u) + 8 * math.sqrt(D + len(J)) * E + 8 * math.sqrt(D) * E * big
            err = 2 * w * ds.abs() + tiny * (dp - delta).abs() + p * (u * (gr.abs() * o.abs()).sum(1, keepdim=True)
                + 8 * math.sqrt(D) * E * (gr.abs() @ b.abs().T + (gr.abs() * o.abs()).sum(1, keepdim=True)))
            res[0][r, :, h] = o
            bound[0][r, :, h] = 2 * w * p @ b.abs() + tiny * b.abs().sum(0)
            res[1][r, :, h] = scale * ds @ a
            bound[1][r, :, h] = abs(scale) * err @ a.abs()
            res[2][n, J, h * Hk // H] += scale * ds.T @ x
            bound[2][n, J, h * Hk // H] += abs(scale) * err.T @ x.abs()
            size[2][n, J, h * Hk // H] += abs(scale) * ds.abs().T @ x.abs()
            res[3][n, J, h * Hk // H] += p.T @ gr
            bound[3][n, J, h * Hk // H] += (2 * w * p + tiny).T @ gr.abs()
            size[3][n, J, h * Hk // H] += p.T @ gr.abs()
    rows = R * T * (H // Hk)
    for i in range(4):  # sums over the rows, and the rounding of the result
        bound[i] += u * res[i].abs() + 8 * math.sqrt(rows) * E * size[i] + tiny
    return res, bound


def check(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    err = (got - want).abs()
    bad = ~(err <= bound + 1e-30)
    assert not bool(bad.any()), "%s: %d of %d beyond the bound, worst %g of its bound" % (
        what, int(bad.sum()), err.numel(), float((err / (bound + 1e-30)).nan_to_num(1e9).max()))


def make(R, T, H, Hk, D, N, L, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    t = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    return t(R, T, H, D), t(N, L, Hk, D), t(N, L, Hk, D), t(R, T, H, D)


def run(q, k, v, g, **kw):
    q, k, v = (t.cuda().requires_grad_() for t in (q, k, v))
    out = cross_attention(q, k, v, **kw)
    return (out,) + torch.autograd.grad(out, (q, k, v), g.cuda())


NAMES = "out", "dq", "dk", "dv"
SHAPES = [  # R, T, H, Hk, D, N, L
    (3, 1, 1, 1, 1, 3, 1),
    (2, 5, 4, 2, 16, 2, 7),
    (1, 64, 2, 2, 32, 1, 64),
    (2, 65, 2, 1, 64, 2, 129),
    (1, 130, 3, 3, 128, 1, 257),
    (2, 33, 4, 1, 72, 2, 300),
    (1, 9, 2, 2, 33, 1, 70),
    (1, 3, 2, 2, 200, 1, 97),
    (1, 2, 1, 1, 256, 1, 40),
    (2, 1, 8, 2, 128, 2, 1500),
    (1, 700, 1, 1, 32, 1, 5),
    (4, 1, 32, 4, 40, 4, 517),
    (2, 150, 4, 2, 33, 2, 1000),  # large enough that odd head sizes are padded
    (1, 260, 2, 2, 100, 1, 2100),
    (3, 70, 6, 1, 64, 3, 140),    # six heads share a key head: 64 rows are no whole tokens
    (2, 300, 2, 2, 128, 2, 260),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_formula(shape, dtype):
    R, T, H, Hk, D, N, L = shape
    q, k, v, g = make(*shape, dtype)
    res, bound = reference(q, k, v, g, list(range(R)), torch.ones(N, L, dtype=torch.bool), D ** -0.5, dtype)
    for name, a, b, c in zip(NAMES, run(q, k, v, g), res, bound):
        check(a, b, c, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind", ["lengths", "mask", "both"])
@pytest.mark.parametrize("tokens,dim", [(1, 32), (49, 64), (3, 20), (2, 128)])
def test_regions_of_images_with_states_left_out(dtype, kind, tokens, dim):
    """Regions in no order, images without regions, without states, indices outside; the states left out hold NaN and infinities."""
    R, N, L, H, Hk = 23, 6, 211, 4, 2
    q, k, v, g = make(R, tokens, H, Hk, dim, N, L, dtype, seed=1)
    gen = torch.Generator().manual_seed(2)
    index = torch.randint(0, N - 1, (R,), generator=gen).float()  # image 5: no region
    index[4], index[9], index[11] = -1, N, float("nan")
    lengths = torch.tensor([L, 0, 1, 130, -3, 400])
    mask = torch.rand(N, L, generator=gen) < 0.6
    mask[0, :128] = False
    mask[3] = False
    allowed = torch.ones(N, L, dtype=torch.bool)
    kw = dict(batch_index=index.cuda(), scale=0.3)
    if kind != "mask":
        allowed &= torch.arange(L) < lengths[:, None]
        kw["lengths"] = lengths.cuda().to(torch.int32 if dim == 32 else torch.int64)
    if kind != "lengths":
        allowed &= mask
        kw["mask"] = mask.cuda()
    image = [int(i) if i == i and 0 <= i < N else -1 for i in index.tolist()]
    res, bound = reference(q, k, v, g, image, allowed, 0.3, dtype)
    dirty = torch.tensor([float("nan"), float("inf"), -float("inf")])[torch.randint(0, 3, k.shape, generator=gen)].to(dtype)
    keep = allowed[:, :, None, None]
    from medvision_b200 import _C, _lib
    _C.last_status()
    got = run(q, torch.where(keep, k, dirty), torch.where(keep, v, dirty), g, **kw)
    assert _C.last_status() == _lib.MVR_STATUS_BAD_BATCH_INDEX
    for name, a, b, c in zip(NAMES, got, res, bound):
        check(a, b, c, name)
    assert not bool(got[2].detach().cpu()[~allowed].any()) and not bool(got[3].detach().cpu()[~allowed].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_strides_and_broadcast_states(dtype):
    R, T, H, D, L = 3, 6, 4, 32, 90
    q, k, v, g = make(R, T, H, H, D, R, L, dtype, seed=3)
    allowed = torch.ones(R, L, dtype=torch.bool)
    res, bound = reference(q, k, v, g, [0, 1, 2], allowed, D ** -0.5, dtype)
    views = [q.transpose(1, 2).contiguous().transpose(1, 2),         # heads before tokens
             k.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2),  # a map's layout: states innermost
             torch.cat([v, v], 3)[..., :D]]                           # rows with a gap
    wide = torch.empty(R, T, H, D + 1, dtype=dtype)                   # rows that start at odd places
    wide[..., 1:] = g
    for name, a, b, c in zip(NAMES, run(*views, wide[..., 1:]), res, bound):
        check(a, b, c, name)
    off = torch.empty(k.numel() + 1, dtype=dtype)                     # states that are not 16-byte aligned
    off[1:] = k.reshape(-1)
    for name, a, b, c in zip(NAMES, run(q, off[1:].view(k.shape), v, g), res, bound):
        check(a, b, c, name)
    # one image's states for all regions
    res, bound = reference(q, k[:1].expand(R, -1, -1, -1), v[:1].expand(R, -1, -1, -1), g, [0, 1, 2], allowed, D ** -0.5, dtype)
    leaves = [t.cuda().requires_grad_() for t in (q, k[:1], v[:1])]
    out = cross_attention(leaves[0], leaves[1].expand(R, -1, -1, -1), leaves[2].expand(R, -1, -1, -1))
    grads = torch.autograd.grad(out, leaves, g.cuda())
    check(out, res[0], bound[0], "out")
    for i in (1, 2):  # three rounded gradients are added, and each sum is rounded
        check(grads[i], res[1 + i].sum(0, keepdim=True), (bound[1 + i] + 2 * HALF[dtype] * res[1 + i].abs()).sum(0, keepdim=True), NAMES[1 + i])


@pytest.mark.gpu
def test_gradients_agree_with_differences():
    q, k, v, g = (t.cuda() for t in make(2, 3, 2, 1, 8, 2, 11, torch.float32, seed=4))
    f = lambda *t: float((cross_attention(*t).detach().double() * g.double()).sum())  # noqa: E731
    grads = run(q, k, v, g)[1:]
    gen = torch.Generator().manual_seed(5)
    for i in range(3):
        d = torch.randn(grads[i].shape, generator=gen).cuda()
        h = 2.0 ** -7
        at = lambda s: [t + s * h * d if j == i else t for j, t in enumerate((q, k, v))]  # noqa: E731
        slope = (8 * (f(*at(1)) - f(*at(-1))) - (f(*at(2)) - f(*at(-2)))) / (12 * h)
        want = float((grads[i].double() * d.double()).sum())
        # each value of f is a sum of 96 float terms of size about 1: off by at most 96 * 2^-22; fourth order in h beyond that
        assert abs(slope - want) <= 18 * 96 * 2.0 ** -22 / (12 * h) + 200 * h ** 4 * max(1, abs(want)), (i, slope, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_extreme_scores(dtype):
    """One score far above the others, and all scores equal: the softmax is formed about the maximum."""
    R, L, D = 1, 150, 16
    q, k, v, g = make(R, 2, 1, 1, D, R, L, dtype, seed=6)
    q, k = q * 8, k * 8
    k[0, 77] = q[0, 0, 0] * 2  # about 16 000 / 4 above
    q[0, 1] = 0
    res, bound = reference(q, k, v, g, [0], torch.ones(1, L, dtype=torch.bool), 0.25, dtype)
    for name, a, b, c in zip(NAMES, run(q, k, v, g, scale=0.25), res, bound):
        check(a, b, c, name)


@pytest.mark.gpu
def test_the_same_call_gives_the_same_bits_on_any_stream_and_in_a_graph():
    q, k, v, g = make(40, 7, 4, 2, 64, 3, 1300, torch.float16, seed=7)
    index = torch.randint(0, 3, (40,), generator=torch.Generator().manual_seed(8)).cuda()
    want = run(q, k, v, g, batch_index=index)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        again = run(q, k, v, g, batch_index=index)
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    # a captured step, replayed on new values, beside a second graph that is captured from the same memory pool's leaves
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    gc = g.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(cross_attention(*leaves, batch_index=index), leaves, gc)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = cross_attention(*leaves, batch_index=index)
            grads = torch.autograd.grad(out, leaves, gc)
        graphs.append((graph, (out,) + grads))
    with torch.no_grad():
        for t in leaves:
            t.mul_(0.5)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    fresh = run(q * 0.5, k * 0.5, v * 0.5, g, batch_index=index)
    for _, results in graphs:
        assert all(torch.equal(a, b) for a, b in zip(results, fresh))


@pytest.mark.gpu
def test_a_thread_that_has_not_called_cuda_gets_the_same_kernels():
    """Tensor maps need a context: without one the call would take the kernels of float arithmetic, whose last bits differ."""
    import subprocess
    import sys
    import threading
    q, k, v, g = make(2, 70, 4, 2, 64, 2, 600, torch.float16, seed=12)
    want = run(q, k, v, g)
    got, cuda = [], [t.cuda() for t in (q, k, v)]
    torch.cuda.synchronize()
    thread = threading.Thread(target=lambda: got.append(cross_attention(*cuda)))
    thread.start()
    thread.join()
    assert torch.equal(got[0], want[0])
    # the first gradient of a process, in autograd's new thread, equals the second
    code = ("import torch; from medvision_b200.ops import cross_attention as f\n"
            "t = [torch.randn(2, 300, 4, 64, device='cuda', dtype=torch.float16, requires_grad=True) for _ in range(3)]\n"
            "a, b = (torch.autograd.grad(f(*t).sum(), t) for _ in range(2))\n"
            "assert all(torch.equal(x, y) for x, y in zip(a, b))\n")
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.gpu
def test_many_regions_of_many_images_are_grouped_right():
    R, N, L, D = 5000, 700, 3, 8
    q, k, v, _ = make(R, 1, 1, 1, D, N, L, torch.float32, seed=9)
    index = torch.randint(-1, N + 1, (R,), generator=torch.Generator().manual_seed(10))
    for t in (torch.int64, torch.int16, torch.float64, torch.float32):
        out = cross_attention(q.cuda(), k.cuda(), v.cuda(), batch_index=index.cuda().to(t)).cpu().double()
        at = index.clamp(0, N - 1)
        p = torch.softmax(torch.einsum("rd,rld->rl", q[:, 0, 0].double(), k[at, :, 0].double()) * D ** -0.5, 1)
        want = torch.einsum("rl,rld->rd", p, v[at, :, 0].double())
        want[(index < 0) | (index >= N)] = 0
        # sums of 3 and 8 terms of size about 1
        assert float((out[:, 0, 0] - want).abs().max()) <= 64 * E * 8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_states_beyond_32_bits(dtype):
    """More than 2^32 elements of keys: the last states of a long cache, read alone."""
    L, Hk, D = 2 ** 20 + 40, 64, 64
    q, k5, v5, _ = make(1, 2, Hk, Hk, D, 1, 5, dtype, seed=11)
    k = torch.full((1, L, Hk, D), float("nan"), dtype=dtype, device="cuda")
    v = torch.full((1, L, Hk, D), float("nan"), dtype=dtype, device="cuda")
    k[:, -5:], v[:, -5:] = k5.cuda(), v5.cuda()
    assert k.numel() > 2 ** 32
    mask = torch.zeros(1, L, dtype=torch.bool, device="cuda")
    mask[:, -5:] = True
    res, bound = reference(q, k5, v5, torch.zeros_like(q), [0], torch.ones(1, 5, dtype=torch.bool), D ** -0.5, dtype)
    check(cross_attention(q.cuda(), k, v, mask=mask), res[0], bound[0], "out")


@pytest.mark.gpu
def test_the_status_word_is_clean_after_all_kinds_of_calls():
    """No wait of the kernels ran out."""
    from medvision_b200 import _C
    _C.last_status()
    for dtype in HALF:
        for shape in [(2, 300, 4, 2, 64, 2, 1000), (1, 300, 2, 2, 128, 1, 700), (8, 1, 8, 2, 128, 8, 3000)]:
            run(*make(*shape, dtype))
    assert _C.last_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", [(2, 5, 4, 2, 33, 2, 40), (2, 140, 4, 2, 64, 2, 700), (2, 140, 4, 2, 128, 2, 700)])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_scales_that_are_not_positive(shape, dtype, scale):
    R, T, H, Hk, D, N, L = shape
    q, k, v, g = make(*shape, dtype, seed=11)
    allowed = torch.rand(N, L, generator=torch.Generator().manual_seed(12)) < 0.6
    res, bound = reference(q, k, v, g, list(range(R)), allowed, scale, dtype)
    for name, a, b, c in zip(NAMES, run(q, k, v, g, mask=allowed.cuda(), scale=scale), res, bound):
        check(a, b, c, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("R,T,N", [(128, 1, 256), (129, 1, 256), (128, 1, 257), (64, 2, 3), (43, 3, 3), (1, 1, 1)])
def test_edges_of_the_ways_regions_are_found(dtype, R, T, N):
    """128 rows and 256 images are the most that a kernel looks through itself; many regions in one image, and some in none."""
    from medvision_b200 import _C, _lib
    L = 70 if dtype == torch.float16 else 2 ** 13  # (float: enough scores for the tensor cores)
    if dtype == torch.float32 and N > 3:
        L = 2 ** 12
    q, k, v, g = make(R, T, 1, 1, 16, 1, L, dtype, seed=13)
    k, v = k.expand(N, L, 1, 16), v.expand(N, L, 1, 16)
    index = torch.randint(-1, N + 1, (R,), generator=torch.Generator().manual_seed(14))
    index[: R // 2] = N - 1
    _C.last_status()
    with torch.no_grad():
        got = cross_attention(q.cuda(), k.cuda(), v.cuda(), batch_index=index.cuda())
    one, bound = reference(q, k[:1], v[:1], g, [0 if 0 <= i < N else -1 for i in index.tolist()], torch.ones(1, L, dtype=torch.bool), 0.25, dtype)
    check(got, one[0], bound[0], "out")
    outside = bool(((index < 0) | (index >= N)).any())
    assert _C.last_status() == (_lib.MVR_STATUS_BAD_BATCH_INDEX if outside else 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dim", [64, 128])
def test_states_that_no_region_reads_get_zero_gradients(dtype, dim):
    q, k, v, g = make(150, 20, 2, 1, dim, 3, 300, dtype, seed=15)
    index = torch.ones(150)
    out, dq, dk, dv = run(q, k, v, g, batch_index=index.cuda())
    for t in (dk, dv):
        assert not bool(t[[0, 2]].any()) and bool(t[1].any())
    none = run(q[:0], k, v, g[:0], batch_index=index[:0].cuda())
    assert none[0].shape == q[:0].shape and not bool(none[2].any()) and not bool(none[3].any())


@pytest.mark.gpu
def test_empty_calls():
    for shape in [(0, 2, 2, 2, 16, 0, 5), (2, 0, 2, 2, 16, 2, 5), (2, 2, 2, 2, 16, 2, 0)]:
        q, k, v, g = make(*shape, torch.float16)
        got = run(q, k, v, g)
        assert all(not bool(t.any()) for t in got) and got[0].shape == q.shape and got[2].shape == k.shape
    q, k, v, g = make(0, 2, 2, 2, 16, 3, 5, torch.float16)
    got = run(q, k, v, g, batch_index=torch.zeros(0).cuda())
    assert not bool(got[2].any()) and got[2].shape == k.shape
    q, k, v, g = make(4, 2, 2, 2, 16, 0, 5, torch.float16)
    assert not bool(run(q, k, v, g, batch_index=torch.zeros(4).cuda())[0].any())


def test_refusals():
    q, k, v, _ = make(2, 3, 4, 2, 16, 2, 5, torch.float32)
    with pytest.raises(RuntimeError, match="cross_attention is not implemented on CPU"):
        cross_attention(q, k, v)
    with pytest.raises(RuntimeError, match="not implemented for 'float64'"):
        cross_attention(q.double(), k.double(), v.double())
    with pytest.raises(RuntimeError, match="expected scalar type torch.float32 but found torch.float16"):
        cross_attention(q, k.half(), v)
    with pytest.raises(RuntimeError, match="expected query"):
        cross_attention(q[0], k, v)
    with pytest.raises(RuntimeError, match="same shape"):
        cross_attention(q, k, v[:, 1:])
    with pytest.raises(RuntimeError, match="same head size"):
        cross_attention(q[..., :8], k, v)
    with pytest.raises(RuntimeError, match="multiple of the number of key heads"):
        cross_attention(q[:, :, :3], k, v)
    with pytest.raises(RuntimeError, match="head sizes up to 256"):
        cross_attention(torch.zeros(1, 1, 1, 257), torch.zeros(1, 1, 1, 257), torch.zeros(1, 1, 1, 257))
    with pytest.raises(RuntimeError, match="heads and head size must not be 0"):
        cross_attention(q[..., :0], k[..., :0], v[..., :0])
    with pytest.raises(RuntimeError, match="one region per image"):
        cross_attention(q[:1], k, v)
    with pytest.raises(RuntimeError, match="one element per region"):
        cross_attention(q, k, v, batch_index=torch.zeros(3))
    with pytest.raises(RuntimeError, match="batch_index cannot be of type bool"):
        cross_attention(q, k, v, batch_index=torch.zeros(2, dtype=torch.bool))
    with pytest.raises(RuntimeError, match="one element per image"):
        cross_attention(q, k, v, lengths=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="lengths must be int32 or int64"):
        cross_attention(q, k, v, lengths=torch.zeros(2))
    with pytest.raises(RuntimeError, match="mask must be .images, states."):
        cross_attention(q, k, v, mask=torch.ones(2, 4, dtype=torch.bool))
    with pytest.raises(RuntimeError, match="mask must be bool"):
        cross_attention(q, k, v, mask=torch.ones(2, 5))
    with pytest.raises(RuntimeError, match="scale must be finite"):
        cross_attention(q, k, v, scale=math.inf)
    with pytest.raises(RuntimeError, match="scale must be finite"):  # (in float32)
        cross_attention(q, k, v, scale=1e300)
    with pytest.raises(TypeError, match="query must be a Tensor"):
        cross_attention(None, k, v)


def test_c_entry_checks_before_any_cuda_call():
    from medvision_b200 import _lib
    L, null = _lib.lib, None

    def call(backward=False, bytes=None, **kw):
        a = _lib.Attention(dtype=1, R=2, T=3, Hq=4, Hk=2, N=2, L=50, D=16, q=16, k=16, v=16, out=16)
        for name, value in kw.items():
            setattr(a, name, value)
        if bytes is None:
            need = ctypes.c_int64()
            rc = L.mvr_attention_workspace(ctypes.byref(a), int(backward), ctypes.byref(need))
            return rc, need.value
        if backward:
            return L.mvr_attention_backward(ctypes.byref(a), 16, bytes, null, null)
        return L.mvr_attention_forward(ctypes.byref(a), 16, bytes, null, null)

    assert call()[0] == 0
    assert call(dtype=2)[0] == -1 and call(R=-1)[0] == -5 and call(Hq=3)[0] == -15 and call(D=257)[0] == -16
    assert call(R=3)[0] == -5 and call(R=3, has_index=1)[0] == 0
    assert call(N=10 ** 6, R=10 ** 6)[0] == 0 and call(N=10 ** 6, has_index=1)[0] == -9
    assert call(T=2 ** 31)[0] == -9 and call(R=2 ** 28, N=2 ** 28, T=64)[0] == -9
    assert L.mvr_attention_forward(None, null, 0, null, null) == -6
    big = 1 << 40
    assert call(bytes=big, q=null) == -6 and call(bytes=big, out=null) == -6
    assert call(bytes=big, has_index=1) == -6  # no index
    assert call(bytes=big, has_index=1, index=16, index_type=8) == -1
    assert call(backward=True, bytes=big) == -6  # no gradient
    assert call(has_index=1)[1] > 0 and call(bytes=0, has_index=1, index=16) == -14
    assert "workspace" in _lib.strerror(-14)
    # nothing to do: no launch, no error
    assert call(bytes=big, T=0) == 0 and call(bytes=big, R=0, N=0) == 0


@pytest.mark.gpu
def test_second_derivatives_and_tangents_are_refused():
    import torch.autograd.forward_ad as fwAD
    q, k, v, g = (t.cuda() for t in make(1, 2, 1, 1, 8, 1, 4, torch.float32))
    q.requires_grad_()
    gq, = torch.autograd.grad(cross_attention(q, k, v), q, g, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        gq.sum().backward()
    with fwAD.dual_level(), pytest.raises(NotImplementedError, match="no forward-mode derivative"):
        cross_attention(fwAD.make_dual(q.detach(), torch.ones_like(q)), k, v)
