"""ops.rotary_positions against its formula in float64: both kinds of pairs, sections, types, far positions, strides, gradients, graphs,
and what it refuses.

Tolerances.  e = 2^-24, u half a step of the type.  Sine and cosine are within 4 e (a float's rounding, the function's, the correction's),
the products and their sum three roundings more: 8 e (|a| + |b|), and the result's own u.  A position p adds 8 |p| 2^-53 of turns' rounding
on both sides.  float16 adds its smallest step 2^-25."""
import ctypes
import math

import pytest
import torch

from medvision_b200 import _lib
from medvision_b200.ops import rotary_positions

from test_cross_attention import E, HALF, check


def even(dim, axes):
    return [dim // 2 // axes + (i < dim // 2 % axes) for i in range(axes)]


def reference(x, positions, sections, base, interleaved, sign=1):
    u, tiny = HALF[x.dtype], 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    y = x.detach().cpu().double().clone()
    bound = torch.zeros_like(y)
    P, i = sum(sections), 0
    for axis, n in enumerate(sections):
        place = positions[..., axis].detach().cpu().double()[..., None]
        for k in range(n):
            angle = sign * place * base ** (-k / n)
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + P)
            s, t = y[..., a].clone(), y[..., b].clone()
            y[..., a], y[..., b] = s * angle.cos() - t * angle.sin(), s * angle.sin() + t * angle.cos()
            error = (8 * E + 8 * place.abs() * base ** (-k / n) * 2.0 ** -53) * (s.abs() + t.abs())
            bound[..., a], bound[..., b] = error + u * y[..., a].abs() + tiny, error + u * y[..., b].abs() + tiny
            i += 1
    return y, bound


def make(N, L, H, D, axes, dtype, kind=torch.float32, far=300.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, L, H, D, generator=g).to(dtype)
    return x, ((torch.rand(N, L, axes, generator=g) - 0.3) * far).to(kind)


def compare(x, positions, sections, interleaved=False, base=1e4, key=None):
    given = even(x.shape[-1], positions.shape[-1]) if sections is None else sections
    leaves = [t.cuda().requires_grad_() for t in (x, key) if t is not None]
    out = rotary_positions(leaves[0], positions.cuda(), leaves[1] if key is not None else None, sections, base, interleaved)
    out = out if key is not None else (out,)
    grads = [torch.randn(t.shape, generator=torch.Generator().manual_seed(9)).to(t.dtype) for t in leaves]
    back = torch.autograd.grad(out, leaves, [g.cuda() for g in grads])
    for t, o, g, b in zip((x, key), out, grads, back):
        assert o.is_contiguous() and o.dtype == t.dtype
        check(o, *reference(t, positions, given, base, interleaved), "turned")
        check(b, *reference(g, positions, given, base, interleaved, -1), "gradient")


SHAPES = [  # N, L, H, D, axes, sections
    (1, 1, 1, 1, 1, [0]),
    (1, 1, 1, 2, 1, None),
    (2, 3, 4, 16, 3, None),
    (3, 50, 8, 64, 2, None),
    (2, 129, 3, 128, 4, [10, 0, 50, 4]),
    (2, 17, 5, 33, 3, [5, 6, 5]),
    (1, 33, 2, 40, 2, [4, 6]),           # columns behind the pairs
    (2, 20, 1, 24, 1, [12]),
    (2, 9, 2, 72, 3, None),
    (1, 700, 2, 256, 2, None),
    (5, 1, 40, 128, 3, [16, 24, 24]),
    (1, 3, 2, 512, 1, [256]),
    (1, 3, 2, 700, 2, [100, 150]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_formula(shape, interleaved, dtype):
    N, L, H, D, axes, sections = shape
    x, at = make(N, L, H, D, axes, dtype)
    compare(x, at, sections, interleaved)
    compare(x, at, sections, interleaved, base=100.0, key=make(N, L, max(1, H // 2), D, 1, dtype, seed=1)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("kind,far", [(torch.int32, 2 ** 31 - 1), (torch.int64, 2 ** 31), (torch.float32, 3e7), (torch.float32, 1e-3)])
def test_far_and_near_positions(kind, far):
    x, _ = make(2, 60, 2, 64, 1, torch.float32)
    g = torch.Generator().manual_seed(3)
    at = ((torch.rand(2, 60, 2, generator=g, dtype=torch.float64) - 0.5) * 2 * far).to(kind)
    at[0, 0] = 0
    at[0, 1] = int(far) if kind != torch.float32 else far
    compare(x, at, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides(dtype, interleaved):
    """Parts of a projection's rows, heads before tokens, rows at odd addresses, expanded and transposed positions and gradients."""
    rows, _ = make(2, 30, 12, 64, 1, dtype, seed=4)
    at = torch.randint(0, 500, (30, 3), generator=torch.Generator().manual_seed(5)).expand(2, 30, 3)
    q, k, _ = rows.cuda().split([8, 2, 2], 2)
    a, b = rotary_positions(q, at.cuda(), k, interleaved=interleaved)
    check(a, *reference(rows[:, :, :8], at, even(64, 3), 1e4, interleaved), "query")
    check(b, *reference(rows[:, :, 8:10], at, even(64, 3), 1e4, interleaved), "key")
    turned = rows.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    places = at.contiguous().permute(2, 0, 1).contiguous().permute(1, 2, 0).cuda()
    want, bound = reference(rows, at, even(64, 3), 1e4, interleaved)
    check(rotary_positions(turned, places, interleaved=interleaved), want, bound, "transposed")
    odd = torch.cat([rows.flatten()[:1], rows.flatten()]).cuda()[1:].view(rows.shape)
    assert odd.data_ptr() % 16
    check(rotary_positions(odd, places, interleaved=interleaved), want, bound, "odd address")
    apart = torch.stack([rows, rows], -1).cuda()[..., 0]
    check(rotary_positions(apart, places, interleaved=interleaved), want, bound, "columns apart")
    leaf = rows.cuda().requires_grad_()
    one = torch.ones((), dtype=dtype, device="cuda").expand(rows.shape)
    grad, = torch.autograd.grad(rotary_positions(leaf, places, interleaved=interleaved), leaf, one)
    check(grad, *reference(torch.ones_like(rows), at, even(64, 3), 1e4, interleaved, -1), "gradient")


@pytest.mark.gpu
def test_one_of_two_gradients():
    x, at = make(2, 5, 4, 16, 1, torch.float32)
    for which in (0, 1):
        leaves = [x.cuda(), x.cuda()[:, :, :2]]
        leaves[which].requires_grad_()
        out = rotary_positions(leaves[0], at.cuda(), leaves[1])
        grad, = torch.autograd.grad(out[which].sum(), leaves[which])
        check(grad, *reference(torch.ones(leaves[which].shape), at, [8], 1e4, False, -1), "gradient")
    both = [t.cuda().requires_grad_() for t in (x, x)]
    out = rotary_positions(both[0], at.cuda(), both[1])
    assert torch.autograd.grad(out[1].sum(), both, allow_unused=True)[0] is None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_products_depend_on_distances(dtype):
    """What the operator is for: products of turned queries and keys at places that differ by as much are alike, to the rounding of the turned
    values (2 u of |q||k|, and angles' 16 e)."""
    q, k = (torch.randn(64, generator=torch.Generator().manual_seed(s)).to(dtype).cuda() for s in (0, 1))
    at = torch.tensor([[[3, 40, 7]], [[3 + 5, 40 - 17, 7 + 100]], [[100003, 90040, 50007]], [[100003 + 5, 90040 - 17, 50007 + 100]]], device="cuda")
    x = torch.stack([q, k, q, k]).view(4, 1, 1, 64)
    y = rotary_positions(x, at).double().view(4, 64)
    assert abs(float(y[0] @ y[1] - y[2] @ y[3])) <= 4 * (2 * HALF[dtype] + 16 * E) * float(q.double().norm() * k.double().norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_what_is_not_finite_stays_in_its_pair(dtype):
    x, at = make(1, 4, 2, 16, 1, dtype)
    want = rotary_positions(x.cuda(), at.cuda())
    x[0, 1, 0, 3], x[0, 2, 1, 12] = math.nan, math.inf
    got = rotary_positions(x.cuda(), at.cuda())
    bad = torch.zeros(1, 4, 2, 16, dtype=torch.bool)
    bad[0, 1, 0, [3, 11]] = bad[0, 2, 1, [4, 12]] = True
    assert torch.equal(got.cpu()[~bad], want.cpu()[~bad]) and not bool(got.cpu()[bad].isfinite().any())


@pytest.mark.gpu
def test_streams_graphs_and_empty_inputs():
    x, at = make(2, 100, 4, 64, 2, torch.bfloat16)
    x, at = x.cuda(), at.cuda()
    want = rotary_positions(x, at)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = rotary_positions(x, at)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    leaf, grad = x.clone().requires_grad_(), torch.randn_like(x)
    torch.autograd.grad(rotary_positions(leaf, at), leaf, grad)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary_positions(leaf, at)
        back, = torch.autograd.grad(out, leaf, grad)
    for k in range(2):
        at.add_(1000 * k)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, rotary_positions(x, at))
        assert float((rotary_positions(back, at) - grad).abs().max()) <= 8 * HALF[torch.bfloat16] * float(grad.abs().max())
    for shape in ((0, 3, 2, 16), (2, 0, 2, 16)):
        y = torch.zeros(shape, device="cuda")
        assert rotary_positions(y, torch.zeros(*shape[:2], 3, device="cuda")).shape == shape


@pytest.mark.gpu
def test_places_beyond_32_bits():
    N, L, H, D = 2, 2 ** 17 + 3, 128, 128
    x = torch.ones(1, 1, H, D, dtype=torch.float16, device="cuda").expand(N, L, H, D)
    at = torch.zeros(N, L, 1, device="cuda")
    at[-1, -1] = 5.0
    out = rotary_positions(x, at)
    assert out.numel() > 2 ** 32 and bool((out[0, ::1000] == 1).all())
    check(out[-1:, -1:], *reference(x[-1:, -1:], at[-1:, -1:], [64], 1e4, False), "last")


@pytest.mark.gpu
def test_a_gradient_of_the_gradient_is_refused():
    x, at = make(1, 4, 1, 8, 1, torch.float32)
    leaf = x.cuda().requires_grad_()
    g = torch.ones_like(leaf, requires_grad=True)
    grad, = torch.autograd.grad(rotary_positions(leaf, at.cuda()), leaf, g, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        grad.sum().backward()


def test_refusals():
    x, at = make(2, 3, 4, 16, 3, torch.float32)
    with pytest.raises(RuntimeError, match="rotary_positions is not implemented on CPU"):
        rotary_positions(x, at)
    with pytest.raises(RuntimeError, match="not implemented for 'float64'"):
        rotary_positions(x.double(), at)
    with pytest.raises(RuntimeError, match="expected query"):
        rotary_positions(x[0], at)
    with pytest.raises(RuntimeError, match="expected scalar type"):
        rotary_positions(x, at, x.half())
    with pytest.raises(RuntimeError, match="images, states and head size"):
        rotary_positions(x, at, x[..., :8])
    for bad in (at[0], at[:1], at[:, :2]):
        with pytest.raises(RuntimeError, match="positions must be \\(images, states, axes\\)"):
            rotary_positions(x, bad)
    with pytest.raises(RuntimeError, match="float32, int32 or int64"):
        rotary_positions(x, at.double())
    with pytest.raises(RuntimeError, match="1 to 4 axes"):
        rotary_positions(x, torch.zeros(2, 3, 5))
    with pytest.raises(RuntimeError, match="no gradient of positions"):
        rotary_positions(x, at.clone().requires_grad_())
    for sections in ([8], [1, 2, 3, 4, 5]):
        with pytest.raises(RuntimeError, match="one element per axis"):
            rotary_positions(x, at, sections=sections)
    for sections in ([3, 3, 3], [-1, 2, 2], [2 ** 40, 0, 0]):
        with pytest.raises(RuntimeError, match="half of the head size"):
            rotary_positions(x, at, sections=sections)
    with pytest.raises(RuntimeError, match="at most 256 pairs"):
        rotary_positions(torch.zeros(2, 3, 1, 600), at)
    for base in (0.0, -1.0, 0.99, math.inf, math.nan):
        with pytest.raises(RuntimeError, match="base must be"):
            rotary_positions(x, at, base=base)
    with pytest.raises(TypeError):
        rotary_positions(x, at, sections=5)
    with pytest.raises(TypeError):
        rotary_positions(x, at, sections=[1.5, 1, 1])


def test_the_library_refuses_before_it_launches():
    def call(**kw):
        a = _lib.Rotary(dtype=0, axes=1, N=1, L=1, D=8, base=1e4)
        a.heads[0], a.sections[0] = 1, 4
        for k, v in kw.items():
            if k in ("heads", "sections"):
                getattr(a, k)[0] = v
            else:
                setattr(a, k, v)
        return _lib.lib.mvr_rotary_positions(a, None)
    assert _lib.lib.mvr_rotary_positions(None, None) == -6 and call() == -6
    assert call(dtype=2) == call(position_dtype=6) == -1
    assert call(heads=0) == call(D=0) == call(N=-1) == -5
    assert call(axes=0) == call(axes=5) == call(sections=5) == call(sections=-1) == call(base=0.0) == call(base=math.nan) == -22
    assert call(sections=257, D=600) == -16 and call(L=2 ** 31) == -9
    assert call(N=0) == 0
