"""ops.group_norm against its formula in float64: forward and gradients over groups, shapes, types and activations, statistics far from 0,
what is not finite, other streams and graphs, and what it refuses.

Tolerances.  u: half a step of the type, e = 2^-24, m: values of a group.  Sums of n terms in float have errors that grow with the square
root, 8 sqrt(n) e of their size covers six standard deviations.
  r = 8 sqrt(m) e:  relative error of the deviation;  mean:  r std + 4 e |mean|
  xhat:  dh = |xhat| (r + 4 e) + (r + 4 e |mean| rstd + e |xhat|);   z:  dz = |w| dh + 2 e (|z| + |b|)
  y:     1.2 dz + a |y| + u |y|          (slopes of the activations are below 1.2; a: their own error, 16 e, in half types 2^-18)
  slope: its own is below 1.2 again:  ds = |dy| (1.2 dz + 2 a); a relu's is exact, but may be either where |z| <= dz
  db, dw:  sum ds, sum (ds |xhat| + |s| dh), and 8 sqrt(n) e of the terms' sizes
  dx:    rstd (|w| ds + mean's errors + |xhat| m2's error + |m2| dh + 4 e of the terms) + (r + 4 e + u) |dx|
float16 adds its smallest step 2^-25.
"""
import ctypes
import math

import pytest
import torch

from medvision_b200 import _lib
from medvision_b200.ops import GroupNorm, group_norm

from test_cross_attention import E, HALF, check

ACTS = [None, "relu", "silu", "gelu"]


def act(z, kind):
    """act(z), act'(z) in float64."""
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double()
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if kind == "gelu":
        p = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def reference(x, groups, weight, bias, dy, kind, eps=1e-5, parameter=torch.float32):
    """(value, bound) of y, dx, dweight, dbias."""
    dtype = x.dtype
    u, tiny = HALF[dtype], 2.0 ** -25 if dtype == torch.float16 else 0.0
    x, dy = x.detach().cpu().double(), dy.detach().cpu().double()
    shape, (N, C) = x.shape, (x.shape[0], x.shape[-1])
    x, dy = x.reshape(N, -1, groups, C // groups), dy.reshape(N, -1, groups, C // groups)
    w = (torch.ones(C) if weight is None else weight.detach().cpu()).double().view(groups, -1)
    b = (torch.zeros(C) if bias is None else bias.detach().cpu()).double().view(groups, -1)
    S, m = x.shape[1], x.shape[1] * x.shape[3]
    mean = x.mean((1, 3), keepdim=True)
    rstd = (((x - mean) ** 2).mean((1, 3), keepdim=True) + eps) ** -0.5
    h = (x - mean) * rstd
    z = h * w + b
    y, slope = act(z, kind)
    a = 16 * E if dtype == torch.float32 else 2.0 ** -18
    r = 8 * math.sqrt(m) * E
    eh = h.abs() * (r + 4 * E) + (r + 4 * E * mean.abs() * rstd + E * h.abs())
    ez = w.abs() * eh + 2 * E * (z.abs() + b.abs())
    ey = 1.2 * ez + (a + u) * y.abs() + tiny
    s = dy * slope
    es = dy.abs() * ((z.abs() <= ez).double() if kind == "relu" else 1.2 * ez + 2 * a if kind else 0.0)
    n = 8 * math.sqrt(N * S) * E
    up = HALF[parameter]
    dw, db = (s * h).sum((0, 1)), s.sum((0, 1))
    tp = 2.0 ** -25 if parameter == torch.float16 else 0.0
    edw = (es * h.abs() + s.abs() * eh).sum((0, 1)) + n * (s * h).abs().sum((0, 1)) + up * dw.abs() + tp
    edb = es.sum((0, 1)) + n * s.abs().sum((0, 1)) + up * db.abs() + tp
    avg = lambda t: t.mean((1, 3), keepdim=True)  # noqa: E731
    m1, m2 = avg(s * w), avg(s * w * h)
    e1 = avg(es * w.abs()) + r * avg((s * w).abs())
    e2 = avg((es * h.abs() + s.abs() * eh) * w.abs()) + r * avg((s * w * h).abs())
    dx = rstd * (s * w - m1 - h * m2)
    ex = rstd * (w.abs() * es + e1 + h.abs() * e2 + m2.abs() * eh + 4 * E * ((s * w).abs() + m1.abs() + (h * m2).abs())) + (r + 4 * E + u) * dx.abs() + tiny
    return [t.reshape(shape) for t in (y, dx)] + [dw.reshape(C), db.reshape(C)], [t.reshape(shape) for t in (ey, ex)] + [edw.reshape(C), edb.reshape(C)]


def make(shape, dtype, seed=0, offset=0.0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = torch.randn(shape, generator=g) * (torch.rand(C, generator=g) + 0.5) * spread + torch.randn(C, generator=g) * spread + offset
    return x.to(dtype), 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g), torch.randn(shape, generator=g).to(dtype)


def run(x, groups, weight, bias, dy, kind, **kw):
    leaves = [t.cuda().requires_grad_() for t in (x, weight, bias)]
    y = group_norm(leaves[0], groups, leaves[1], leaves[2], activation=kind, **kw)
    return (y,) + torch.autograd.grad(y, leaves, dy.cuda())


NAMES = "y", "dx", "dw", "db"
SHAPES = [  # shape, groups
    ((1, 1, 16), 1),
    ((1, 16), 2),
    ((2, 3, 8), 2),
    ((2, 5, 6, 7, 12), 3),        # rows of 24 bytes
    ((3, 211, 33), 11),           # odd rows
    ((2, 1000, 64), 8),
    ((1, 5000, 8), 8),            # one channel a group
    ((2, 777, 84), 7),
    ((1, 3, 2600), 1),
    ((2, 7, 5000), 1),            # a group of more vectors than a CTA has threads
    ((1, 200, 9000), 3),
    ((1, 5, 8008), 8),            # vectors over two groups, and more of them than threads
    ((2, 9, 4100), 4),
    ((1, 40, 2056), 257),
    ((300, 49, 32), 4),           # many small images
    ((2, 4097, 320), 32),
    ((1, 70000, 20), 2),          # passes: too large for shared memory
    ((2, 60001, 64), 1),
    ((1, 9000, 5), 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind", ACTS)
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_against_the_formula(shape, groups, kind, dtype):
    args = make(shape, dtype)
    want, bound = reference(args[0], groups, *args[1:], kind)
    for name, a, b, c in zip(NAMES, run(args[0], groups, *args[1:], kind), want, bound):
        check(a, b, c, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape,groups", [((2, 300, 24), 3), ((1, 80000, 16), 2), ((2, 9, 640), 5), ((1, 20000, 7), 7)])
def test_parameters_in_the_inputs_type_and_left_out(shape, groups, dtype):
    x, w, b, dy = make(shape, dtype, seed=1)
    w, b = w.to(dtype), b.to(dtype)
    want, bound = reference(x, groups, w, b, dy, "silu", parameter=dtype)
    got = run(x, groups, w, b, dy, "silu")
    assert got[2].dtype == got[3].dtype == dtype
    for name, a, c, e in zip(NAMES, got, want, bound):
        check(a, c, e, name)
    for keep_w, keep_b in ((True, False), (False, True), (False, False)):
        want, bound = reference(x, groups, w if keep_w else None, b if keep_b else None, dy, "gelu", parameter=dtype)
        leaves = [t.cuda().requires_grad_() if keep else None for t, keep in ((x, True), (w, keep_w), (b, keep_b))]
        y = group_norm(leaves[0], groups, leaves[1], leaves[2], activation="gelu")
        got = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], dy.cuda()))
        check(y, want[0], bound[0], "y")
        for i, leaf in enumerate(leaves):
            if leaf is not None:
                check(next(got), want[i + 1], bound[i + 1], NAMES[i + 1])


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((2, 500, 32), 4), ((1, 100000, 12), 3)])
def test_statistics_far_from_zero(shape, groups):
    """Air at -1000 with a deviation of 1, and first values that are not typical of what follows."""
    for offset, spread in ((-1000.0, 1.0), (1e5, 2.0)):
        args = make(shape, torch.float32, seed=2, offset=offset, spread=spread)
        want, bound = reference(args[0], groups, *args[1:], None)
        for name, a, b, c in zip(NAMES, run(args[0], groups, *args[1:], None), want, bound):
            check(a, b, c, name)
    x, w, b, dy = make(shape, torch.float32, seed=3, offset=-1000.0)
    x[:, :40] = 0.0
    want, bound = reference(x, groups, w, b, dy, "silu")
    check(run(x, groups, w, b, dy, "silu")[0], want[0], bound[0], "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_constant_groups_and_values_that_are_not_finite(dtype):
    x = torch.full((2, 50, 16), 3.0, dtype=dtype)
    w, b = torch.full((16,), 2.0), torch.arange(16.0) / 8
    y, dx, dw, db = run(x, 4, w, b, torch.ones_like(x), None)
    assert torch.equal(y.cpu(), b.to(dtype).expand(2, 50, 16)) and not bool(dx.any()) and not bool(dw.any()) and bool((db == 100).all())
    for bad in (math.nan, math.inf, -math.inf):  # one group of one image is spoilt, no other
        x, w, b, dy = make((2, 50, 16), dtype, seed=4)
        clean = run(x, 4, w, b, dy, "silu")
        x[1, 7, 5] = bad
        got = run(x, 4, w, b, dy, "silu")
        same = torch.ones(2, 50, 16, dtype=torch.bool)
        same[1, :, 4:8] = False
        for i in (0, 1):
            assert torch.equal(got[i].cpu()[same], clean[i].cpu()[same]) and bool(got[i].cpu()[~same].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ACTS)
def test_large_arguments_of_the_activations(kind):
    b = torch.tensor([-1e4, -100.0, -30.0, 30.0, 100.0, 1e4, -3e38, 3e38])
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.zeros(1, 4, 8, dtype=dtype)
        leaf = x.cuda().requires_grad_()
        y = group_norm(leaf, 1, None, b.cuda(), activation=kind)
        want = act(b.double(), kind)[0]
        assert torch.allclose(y.cpu().double(), want.expand(1, 4, 8), rtol=2 * HALF[dtype] + 64 * E, atol=1e-10)
        assert bool(torch.autograd.grad(y, leaf, torch.ones_like(y))[0].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_views(dtype):
    x, w, b, dy = make((2, 6, 5, 4, 24), dtype, seed=5)
    want = run(x, 3, w, b, dy, "silu")
    maps = x.permute(0, 4, 1, 2, 3).contiguous(memory_format=torch.channels_last_3d).cuda()  # (N, C, D, H, W)
    got = group_norm(maps.permute(0, 2, 3, 4, 1), 3, w.cuda(), b.cuda(), activation="silu")
    assert torch.equal(got, want[0])
    odd = torch.cat([x.flatten()[:1], x.flatten()]).cuda()[1:].view(x.shape)  # not 16-byte aligned
    assert odd.data_ptr() % 16
    leaf = odd.requires_grad_()
    got = group_norm(leaf, 3, w.cuda(), b.cuda(), activation="silu")
    ref, bound = reference(x, 3, w, b, dy, "silu")
    check(got, ref[0], bound[0], "y")
    check(torch.autograd.grad(got, leaf, dy.cuda())[0], ref[1], bound[1], "dx")
    wide = torch.randn(2, 120, 48).to(dtype).cuda()
    assert torch.equal(group_norm(wide[..., :24], 3), group_norm(wide[..., :24].contiguous(), 3))
    one = group_norm(x.cuda().requires_grad_(), 3)
    g, = torch.autograd.grad(one, one.grad_fn.next_functions[0][0].variable, torch.ones((), dtype=dtype, device="cuda").expand(x.shape))
    assert bool(g.isfinite().all())


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences along random directions with step 2^-5: its square times the third derivative stays below 3e-3 of the slope here,
    and the values' rounding is 2^-24 sqrt(values) / step."""
    x, w, b, dy = (t.cuda() for t in make((2, 30, 12), torch.float32, seed=6))
    for kind in (None, "silu", "gelu"):
        grads = run(x, 3, w, b, dy, kind)[1:]
        gen = torch.Generator("cuda").manual_seed(0)
        for i, t in enumerate((x, w, b)):
            d = torch.randn(t.shape, generator=gen, device="cuda")
            d = d / d.norm()
            f = lambda s: float((group_norm(*[v + s * d if v is t else v for v in (x,)], 3, *[v + s * d if v is t else v for v in (w, b)],  # noqa: E731
                                            activation=kind).double() * dy).sum())
            step = 2.0 ** -5
            assert abs((f(step) - f(-step)) / (2 * step) - float((grads[i].double() * d).sum())) <= 3e-3 * float(grads[i].norm()) + 40 * E * float(dy.norm()) / step


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 100, 32), (1, 90000, 32)])
def test_repeatable_streams_and_graphs(shape):
    args = make(shape, torch.float16, seed=7)
    first = run(args[0], 4, *args[1:], "silu")
    for a, b in zip(first, run(args[0], 4, *args[1:], "silu")):
        assert torch.equal(a, b)
    graphs = []
    for seed in (7, 8):
        x, w, b, dy = (t.cuda() for t in make(shape, torch.float16, seed=seed))
        leaves = [t.requires_grad_() for t in (x, w, b)]

        def step(leaves=leaves, dy=dy):
            y = group_norm(leaves[0], 4, *leaves[1:], activation="silu")
            return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            warm = step()
        torch.cuda.current_stream().wait_stream(side)
        if seed == 7:
            for a, b in zip(first, warm):
                assert torch.equal(a, b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got, step, leaves[0]))
    for turn in range(2):
        for graph, got, step, x in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, got, step, x in graphs:
            for a, b in zip(got, step()):
                assert torch.equal(a, b)
            with torch.no_grad():
                x.mul_(1.5)


@pytest.mark.gpu
def test_places_beyond_32_bits():
    """The last rows of 2^32 + 2^16 values: their offsets, and counts of a group beyond 2^24."""
    S, C = 2 ** 26 + 2 ** 10, 64
    x = torch.zeros(1, S, C, dtype=torch.float16, device="cuda")
    x[:, ::2] = 2.0
    x[0, -1, -1] = 6.0
    y = group_norm(x, 2, eps=0.0)
    assert bool((y[0, :8:2] == 1).all()) and bool((y[0, 1:8:2] == -1).all())
    assert bool((y[0, -2] == 1).all()) and bool((y[0, -1, :-1] == -1).all()) and float(y[0, -1, -1]) == 5.0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_empty_inputs(dtype):
    for shape in ((0, 5, 8), (2, 0, 8), (2, 0, 3, 8)):
        x, w, b = torch.zeros(shape, dtype=dtype), torch.ones(8), torch.zeros(8)
        y, dx, dw, db = run(x, 2, w, b, x, "silu")
        assert y.shape == dx.shape == x.shape and not bool(dw.any()) and not bool(db.any())


@pytest.mark.gpu
def test_the_layer():
    layer = GroupNorm(4, 32, activation="silu", device="cuda")
    x = torch.randn(2, 7, 32, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(layer(x), group_norm(x, 4, layer.weight, layer.bias, activation="silu"))
    layer(x).float().sum().backward()
    assert layer.weight.grad is not None and layer.bias.grad is not None
    plain = GroupNorm(4, 32, affine=False)
    assert not list(plain.parameters()) and torch.equal(plain(x), group_norm(x, 4))


@pytest.mark.gpu
def test_a_gradient_of_the_gradient_is_refused():
    x = torch.randn(1, 8, 8, device="cuda", requires_grad=True)
    grad, = torch.autograd.grad(group_norm(x, 2).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        grad.sum().backward()


def test_refusals():
    x = torch.zeros(2, 5, 8)
    with pytest.raises(RuntimeError, match="group_norm is not implemented on CPU"):
        group_norm(x, 2)
    with pytest.raises(RuntimeError, match="not implemented for 'float64'"):
        group_norm(x.double(), 2)
    with pytest.raises(RuntimeError, match="expected \\(images, ..., channels\\)"):
        group_norm(x[0, 0], 2)
    for groups in (0, 3, -2, 16):
        with pytest.raises(RuntimeError, match="must divide"):
            group_norm(x, groups)
    with pytest.raises(RuntimeError, match="a channel at least"):
        group_norm(x[..., :0], 1)
    for eps in (-1.0, math.nan, math.inf, 1e300):
        with pytest.raises(RuntimeError, match="eps must be finite"):
            group_norm(x, 2, eps=eps)
    with pytest.raises(RuntimeError, match="one element per channel"):
        group_norm(x, 2, torch.ones(7))
    with pytest.raises(RuntimeError, match="input's type or float32"):
        group_norm(x, 2, torch.ones(8).half())
    with pytest.raises(RuntimeError, match="of the same type"):
        group_norm(x.half(), 2, torch.ones(8), torch.zeros(8).half())
    with pytest.raises(ValueError, match="activation must be one of"):
        group_norm(x, 2, activation="tanh")
    with pytest.raises(ValueError, match="must divide"):
        GroupNorm(3, 8)
    with pytest.raises(ValueError, match="activation must be one of"):
        GroupNorm(2, 8, activation="tanh")
    with pytest.raises(TypeError):
        group_norm(x, 2.5)


def test_the_library_refuses_before_it_launches():
    lib, size = _lib.lib, ctypes.c_int64()
    good = dict(dtype=1, parameter_dtype=0, activation=2, eps=1e-5, N=1, S=200000, C=64, groups=8)
    assert lib.mvr_group_norm_workspace(_lib.GroupNorm(**good), 0, size) == 0 and size.value > 0
    assert lib.mvr_group_norm_workspace(None, 0, size) == -6 and lib.mvr_group_norm_workspace(_lib.GroupNorm(**good), 0, None) == -6
    for field, value, code in (("dtype", 2, -1), ("parameter_dtype", 3, -1), ("activation", 4, -21), ("groups", 0, -20), ("groups", 5, -20), ("C", 0, -5),
                               ("S", -1, -5), ("eps", -1.0, -5), ("S", 2 ** 60, -9)):
        assert lib.mvr_group_norm_workspace(_lib.GroupNorm(**dict(good, **{field: value})), 1, size) == code, field
    assert lib.mvr_group_norm_forward(_lib.GroupNorm(**good), None, 0, None) == -6
    assert lib.mvr_group_norm_forward(_lib.GroupNorm(**dict(good, x=16, out=16, mean=16, rstd=16)), None, 0, None) == -14
    assert lib.mvr_group_norm_forward(_lib.GroupNorm(**dict(good, S=0)), None, 0, None) == 0
