"""ops.label_log_probs against its definition in float64: both layouts, labels that are not given, equal scores, infinities, the
gradient, and what it refuses.

Tolerances.  e = 2^-24.  log sum exp of K scores in float: the running sums are off by sqrt(K) roundings of random sign (8 sqrt(K) e
covers six standard deviations, the functions' ulps and the shifts of the maximum), the difference x - lse by one rounding of a number
of its size: (8 sqrt(K) + 4 + |x - lse| + |max|) e.  Entropy: a weighted mean of such differences.  A gradient is such a weight times
a + b (log p + H), off relatively by twice that, and rounded once to the scores' type."""
import math

import pytest
import torch

from medvision_b200.ops import label_log_probs

E = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def reference(x, y, top, a=None, b=None):
    """x (N, K, ...) float64, y (N, ...) int64: log_prob, entropy, values and classes of the alternatives, gradient."""
    K = x.shape[1]
    logs = torch.log_softmax(x, 1)
    given = (y >= 0) & (y < K)
    lp = torch.where(given, logs.gather(1, torch.where(given, y, 0).unsqueeze(1)).squeeze(1), 0.0)
    p = logs.exp()
    plogs = torch.where(p == 0, 0.0, p * logs)
    h = -plogs.sum(1)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    grad = None
    if a is not None:
        a = torch.where(given, a, 0.0).unsqueeze(1)
        grad = -(p * a + b.unsqueeze(1) * (plogs + p * h.unsqueeze(1)))
        grad = grad.scatter_add(1, torch.where(given, y, 0).unsqueeze(1), a)
    return lp, h, logs.gather(1, order), order, grad


def check(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | ((got != got) & (want != want))
    bad = ~(same | ((got - want).abs() <= bound))
    assert not bool(bad.any()), "%s: %d of %d beyond the bound" % (what, int(bad.sum()), got.numel())


def compare(x, labels, top, y=None, seed=0, scale_of_gradients=1.0):
    """x as the user passes it (any layout, on the GPU), labels on the GPU."""
    dtype, K = x.dtype, x.shape[1]
    xd = x.detach().cpu().double()
    y = (labels if y is None else y).cpu().long().reshape((x.shape[0],) + tuple(x.shape[2:]))
    g = torch.Generator().manual_seed(seed)
    a, b = (torch.randn(y.shape, generator=g) * scale_of_gradients for _ in range(2))
    lp, h, tv, tc, grad = reference(xd, y, top, a.double(), b.double())
    leaf = x.detach().requires_grad_()
    got = label_log_probs(leaf, labels, top)
    assert got.log_prob.shape == labels.shape and got.entropy.shape == labels.shape
    big = xd.abs().where(xd.isfinite(), torch.zeros(())).amax(1) if K else 0
    e = (8 * math.sqrt(K) + 4 + 2 * big) * E
    check(got.log_prob.reshape(y.shape), lp, e + 4 * E * lp.abs(), "log_prob")
    check(got.entropy.reshape(y.shape), h, 2 * e * (1 + h.abs()), "entropy")
    if top:
        assert torch.equal(got.top_label.cpu().long(), tc)
        assert got.top_label.dtype == torch.int32 and not got.top_log_prob.requires_grad
        check(got.top_log_prob, tv, e.unsqueeze(1) + 4 * E * tv.abs(), "top")
    else:
        assert got.top_label is None and got.top_log_prob is None
    gx, = torch.autograd.grad((got.log_prob, got.entropy), leaf, (a.cuda().view(labels.shape), b.cuda().view(labels.shape)))
    assert gx.dtype == dtype
    p = torch.softmax(xd, 1)
    logp = torch.log_softmax(xd, 1).where(p > 0, torch.zeros(()))
    size = p * (a.unsqueeze(1).abs() + b.unsqueeze(1).abs() * (logp.abs() + h.unsqueeze(1) + 1))
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    check(gx, grad, HALF[dtype] * grad.abs() + 4 * e.unsqueeze(1) * (1 + logp.abs()) * size + 2 * E * a.unsqueeze(1).abs() + tiny, "gradient")
    return got


def scores(shape, dtype, seed=0, scale=3.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,K,top", [(1, 1, 1), (5, 2, 0), (3, 31, 16), (9, 81, 5), (2, 1024, 16), (7, 1025, 8), (3, 4099, 1), (2, 33000, 16), (130, 17, 3), (1, 140001, 4)])
def test_rows(dtype, rows, K, top):
    y = torch.randint(-1, K + 1, (rows,), generator=torch.Generator().manual_seed(1))
    compare(scores((rows, K), dtype).cuda(), y.int().cuda(), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape,top", [((2, 3, 5, 7), 2), ((1, 14, 4, 6, 8), 3), ((3, 2, 64), 1), ((2, 33, 10, 12), 16), ((1, 5, 1, 301), 5),
                                       ((2, 1, 9), 0), ((2, 9, 256), 2), ((1, 70, 3, 4), 0)])
@pytest.mark.parametrize("labels", [torch.uint8, torch.int16, torch.int32, torch.int64])
def test_maps(dtype, shape, top, labels):
    K = shape[1]
    y = torch.randint(0, K + 1, (shape[0],) + shape[2:], generator=torch.Generator().manual_seed(2)).to(labels)
    if labels != torch.uint8:
        y[y == K] = -100
    x = scores(shape, dtype)
    compare(x.cuda(), y.cuda(), top)
    compare(x.cuda(), y.unsqueeze(1).cuda(), top)          # (N, 1, ...), as label fields are


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_layouts(dtype):
    K, top = 37, 4
    x = scores((3, K, 6, 10), dtype).cuda()
    y = torch.randint(0, K, (3, 6, 10), generator=torch.Generator().manual_seed(3)).cuda()
    want = compare(x, y, top)
    last = x.contiguous(memory_format=torch.channels_last)
    wide = torch.zeros((3, K + 3, 6, 10), dtype=dtype, device="cuda")
    wide[:, 2:K + 2] = x
    gaps = torch.zeros((3, K, 6, 11), dtype=dtype, device="cuda")
    gaps[..., :10] = x
    for other in (last, wide[:, 2:K + 2], gaps[..., :10], x.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(other, x)
        compare(other, y, top)
        assert torch.equal(label_log_probs(other, y, top).top_label, want.top_label)
    rows = scores((9, 2050), dtype, 4).cuda()
    padded = torch.zeros((9, 2057), dtype=dtype, device="cuda")
    padded[:, 1:2051] = rows
    y = torch.arange(9).cuda() * 200
    for other in (rows, padded[:, 1:2051], rows.t().contiguous().t()):
        compare(other, y, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [40, 3000])
@pytest.mark.parametrize("rows", [True, False])
def test_equal_scores_go_to_the_lowest_class(K, rows):
    x = torch.zeros(4, K)
    x[1] = torch.randint(0, 3, (K,), generator=torch.Generator().manual_seed(5)).float()
    x[2, 7:] = 1.5
    x[3] = -torch.arange(K).float() // 4
    y = torch.tensor([0, 3, 9, 5])
    if not rows:
        x, y = x.t().reshape(1, K, 2, 2).contiguous(), y.view(1, 2, 2)
    for dtype in HALF:
        for top in (1, 2, 5, 16):
            compare(x.to(dtype).cuda(), y.cuda(), top)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [21, 2000])
@pytest.mark.parametrize("rows", [True, False])
@pytest.mark.parametrize("dtype", HALF)
def test_infinities(K, rows, dtype):
    inf = float("inf")
    x = scores((5, K), dtype, 6)
    x[0, ::2] = -inf                   # classes that cannot be
    x[1, 1:] = -inf                    # a single one that can
    x[3, : K - 2] = -inf
    y = torch.tensor([2, 0, 3, K - 1, 4])
    a = x if rows else x.t().reshape(1, K, 5).contiguous()
    b = y if rows else y.view(1, 5)
    compare(a.cuda(), b.cuda(), 2)     # row 0: the label's probability is 0
    x = scores((3, K), dtype, 7)
    x[0] = -inf
    x[1, K // 2] = float("nan")
    x[2, 3] = inf
    y = torch.tensor([1, -1, 3])
    a = (x if rows else x.t().reshape(1, K, 3).contiguous()).cuda().requires_grad_()
    b = (y if rows else y.view(1, 3)).cuda()
    got = label_log_probs(a, b, 2)
    lp, h = got.log_prob.detach().flatten(), got.entropy.detach().flatten()
    assert float(lp[0]) == -inf and float(h[0]) == 0
    assert float(lp[1]) == 0 and bool(h[1].isnan())  # no label is given
    assert bool(lp[2].isnan()) and bool(h[2].isnan())
    first = (got.top_label if rows else got.top_label[0].t()).cpu()
    assert first[0].tolist() == [0, 1] and int(first[1, 0]) == K // 2 and int(first[2, 0]) == 3
    g, = torch.autograd.grad((got.log_prob, got.entropy), a, (torch.ones_like(got.log_prob), torch.ones_like(got.entropy)))
    g = g if rows else g[0].t()
    assert not bool(g[0].any()) and bool(g[1].isnan().any())


@pytest.mark.gpu
def test_far_scores_and_large_offsets():
    """Scores of one size far from 0: only their differences count."""
    x = scores((6, 50), torch.float32, 8) + 4096.0
    y = torch.arange(6)
    compare(x.cuda(), y.cuda(), 3)
    compare(x.t().reshape(1, 50, 6).contiguous().cuda(), y.view(1, 6).cuda(), 3)
    x[:, 10] += 300  # one class has all the probability
    compare(x.cuda(), y.cuda(), 3)


@pytest.mark.gpu
def test_gradient_agrees_with_differences_and_each_output_alone():
    x = scores((4, 9, 5), torch.float32, 9, 1.0).cuda().requires_grad_()
    y = torch.randint(-1, 9, (4, 5), generator=torch.Generator().manual_seed(10)).cuda()
    g = torch.Generator().manual_seed(11)
    a, b = (torch.randn(4, 5, generator=g).cuda() for _ in range(2))
    got = label_log_probs(x, y)
    both, = torch.autograd.grad((got.log_prob, got.entropy), x, (a, b), retain_graph=True)
    ga, = torch.autograd.grad(got.log_prob, x, a, retain_graph=True)
    gb, = torch.autograd.grad(got.entropy, x, b)
    torch.testing.assert_close(ga + gb, both, rtol=0, atol=2.0 ** -20)  # numbers up to some 4, three roundings each
    d, h = torch.randn(x.shape, generator=g).cuda(), 2.0 ** -6

    def f(s):
        r = label_log_probs(x.detach() + s * h * d, y)
        return float((r.log_prob.double() * a).sum() + (r.entropy.double() * b).sum())

    slope = (8 * (f(1) - f(-1)) - (f(2) - f(-2))) / (12 * h)
    # 40 float values of size up to 8 in f: 40 * 8 * 2^-24 * 4 each; fourth order in h
    assert abs(slope - float((both.double() * d).sum())) <= 18 * 40 * 32 * E / (12 * h) + 500 * h ** 4


@pytest.mark.gpu
def test_empty_and_graphs():
    for shape in [(0, 5), (2, 5, 0), (0, 5, 3)]:
        r = label_log_probs(torch.zeros(shape).cuda().requires_grad_(), torch.zeros((shape[0],) + shape[2:], dtype=torch.int32).cuda(), 2)
        assert r.log_prob.shape == (shape[0],) + shape[2:] and r.top_label.shape == (shape[0], 2) + shape[2:]
        r.log_prob.sum().backward()
    x = scores((70, 1500), torch.float16).cuda().requires_grad_()
    y = torch.arange(70).cuda()
    torch.autograd.grad(label_log_probs(x, y, 3).log_prob.sum(), x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = label_log_probs(x, y, 3)
        g, = torch.autograd.grad(r.log_prob.sum() + r.entropy.sum(), x)
    with torch.no_grad():
        x.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    fresh = label_log_probs(x, y, 3)
    assert all(torch.equal(a, b) for a, b in zip(r, fresh))
    assert torch.equal(g, torch.autograd.grad(fresh.log_prob.sum() + fresh.entropy.sum(), x)[0])


@pytest.mark.gpu
def test_many_items_and_positions_beyond_one_launch():
    x = scores((40000, 3, 2), torch.float16, 12)
    y = torch.randint(-1, 3, (40000, 2), generator=torch.Generator().manual_seed(13))
    compare(x.cuda(), y.cuda(), 1)
    n = 2 ** 30 + 6                                # a launch takes 2^30 positions; outputs pass 2^32 bytes
    x = torch.zeros(1, 2, n, dtype=torch.float16, device="cuda")
    x[0, 1, -8:] = torch.arange(8).half().cuda()
    y = torch.zeros(1, n, dtype=torch.uint8, device="cuda")
    y[0, -3:] = 1
    leaf = x.requires_grad_()
    got = label_log_probs(leaf, y, 1)
    lp, h, tv, tc, _ = reference(x[..., -8:].detach().cpu().double(), y[:, -8:].cpu().long(), 1)
    check(got.log_prob[:, -8:], lp, 64 * E, "log_prob")
    check(got.entropy[:, -8:], h, 64 * E, "entropy")
    assert torch.equal(got.top_label[..., -8:].cpu().long(), tc)
    g, = torch.autograd.grad(got.log_prob, leaf, torch.ones_like(got.log_prob))
    want = torch.nn.functional.one_hot(y[0, -8:].cpu().long(), 2).t() - torch.softmax(x[0, :, -8:].detach().cpu().double(), 0)
    check(g[0, :, -8:], want, 2.0 ** -11, "gradient")
    assert bool((g[0, 0, :4] == 0.5).all())


def test_refusals():
    x, y = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="label_log_probs is not implemented on CPU"):
        label_log_probs(x, y)
    with pytest.raises(RuntimeError, match="not implemented for 'float64'"):
        label_log_probs(x.double(), y)
    with pytest.raises(RuntimeError, match="not implemented for labels of type 'float32'"):
        label_log_probs(x, y.float())
    with pytest.raises(RuntimeError, match="labels must be"):
        label_log_probs(x, y[:2])
    with pytest.raises(RuntimeError, match="labels must be"):
        label_log_probs(x.view(3, 5, 1), torch.zeros(3, 2, 1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="expected class scores"):
        label_log_probs(x[0], y)
    with pytest.raises(RuntimeError, match="a class at least"):
        label_log_probs(x[:, :0], y)
    for top in (-1, 6, 17):
        with pytest.raises(RuntimeError, match="top must be between 0 and 16"):
            label_log_probs(x if top < 17 else torch.zeros(3, 50), y, top)


def test_c_entry_checks_before_any_cuda_call():
    from medvision_b200 import _lib
    f, b = _lib.lib.mvr_label_log_probs_forward, _lib.lib.mvr_label_log_probs_backward

    def fwd(x=16, dtype=0, label_dtype=2, batch=2, classes=4, space=1, top=0, out=16, best=16):
        return f(x, dtype, 16, label_dtype, out, 16, None, best, best, batch, classes, space, classes, 1, top, None)
    assert fwd(dtype=2) == -1 and fwd(label_dtype=4) == -1 and fwd(batch=-1) == -5 and fwd(classes=0) == -5
    assert fwd(classes=2 ** 31) == -9 and fwd(top=5) == -18 and fwd(top=-1) == -18 and fwd(classes=40, top=17) == -18
    assert fwd(x=None) == -6 and fwd(out=None) == -6 and fwd(top=1, best=None) == -6 and fwd(batch=0, x=None) == 0
    assert b(16, 0, 16, 2, None, 16, None, None, 16, 2, 4, 1, 4, 1, 4, 1, None) == -6
    assert b(16, 5, 16, 2, 16, 16, None, None, 16, 2, 4, 1, 4, 1, 4, 1, None) == -1
