"""ops.label_log_probs on scores far from 0, whose differences alone count, and near certainty.

Tolerances.  e = 2^-24, s_c the distance of a score from the largest.  A difference of float scores is off by half a step of itself, and a
sum of K exponentials by 8 sqrt(K) e (six standard deviations, the functions' ulps):
  log_prob of c   (8 sqrt(K) + 4 + 2 s_c) e + 4 e |log_prob|        entropy   2 (8 sqrt(K) + 4 + 2 H) e (1 + H)
  gradient        half a step of the result + 4 (8 sqrt(K) + 4 + 2 s_c) e (1 + |log p_c|) p_c (|a| + |b| (|log p_c| + H + 1)) + 2 e |a|
None of them knows how far from 0 the scores are.
"""
import ctypes
import math

import pytest
import torch

from medvision_b200.ops import label_log_probs

from test_label_log_probs import E, HALF, check, reference


def compare(x, labels, top):
    dtype, K = x.dtype, x.shape[1]
    xd = x.detach().cpu().double()
    y = labels.cpu().long()
    g = torch.Generator().manual_seed(0)
    a, b = (torch.randn(y.shape, generator=g) for _ in range(2))
    lp, h, tv, tc, grad = reference(xd, y, top, a.double(), b.double())
    leaf = x.detach().requires_grad_()
    got = label_log_probs(leaf, labels, top)
    root = 8 * math.sqrt(K) + 4
    check(got.log_prob, lp, (root + 6 * lp.abs()) * E, "log_prob")       # (2 s <= 2 |log_prob|)
    check(got.entropy, h, 2 * (root + 2 * h) * E * (1 + h), "entropy")
    if top:
        assert torch.equal(got.top_label.cpu().long(), tc)
        check(got.top_log_prob, tv, (root + 6 * tv.abs()) * E, "top")
    gx, = torch.autograd.grad((got.log_prob, got.entropy), leaf, (a.cuda(), b.cuda()))
    check(gx, grad, gradient_bound(xd, grad, a, b, h, root, dtype), "gradient")


def gradient_bound(xd, grad, a, b, h, root, dtype):
    p, logp = torch.softmax(xd, 1), torch.log_softmax(xd, 1)
    a, b, h = (t.double().unsqueeze(1) for t in (a, b, h))
    far = xd.amax(1, keepdim=True) - xd
    size = p * (a.abs() + b.abs() * (logp.abs() + h + 1))
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    return HALF[dtype] * grad.abs() + 4 * (root + 2 * far) * E * (1 + logp.abs()) * size + 2 * E * a.abs() + tiny


def scores(shape, offset, dtype=torch.float32, seed=0):
    """Spread over a few steps of the type at the offset, at least 1."""
    step = max(1.0, float(abs(offset)) * torch.finfo(dtype).eps * 2)
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * step
    return (x + offset).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [8192.0, -8192.0, 1e6, -1e6, 3e7])
@pytest.mark.parametrize("K,top", [(2, 1), (14, 2), (50, 3), (900, 5), (1500, 3), (5001, 2), (40000, 1)])
def test_offsets_of_rows(K, top, offset):
    x = scores((5, K), offset)
    y = torch.randint(-1, K, (5,), generator=torch.Generator().manual_seed(1))
    compare(x.cuda(), y.cuda(), top)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [8192.0, -8192.0, 1e6, -1e6, 3e7])
@pytest.mark.parametrize("K,top", [(1, 0), (4, 1), (14, 2), (40, 3), (300, 0)])
@pytest.mark.parametrize("space", [(4, 6), (3, 7)])  # pairs of positions, and one at a time
def test_offsets_of_maps(K, top, offset, space):
    x = scores((2, K) + space, offset)
    y = torch.randint(-1, K, (2,) + space, generator=torch.Generator().manual_seed(2))
    compare(x.cuda(), y.cuda(), top)
    compare(x.cuda().contiguous(memory_format=torch.channels_last), y.cuda(), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("K", [14, 3000])
def test_offsets_of_half_scores(K, dtype):
    for offset in (1024.0, -20000.0):
        y = torch.arange(4)
        compare(scores((4, K), offset, dtype).cuda(), y.cuda(), 2)
        compare(scores((1, K, 2, 2), offset, dtype).cuda(), y.view(1, 2, 2).cuda(), 2)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [60, 2000])
@pytest.mark.parametrize("rows", [True, False])
def test_equal_scores_far_from_0_have_equal_probabilities(K, rows):
    """Of K equal scores each has 1 / K; one class only, or many without probability, beside the offset."""
    x = torch.full((4, K), 1e6)
    x[1, 1:] = -float("inf")
    x[2, ::2] = -float("inf")
    x[3] = -float("inf")
    y = torch.tensor([0, 0, 1, 2])
    a, b = (x, y) if rows else (x.t().reshape(1, K, 4).contiguous(), y.view(1, 4))
    leaf = a.cuda().requires_grad_()
    got = label_log_probs(leaf, b.cuda(), 0)
    g, = torch.autograd.grad((got.log_prob, got.entropy), leaf, (torch.ones_like(got.log_prob), torch.zeros_like(got.entropy)))
    g = g.cpu().double() if rows else g[0].t().cpu().double()
    for row, classes in ((0, K), (1, 1), (2, K // 2)):
        want = torch.where(x[row].isfinite(), -1.0 / classes, 0.0).double()
        want[y[row]] += 1
        # (a probability is off by 8 sqrt(K) e and its exponential, relatively; the label's by a rounding of 1)
        assert float((g[row] - want).abs().max()) <= (8 * math.sqrt(K) + 16) * E / classes + 2 * E, row
    assert not bool(g[3].any())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4096, 2), (1, 2, 4096), (4096, 20)])
def test_a_loss_near_certainty(shape):
    """log_prob = -log(1 + r), r between 2^-24 and 2^-9: the sum in float is off by half a step of 1, its logarithm by no more."""
    rest = torch.linspace(-24, -9, 4096) * math.log(2)
    x = torch.full(shape, -200.0)
    if len(shape) == 2:
        x[:, 0], x[:, 1] = 0, rest
        y = torch.zeros(4096, dtype=torch.int64)
    else:
        x[0, 0], x[0, 1] = 0, rest
        y = torch.zeros(1, 4096, dtype=torch.int64)
    got = label_log_probs(x.cuda(), y.cuda(), 1)
    want = torch.log_softmax(x.double(), 1)[:, 0]
    # l = 1 + r: rounded once (2^-24); r itself off by 8 e r; the logarithm's own rounding
    bound = 2.0 ** -24 + 16 * E * want.abs()
    check(got.log_prob, want, bound, "log_prob")
    check(got.top_log_prob[:, 0], want, bound, "top")


@pytest.mark.gpu
@pytest.mark.parametrize("K,space", [(14, 6), (14, 7), (50, 1), (700, 1), (1500, 1)])
def test_large_gradients_and_classes_without_probability(K, space):
    """Gradients scaled by 2^40: a class of probability 0 gets 0 from them, the others their multiples."""
    x = torch.randn(3, K, space, generator=torch.Generator().manual_seed(6))
    x[:, K // 2] = -float("inf")
    x[:, K // 3] = -1e30
    y = torch.randint(-1, K // 3, (3, space), generator=torch.Generator().manual_seed(7))
    leaf = (x if space > 1 else x.squeeze(2)).cuda().requires_grad_()
    got = label_log_probs(leaf, (y if space > 1 else y.squeeze(1)).cuda())
    a, b = (torch.randn(3, space, generator=torch.Generator().manual_seed(8 + i)) * 2.0 ** 40 for i in range(2))
    g, = torch.autograd.grad((got.log_prob, got.entropy), leaf, (a.cuda().view(got.entropy.shape), b.cuda().view(got.entropy.shape)))
    xd = x.double()
    _, h, _, _, grad = reference(xd, y.long(), 0, a.double(), b.double())
    near = xd.where(xd > -1e3, torch.tensor(-60.0, dtype=torch.float64))
    check(g.view(3, K, space), grad, gradient_bound(near, grad, a, b, h, 8 * math.sqrt(K) + 4, torch.float32), "gradient")
    assert not bool(g.view(3, K, space)[:, [K // 2, K // 3]].any())


@pytest.mark.gpu
@pytest.mark.parametrize("K,space", [(14, 6), (14, 7), (50, 1), (700, 1), (1500, 1), (5001, 1)])
@pytest.mark.parametrize("rest", [True, False])
def test_the_c_entries_with_the_rest_of_lse_and_without(K, space, rest):
    """The backward of a caller that keeps lse alone is as near as that of one that keeps what its rounding left too."""
    from medvision_b200 import _lib
    L = _lib.lib
    N, offset = 3, 1e6
    x = scores((N, K, space), offset, seed=3).cuda()
    x[0, K // 3] = -float("inf")
    y = torch.randint(-1, K, (N, space), generator=torch.Generator().manual_seed(4)).int().cuda()
    a, b = (torch.randn(N, space, generator=torch.Generator().manual_seed(5 + i)).cuda() for i in range(2))
    lp, h, lse, left = (torch.full((N, space), 7.0, device="cuda") for _ in range(4))
    gx = torch.full_like(x, 7.0)
    sizes = (N, K, space, K * space, space)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    at = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    f32, i32 = _lib.MVR_F32, 2
    if rest:
        assert L.mvr_label_log_probs_forward_rest(at(x), f32, at(y), i32, at(lp), at(h), at(lse), at(left), None, None, *sizes, 0, stream) == 0
        assert L.mvr_label_log_probs_backward_rest(at(x), f32, at(y), i32, at(lse), at(left), at(h), at(a), at(b), at(gx), *sizes,
                                                   K * space, space, stream) == 0
    else:
        assert L.mvr_label_log_probs_forward(at(x), f32, at(y), i32, at(lp), at(h), at(lse), None, None, *sizes, 0, stream) == 0
        assert L.mvr_label_log_probs_backward(at(x), f32, at(y), i32, at(lse), at(h), at(a), at(b), at(gx), *sizes, K * space, space,
                                              stream) == 0
    xd = x.cpu().double()
    want_lp, want_h, _, _, grad = reference(xd, y.cpu().long(), 0, a.cpu().double(), b.cpu().double())
    check(lp, want_lp, (8 * math.sqrt(K) + 4 + 6 * want_lp.abs()) * E, "log_prob")
    xf = xd.where(xd.isfinite(), torch.tensor(offset - 60.0, dtype=torch.float64))  # (a class of probability 0: any far score bounds it)
    check(gx, grad, gradient_bound(xf, grad, a.cpu(), b.cpu(), want_h, 8 * math.sqrt(K) + 4, torch.float32), "gradient")
    exact = torch.logsumexp(xd, 1)
    if rest:
        check(lse.double() + left.double(), exact, (8 * math.sqrt(K) + 4) * E * (1 + math.log(K)) + 0 * exact, "lse")
        assert not bool((left == 7).any())
    check(lse, exact, exact.abs() * 2.0 ** -23 + 8 * math.sqrt(K) * E, "lse")


def test_c_entries_with_a_rest_check_before_any_cuda_call():
    from medvision_b200 import _lib
    f, b = _lib.lib.mvr_label_log_probs_forward_rest, _lib.lib.mvr_label_log_probs_backward_rest

    def fwd(dtype=0, classes=4, top=0, lse=16, rest=16, batch=2):
        return f(16, dtype, 16, 2, 16, 16, lse, rest, None, None, batch, classes, 1, classes, 1, top, None)
    assert fwd(dtype=2) == -1 and fwd(classes=0) == -5 and fwd(top=5) == -18 and fwd(top=1) == -6
    assert fwd(rest=None) == -6 and fwd(lse=None) == -6 and fwd(batch=0, lse=None) == 0

    def bwd(lse=16, rest=16, batch=2):
        return b(16, 0, 16, 2, lse, rest, 16, None, None, 16, batch, 4, 1, 4, 1, 4, 1, None)
    assert bwd(lse=None) == -6 and bwd(rest=None) == -6 and bwd(batch=0, rest=None) == 0
