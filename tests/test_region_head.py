"""The operators behind the roi modules in one head, as they are used: RoIAlign's bins read an encoder's map by attention, join the
residual stream through dropout, and give the labels' log-probabilities; against the same head in float64, its gradients against the
formulas', in eager mode and as a captured step."""
import math

import pytest
import torch

from medvision_b200.ops import Dropout, RoIAlign, cross_attention, dropout, label_log_probs

from test_dropout import kept

E = 2.0 ** -24
C, HEADS, CLASSES, BINS, SEED, P = 32, 4, 7, (3, 3), 1234, 0.25


def _inputs():
    g = torch.Generator().manual_seed(0)
    features = torch.randn(2, C, 20, 24, generator=g)
    centre, size = torch.rand(11, 2, generator=g) * 16 + 3, torch.rand(11, 2, generator=g) * 6 + 4
    rois = torch.cat([torch.randint(0, 2, (11, 1), generator=g).float(), centre - size / 2, centre + size / 2], 1)
    weights = [torch.randn(a, b, generator=g) / math.sqrt(a) for a, b in ((C, C), (C, C), (C, C), (C, CLASSES))]
    labels = torch.randint(-1, CLASSES, (11,), generator=g)
    body = torch.rand(2, 20 * 24, generator=g) < 0.7
    return features, rois, weights, labels, body


def head(features, rois, weights, labels, body):
    bins = RoIAlign(BINS, 1.0, sampling_ratio=2)(features, rois)                    # (R, C, 3, 3)
    x = bins.flatten(2).transpose(1, 2)                                             # (R, 9, C)
    states = features.flatten(2).transpose(1, 2)                                    # (N, 480, C)
    q, k, v = x @ weights[0], states @ weights[1], states @ weights[2]
    split = lambda t: t.unflatten(2, (HEADS, C // HEADS))  # noqa: E731
    read = cross_attention(split(q), split(k), split(v), batch_index=rois[:, 0], mask=body)
    x = dropout(read.flatten(2), P, SEED, residual=x)
    r = label_log_probs(x.mean(1) @ weights[3], labels, top=3)
    return r, -(r.log_prob.sum() / 11) - 0.1 * r.entropy.mean()


def head64(bins, features, rois, weights, labels, body):
    """The same in float64 from RoIAlign's bins; differentiable in bins, features and weights."""
    x, states = bins.flatten(2).transpose(1, 2), features.flatten(2).transpose(1, 2)
    split = lambda t: t.unflatten(2, (HEADS, C // HEADS))  # noqa: E731
    q, k, v = split(x @ weights[0]), split(states @ weights[1]), split(states @ weights[2])
    at = rois[:, 0].long()
    s = torch.einsum("rthd,rlhd->rhtl", q, k[at]) / math.sqrt(C // HEADS)
    p = torch.softmax(s.masked_fill(~body[at][:, None, None, :], -math.inf), -1)
    read = torch.einsum("rhtl,rlhd->rthd", p, v[at]).flatten(2)
    keep, scale = kept(read.numel(), P, SEED)
    x = x + torch.where(keep.view(read.shape), read * scale, 0.0)
    logs = torch.log_softmax(x.mean(1) @ weights[3], 1)
    given = labels >= 0
    lp = torch.where(given, logs.gather(1, labels.clamp(min=0).unsqueeze(1)).squeeze(1), 0.0)
    h = -(logs.exp() * logs).sum(1)
    return lp, h, logs.topk(3, 1), -(lp.sum() / 11) - 0.1 * h.mean()


@pytest.mark.gpu
def test_a_training_step_and_its_captured_form():
    torch.backends.cuda.matmul.allow_tf32 = False
    features, rois, weights, labels, body = _inputs()
    leaves = [features.cuda().requires_grad_()] + [w.cuda().requires_grad_() for w in weights]
    rest = rois.cuda(), labels.cuda(), body.cuda()
    step = lambda: head(leaves[0], rest[0], leaves[1:], rest[1], rest[2])  # noqa: E731
    r, loss = step()
    grads = torch.autograd.grad(loss, leaves)
    bins = RoIAlign(BINS, 1.0, sampling_ratio=2)(leaves[0], rest[0])
    b64 = bins.detach().cpu().double().requires_grad_()
    l64 = [t.detach().cpu().double().requires_grad_() for t in leaves]
    lp, h, top, loss64 = head64(b64, l64[0], rois, l64[1:], labels, body)
    g64 = list(torch.autograd.grad(loss64, [b64] + l64))
    through_bins, = torch.autograd.grad(bins, leaves[0], g64[0].float().cuda())  # RoIAlign's own gradient, from the exact one of its bins
    g64[1] = g64[1] + through_bins.cpu().double()
    # a chain of some eight float operations with sums of up to 480 terms: 8 * 8 sqrt(480) e of the values' size, which is 10 at most
    tol = 8 * 8 * math.sqrt(480) * E
    assert float((r.log_prob.detach().cpu() - lp).abs().max()) <= 10 * tol
    assert float((r.entropy.detach().cpu() - h).abs().max()) <= 10 * tol
    assert torch.equal(r.top_label.cpu().long(), top.indices)
    for got, want in zip(grads, g64[1:]):
        assert float((got.cpu() - want).norm() / want.norm()) <= 10 * tol
    first = [t.clone() for t in (loss.detach(),) + grads]
    del r, loss, grads, bins  # (no eager graph of the leaves lives while their step is captured)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(step()[1], leaves)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        loss = step()[1]
        grads = torch.autograd.grad(loss, leaves)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss.detach(), first[0])
    for a, b in zip(grads[1:], first[2:]):  # (the features' gradient passes RoIAlign's, whose sums have no fixed order)
        assert float((a - b).norm()) <= 1e-6 * float(b.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_half_precision_head_trains_and_serves(dtype):
    features, rois, weights, labels, body = _inputs()
    features = features.to(torch.float16)  # (RoIAlign takes float16)
    x = RoIAlign(BINS, 1.0, sampling_ratio=2)(features.cuda(), rois.half().cuda()).flatten(2).transpose(1, 2).to(dtype)
    states = features.cuda().flatten(2).transpose(1, 2).to(dtype)
    w = [t.to(dtype).cuda().requires_grad_() for t in weights]
    layer = Dropout(0.1)

    def run():
        q, k, v = ((t @ u).unflatten(2, (HEADS, C // HEADS)) for t, u in ((x, w[0]), (states, w[1]), (states, w[2])))
        y = layer(cross_attention(q, k, v, batch_index=rois[:, 0].cuda(), mask=body.cuda()).flatten(2), x, seed=5)
        return label_log_probs(y.mean(1) @ w[3], labels.cuda(), top=2)

    r = run()
    grads = torch.autograd.grad(-r.log_prob.mean(), w)
    assert all(bool(g.isfinite().all()) and bool(g.any()) for g in grads)
    layer.eval()
    with torch.no_grad():
        served = run()
    assert bool((served.top_log_prob[:, 0] >= served.top_log_prob[:, 1]).all()) and bool((served.log_prob <= 0).all())
