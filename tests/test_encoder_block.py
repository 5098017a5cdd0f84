"""An encoder's block and the head that reads its states, as they are used: a channels-last map is normalised, its queries and keys are turned by
their voxels' places, attend in a window along the scan with a few first states visible, and RoIAlign's bins, turned by their own places,
read the result; against the same in float64, its gradients against the formulas', in eager mode and as a captured step."""
import math

import pytest
import torch

from medvision_b200.ops import GroupNorm, RoIAlign, cross_attention, group_norm, rotary_positions, window_attention

E = 2.0 ** -24
N, C, HEADS, KEY_HEADS, MAP, BINS = 2, 48, 6, 2, (5, 12, 14), (2, 2)
DIM, STATES, GROUPS, WINDOW = C // HEADS, math.prod(MAP), 6, (60, 20, 3)
SECTIONS = [1, 1, 2]


def _inputs():
    g = torch.Generator().manual_seed(0)
    maps = torch.randn(N, C, *MAP, generator=g) + 0.5
    norm = [1 + 0.2 * torch.randn(C, generator=g), 0.2 * torch.randn(C, generator=g)]
    weights = [torch.randn(C, n, generator=g) / math.sqrt(C) for n in (C + 2 * KEY_HEADS * DIM, C, 2 * KEY_HEADS * DIM)]
    places = torch.stack(torch.meshgrid(*(torch.arange(n) for n in MAP), indexing="ij"), -1).reshape(1, STATES, 3).expand(N, STATES, 3)
    rois = torch.tensor([[0.0, 1, 1, 9, 8], [1, 2, 0, 11, 7], [1, 4, 3, 12, 11], [0, 0, 2, 6, 9]])
    lengths = torch.tensor([STATES, STATES - 200])
    return maps, norm, weights, places, rois, lengths


def bin_places(rois):
    """Centres of a region's bins, in the middle slice."""
    step = torch.stack([(rois[:, 4] - rois[:, 2]) / BINS[0], (rois[:, 3] - rois[:, 1]) / BINS[1]], 1)
    k = torch.stack(torch.meshgrid(torch.arange(BINS[0]), torch.arange(BINS[1]), indexing="ij"), -1).reshape(1, -1, 2) + 0.5
    yx = rois[:, [2, 1]][:, None] + k * step[:, None]
    return torch.cat([torch.full_like(yx[..., :1], MAP[0] // 2), yx], -1).float()


def block(maps, norm, weights, places, rois, lengths, at, bins):  # at: places of the bins
    x = group_norm(maps.permute(0, 2, 3, 4, 1), GROUPS, *norm, activation="silu").flatten(1, 3)                  # (N, STATES, C)
    q, k, v = (x @ weights[0]).unflatten(2, (-1, DIM)).split([HEADS, KEY_HEADS, KEY_HEADS], 2)
    q, k = rotary_positions(q, places, k, SECTIONS, base=100.0)
    states = window_attention(q, k, v, *WINDOW, lengths=lengths).flatten(2) + x
    query = rotary_positions((bins @ weights[1]).unflatten(2, (HEADS, DIM)), at, sections=SECTIONS, base=100.0)
    key, value = (states @ weights[2]).unflatten(2, (-1, DIM)).split(KEY_HEADS, 2)
    key = rotary_positions(key, places, sections=SECTIONS, base=100.0)
    return cross_attention(query, key, value, batch_index=rois[:, 0], lengths=lengths)


def turn64(x, places):
    pairs = [(axis, 100.0 ** (-k / n)) for axis, n in enumerate(SECTIONS) for k in range(n)]
    angle = torch.stack([places[..., a].double() * f for a, f in pairs], -1)[:, :, None]
    a, b = x[..., :len(pairs)], x[..., len(pairs):]
    return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1)


def attend64(q, k, v, allowed):
    group = q.shape[2] // k.shape[2]
    k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
    s = torch.einsum("nthd,nlhd->nhtl", q, k) / math.sqrt(q.shape[3])
    some = allowed.any(-1)[:, None, :, None]
    p = torch.where(some, torch.softmax(s.masked_fill(~allowed[:, None], -1e300), -1), 0.0)
    return torch.einsum("nhtl,nlhd->nthd", p, v)


def block64(maps, norm, weights, places, rois, lengths, at, bins):
    rows = maps.reshape(N, GROUPS, -1)
    y = (rows - rows.mean(2, keepdim=True)) / torch.sqrt(rows.var(2, unbiased=False, keepdim=True) + 1e-5)
    z = y.reshape(maps.shape).permute(0, 2, 3, 4, 1) * norm[0] + norm[1]
    x = (z * torch.sigmoid(z)).flatten(1, 3)
    q, k, v = (x @ weights[0]).unflatten(2, (-1, DIM)).split([HEADS, KEY_HEADS, KEY_HEADS], 2)
    t, j = torch.arange(STATES)[:, None], torch.arange(STATES)
    before, after, sinks = WINDOW
    seen = ((j <= t + after) & ((j >= t - before) | (j < sinks)))[None] & (j < lengths[:, None, None])
    states = attend64(turn64(q, places), turn64(k, places), v, seen).flatten(2) + x
    query = turn64((bins @ weights[1]).unflatten(2, (HEADS, DIM)), at)
    key, value = (states @ weights[2]).unflatten(2, (-1, DIM)).split(KEY_HEADS, 2)
    image = rois[:, 0].long()
    valid = (j < lengths[image][:, None])[:, None].expand(-1, query.shape[1], -1)
    return attend64(query, turn64(key, places)[image], value[image], valid)


def _bins(maps, rois):
    return RoIAlign(BINS, 1.0, sampling_ratio=2)(maps[:, :, MAP[0] // 2].contiguous(), rois).flatten(2).transpose(1, 2)


@pytest.mark.gpu
def test_a_training_step_and_its_captured_form():
    torch.backends.cuda.matmul.allow_tf32 = False
    maps, norm, weights, places, rois, lengths = _inputs()
    last = maps.cuda().to(memory_format=torch.channels_last_3d)
    bins = _bins(last, rois.cuda())
    leaves = [t.detach().clone().requires_grad_() for t in [last, bins] + [t.cuda() for t in norm + weights]]
    rest = places.cuda(), rois.cuda(), lengths.cuda(), bin_places(rois).cuda()
    grad = torch.randn(rois.shape[0], 4, HEADS, DIM, generator=torch.Generator().manual_seed(1))
    g = grad.cuda()

    def step():
        out = block(leaves[0], leaves[2:4], leaves[4:], *rest, leaves[1])
        return (out.detach(),) + torch.autograd.grad(out, leaves, g)

    got = step()
    l64 = [t.detach().cpu().double().requires_grad_() for t in leaves]
    out64 = block64(l64[0], l64[2:4], l64[4:], places, rois, lengths, bin_places(rois), l64[1])
    want = (out64.detach(),) + torch.autograd.grad(out64, l64, grad.double())
    # a chain of some twelve float operations with sums of up to 6720 terms (a group of the norm): 12 * 8 sqrt(6720) e of the values' size
    tol = 12 * 8 * math.sqrt(6720) * E
    for a, b in zip(got, want):
        assert float((a.cpu() - b).norm()) <= tol * float(b.norm())
    first = [t.clone() for t in got]
    del got  # (no eager graph of the leaves lives while their step is captured)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, first):  # (the library's products may take other kernels while they are captured)
        assert float((a - b).norm()) <= tol * float(b.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_half_precision_and_one_token_at_a_time(dtype):
    """The block trains in half types; and its window, served token by token over a cache, gives what the whole sequence gives."""
    maps, norm, weights, places, rois, lengths = _inputs()
    layer = GroupNorm(GROUPS, C, activation="silu", device="cuda")
    w = [t.to(dtype).cuda().requires_grad_() for t in weights]
    x = layer(maps.to(dtype).cuda().permute(0, 2, 3, 4, 1)).flatten(1, 3)
    q, k, v = (x @ w[0]).unflatten(2, (-1, DIM)).split([HEADS, KEY_HEADS, KEY_HEADS], 2)
    q, k = rotary_positions(q, places.cuda(), k, SECTIONS, base=100.0)
    whole = window_attention(q, k, v, 60, 0, 3)
    grads = torch.autograd.grad(whole.float().square().mean(), [w[0], layer.weight, layer.bias])
    assert all(bool(t.isfinite().all()) and bool(t.any()) for t in grads)
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    with torch.no_grad():
        for t in (0, 1, 2, 63, 500, STATES - 1):
            one = window_attention(q[:, t:t + 1], k, v, 60, 0, 3, offsets=torch.full((N,), t, device="cuda"), lengths=torch.full((N,), t + 1, device="cuda"))
            # weights and results are rounded to the type in one form and not, or elsewhere, in the other: 2 u of the values' size each
            assert float((one[:, 0].float() - whole[:, t].float()).abs().max()) <= 4 * u * float(v.float().abs().max())
