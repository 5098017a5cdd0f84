"""ops.dropout: the generator against its published answers and a restatement in whole numbers, results and gradients against
the definition, and what it refuses.

Tolerances: a kept element is x * scale in float (scale itself rounded: two roundings, 2 * 2^-24 of it), the residual's addition one
more, and the result one of its type (half a step; float16 has steps of 2^-24 at least)."""
import numpy as np
import pytest
import torch

from medvision_b200.ops import Dropout, dropout

E = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def philox(counter, key, rounds=10):
    """Philox 4x32 on Python integers."""
    c, k = list(counter), list(key)
    for _ in range(rounds):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b % 2 ** 32, (a >> 32) ^ c[3] ^ k[1], a % 2 ** 32]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def kept(n, p, seed, offset=0, first=0):
    cut, out = int(np.floor(p * 65536 + 0.5)), []
    for group in range(first // 8, (first + n + 7) // 8):
        words = philox([group % 2 ** 32, group >> 32, offset % 2 ** 32, offset >> 32], [seed % 2 ** 32, seed >> 32])
        out += [h >= cut for w in words for h in (w & 0xFFFF, w >> 16)]
    return torch.tensor(out[:n]), 65536 / (65536 - cut) if cut < 65536 else 0.0


def test_the_generator_gives_the_published_answers():
    """Known answers that the authors of the generator published with it."""
    assert philox([0] * 4, [0, 0]) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox([2 ** 32 - 1] * 4, [2 ** 32 - 1] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def check(got, want, x, res, dtype):
    err = (got.detach().cpu().double() - want).abs()
    bound = HALF[dtype] * want.abs() + 3 * E * (x.abs() + res.abs()) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert bool((err <= bound).all()), float((err / bound.clamp(min=1e-30)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5, 7), (2, 1027), (33, 64)])
@pytest.mark.parametrize("p,seed,offset", [(0.5, 0, 0), (0.1, 2 ** 64 - 1, 5), (0.0, 1, 2 ** 40), (1.0, 3, 0), (2 ** -16, 12345678901234567, 2 ** 64 - 1)])
def test_results_and_gradients(dtype, shape, p, seed, offset):
    g = torch.Generator().manual_seed(len(shape))
    x, r, u = (torch.randn(shape, generator=g).to(dtype) for _ in range(3))
    keep, scale = kept(x.numel(), p, seed, offset)
    keep = keep.view(shape)
    a, b = x.cuda().requires_grad_(), r.cuda().requires_grad_()
    alone = dropout(a, p, seed, offset)
    scaled = torch.where(keep, x.double() * scale, 0.0)
    check(alone, scaled, scaled, torch.zeros(()), dtype)
    ga, = torch.autograd.grad(alone, a, u.cuda())
    scaled_u = torch.where(keep, u.double() * scale, 0.0)
    check(ga, scaled_u, scaled_u, torch.zeros(()), dtype)
    both = dropout(a, p, seed, offset, residual=b)
    check(both, scaled + r.double(), scaled, r.double(), dtype)
    grads = torch.autograd.grad(both, (a, b), u.cuda())
    assert torch.equal(grads[0], ga) and torch.equal(grads[1].cpu(), u)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_views_dropped_nan_and_negative_seeds(dtype):
    base = torch.randn(5 * 41 + 1, generator=torch.Generator().manual_seed(0)).to(dtype)
    x = base[1:].view(5, 41)                                     # not 16-byte aligned
    want = dropout(x.clone().cuda(), 0.4, 9)
    assert torch.equal(dropout(base.cuda()[1:].view(5, 41), 0.4, 9), want)
    assert torch.equal(dropout(x.t().contiguous().cuda().t(), 0.4, 9), want)  # the row-major place counts, not the memory's
    keep = kept(x.numel(), 0.4, 9)[0].view(5, 41)
    dirty = torch.where(keep, x, torch.tensor(float("nan")).to(dtype))
    assert torch.equal(dropout(dirty.cuda(), 0.4, 9), want)
    assert torch.equal(dropout(x.cuda(), 0.4, -1), dropout(x.cuda(), 0.4, 2 ** 64 - 1))
    seed = torch.tensor(9, device="cuda")
    assert torch.equal(dropout(x.cuda(), 0.4, seed), want)
    assert dropout(x[:0].cuda(), 0.4, 9).shape == (0, 41)


@pytest.mark.gpu
def test_places_beyond_32_bits():
    """The last of 2^32 + 24 elements: their counters' high words and their offsets."""
    n, p, seed = 2 ** 32 + 24, 0.5, 77
    x = torch.ones(n, dtype=torch.float16, device="cuda")
    out = dropout(x, p, seed)
    for first in (2 ** 31 - 8, 2 ** 32 - 16, 2 ** 32 + 8):
        keep, scale = kept(16, p, seed, first=first)
        assert torch.equal(out[first:first + 16].cpu(), torch.where(keep, scale, 0.0).half()), first


@pytest.mark.gpu
def test_share_of_kept_elements_and_independence_of_offsets():
    n = 1 << 22
    x = torch.ones(n, device="cuda")
    a, b = dropout(x, 0.3, 5, 0) != 0, dropout(x, 0.3, 5, 1) != 0
    q = 1 - round(0.3 * 65536) / 65536
    for got, share in ((a, q), (b, q), (a & b, q * q)):
        assert abs(float(got.double().mean()) - share) <= 6 * (share * (1 - share) / n) ** 0.5  # six standard deviations


@pytest.mark.gpu
def test_module_and_graphs():
    layer = Dropout(0.25)
    x, r = torch.randn(64, 100).cuda(), torch.randn(64, 100).cuda()
    torch.manual_seed(11)
    a = layer(x, r)
    torch.manual_seed(11)
    assert torch.equal(a, layer(x, r)) and not torch.equal(a, layer(x, r))
    assert torch.equal(layer.eval()(x), x) and torch.equal(layer(x, r), x + r)
    # a graph that reads its seed from the device: another mask per replay, the gradient with the same one
    seed = torch.tensor([1], device="cuda")
    leaf = x.clone().requires_grad_()
    torch.autograd.grad(dropout(leaf, 0.25, seed), leaf, r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = dropout(leaf, 0.25, seed)
        grad, = torch.autograd.grad(out, leaf, r)
    for s in (3, 4):
        seed.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, dropout(x, 0.25, s)) and torch.equal(grad, dropout(r, 0.25, s))


@pytest.mark.gpu
def test_a_seed_changed_before_the_gradient_is_noticed():
    x, seed = torch.randn(8, device="cuda", requires_grad=True), torch.tensor([1], device="cuda")
    out = dropout(x, 0.5, seed)
    seed += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_refusals():
    x = torch.zeros(4)
    with pytest.raises(RuntimeError, match="dropout is not implemented on CPU"):
        dropout(x, 0.5, 1)
    with pytest.raises(RuntimeError, match="not implemented for 'float64'"):
        dropout(x.double(), 0.5, 1)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="between 0 and 1"):
            dropout(x, p, 1)
    with pytest.raises(ValueError, match="between 0 and 1"):
        Dropout(1.5)
    with pytest.raises(RuntimeError, match="same shape"):
        dropout(x, 0.5, 1, residual=torch.zeros(5))
    with pytest.raises(RuntimeError, match="expected scalar type"):
        dropout(x, 0.5, 1, residual=torch.zeros(4).half())
    with pytest.raises(RuntimeError, match="one int64"):
        dropout(x, 0.5, torch.zeros(1))
    with pytest.raises(RuntimeError, match="one int64"):
        dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))
    for seed in (2 ** 64, -2 ** 63 - 1):
        with pytest.raises(ValueError, match="seed must fit 64 bits"):
            dropout(x, 0.5, seed)
    with pytest.raises(ValueError, match="offset must fit 64 bits"):
        dropout(x, 0.5, 1, offset=2 ** 64)
    with pytest.raises(TypeError):
        dropout(x, 0.5, 1.5)
    assert dropout(x, 0.5, training=False) is x


def test_c_entry_checks_before_any_cuda_call():
    from medvision_b200 import _lib
    f = _lib.lib.mvr_dropout
    assert f(16, None, 16, 2, 4, 0.5, 1, None, 0, None) == -1
    assert f(16, None, 16, 0, -1, 0.5, 1, None, 0, None) == -5
    assert f(16, None, 16, 0, 4, 1.5, 1, None, 0, None) == -17 and f(16, None, 16, 0, 4, float("nan"), 1, None, 0, None) == -17
    assert f(None, None, 16, 0, 4, 0.5, 1, None, 0, None) == -6
    assert f(None, None, None, 0, 0, 0.5, 1, None, 0, None) == 0
