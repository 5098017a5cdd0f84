"""ops.window_attention against its formula in float64: forward, gradients, windows that leave nothing, sequences of every length, odd
sizes and strides, what states that no token reads may hold, other streams and graphs, and what it refuses.

Tolerances: those of tests/test_cross_attention.py, whose arithmetic is the same; each token has a list of states of its own here.
"""
import ctypes
import math

import pytest
import torch

from medvision_b200 import _lib
from medvision_b200.ops import cross_attention, window_attention

from test_cross_attention import E, HALF, NAMES, check


def allowed_states(T, L, before, after, sinks, offset, length):
    place = offset + torch.arange(T)[:, None]
    j = torch.arange(L)
    return (j < length) & (j <= place + after) & ((j >= place - before) | (j < sinks))


def reference(q, k, v, g, before, after, sinks, offsets, lengths, scale, dtype):
    """(value, bound) of out, dq, dk, dv, all float64 on the CPU: the bounds of test_cross_attention.reference, token by token."""
    q, k, v, g = (t.detach().cpu().double() for t in (q, k, v, g))
    N, T, H, D = q.shape
    L, Hk = k.shape[1:3]
    u = HALF[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    res = [torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k)]
    bound, size = [torch.zeros_like(t) for t in res], [torch.zeros_like(t) for t in res]
    for n in range(N):
        ok = allowed_states(T, L, before, after, sinks, offsets[n], lengths[n])
        some = ok.any(1, keepdim=True)
        for h in range(H):
            a, b = torch.where(ok.any(0)[:, None], k[n, :, h * Hk // H], 0.0), torch.where(ok.any(0)[:, None], v[n, :, h * Hk // H], 0.0)
            x, gr = q[n, :, h], g[n, :, h]
            p = torch.where(some, torch.softmax((scale * x @ a.T).masked_fill(~ok, -math.inf), 1), 0.0)
            o = p @ b
            dp = gr @ b.T
            delta = (gr * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            big = float((abs(scale) * x.abs() @ a.abs().T).max()) if L else 0.0
            w = (0 if dtype == torch.float32 else u) + 8 * math.sqrt(D + L) * E + 8 * math.sqrt(D) * E * big
            err = 2 * w * ds.abs() + ok * tiny * (dp - delta).abs() + p * (u * (gr.abs() * o.abs()).sum(1, keepdim=True)
                + 8 * math.sqrt(D) * E * (gr.abs() @ b.abs().T + (gr.abs() * o.abs()).sum(1, keepdim=True)))
            res[0][n, :, h] = o
            bound[0][n, :, h] = 2 * w * p @ b.abs() + tiny * ok.double() @ b.abs()
            res[1][n, :, h] = scale * ds @ a
            bound[1][n, :, h] = abs(scale) * err @ a.abs()
            res[2][n, :, h * Hk // H] += scale * ds.T @ x
            bound[2][n, :, h * Hk // H] += abs(scale) * err.T @ x.abs()
            size[2][n, :, h * Hk // H] += abs(scale) * ds.abs().T @ x.abs()
            res[3][n, :, h * Hk // H] += p.T @ gr
            bound[3][n, :, h * Hk // H] += (2 * w * p + tiny * ok).T @ gr.abs()
            size[3][n, :, h * Hk // H] += p.T @ gr.abs()
    rows = T * (H // Hk)
    for i in range(4):
        bound[i] += u * res[i].abs() + 8 * math.sqrt(max(rows, 1)) * E * size[i] + tiny
    return res, bound


def make(N, T, H, Hk, D, L, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    t = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    return t(N, T, H, D), t(N, L, Hk, D), t(N, L, Hk, D), t(N, T, H, D)


def run(q, k, v, g, *window, **kw):
    q, k, v = (t.cuda().requires_grad_() for t in (q, k, v))
    out = window_attention(q, k, v, *window, **kw)
    return (out,) + torch.autograd.grad(out, (q, k, v), g.cuda())


def compare(shape, window, dtype, offsets=None, lengths=None, seed=0, **kw):
    q, k, v, g = make(*shape, dtype, seed=seed)
    N, T, H, Hk, D, L = shape
    res, bound = reference(q, k, v, g, *window, offsets or [0] * N, [min(max(n, 0), L) for n in (lengths or [L] * N)], D ** -0.5, dtype)
    if offsets is not None:
        kw["offsets"] = torch.tensor(offsets, device="cuda")
    if lengths is not None:
        kw["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for name, a, b, c in zip(NAMES, run(q, k, v, g, *window, **kw), res, bound):
        check(a, b, c, name)


SHAPES = [  # N, T, H, Hk, D, L
    (2, 1, 1, 1, 1, 1),
    (2, 7, 4, 2, 16, 7),
    (1, 64, 2, 2, 32, 64),
    (2, 129, 2, 1, 64, 129),
    (1, 257, 3, 3, 128, 257),
    (2, 300, 4, 1, 72, 300),
    (1, 70, 2, 2, 33, 70),
    (1, 97, 2, 2, 200, 97),
    (1, 40, 1, 1, 256, 40),
    (1, 700, 6, 1, 64, 700),     # six heads share a key head: 64 rows are no whole tokens
    (2, 1100, 2, 2, 40, 1100),
    (1, 600, 8, 1, 128, 600),
]
WINDOWS = [(0, 0, 0), (5, 0, 0), (63, 0, 4), (64, 17, 1), (0, 130, 0), (200, 200, 130), (10 ** 12, 0, 0), (10 ** 12, 10 ** 12, 10 ** 12)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("window", WINDOWS)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_formula(shape, window, dtype):
    compare(shape, window, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("window", [(0, 0, 0), (40, 0, 3), (70, 30, 0), (300, 5, 140)])
@pytest.mark.parametrize("tokens,dim,heads", [(1, 64, 8), (1, 128, 4), (3, 32, 2), (130, 64, 4), (5, 20, 2), (260, 128, 2)])
def test_caches_and_padded_sequences(dtype, window, tokens, dim, heads):
    """Tokens at the end of caches of different lengths, at their beginning, before all states and behind them; lengths 0 and 1, negative
    and beyond the states."""
    L = 421
    lengths = [L, 0, 1, 300, 64, 129, -3, 10 ** 6, 200, 200, 200]
    offsets = [L - tokens, 0, 0, 300 - tokens, 0, 129, 5, 17, -tokens - 10, -2, 10 ** 9]
    compare((len(lengths), tokens, heads, 2, dim, L), window, dtype, offsets, lengths, seed=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("window", [(0, 0, 0), (90, 0, 5), (700, 0, 0), (30, 9, 200)])
@pytest.mark.parametrize("tokens,dim,heads", [(1, 64, 2), (1, 8, 2), (2, 64, 2), (1, 256, 4), (1, 128, 6), (1, 40, 16), (3, 32, 4), (8, 128, 2), (1, 96, 8), (7, 200, 2)])
def test_one_to_eight_rows_of_a_key_head(tokens, dim, heads, window, dtype):
    L = 733
    lengths, offsets = [L, 0, 1, 400, 90, 600], [L - tokens, 0, 0, 400 - tokens, 88, 650]
    compare((len(lengths), tokens, heads, 2, dim, L), window, dtype, offsets, lengths, seed=10)


@pytest.mark.gpu
def test_a_few_rows_with_scores_that_are_not_finite():
    q, k, v, _ = (t.cuda() for t in make(1, 1, 4, 2, 64, 300, torch.float32, seed=11))
    want = window_attention(q, k, v, 299, offsets=299)
    for bad, finite in ((math.nan, False), (math.inf, False), (-math.inf, True)):
        x = k.clone()
        x[0, 200, 0] = torch.sign(q[0, 0, 0]) * bad if bad == bad else bad  # (the first query's score of this state)
        out = window_attention(q, x, v, 299, offsets=299)
        assert torch.equal(out[0, 0, 2:], want[0, 0, 2:]) and bool(out[0, 0, 0].isfinite().all()) == finite


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dim", [20, 64, 128])
def test_unread_states_may_hold_anything(dtype, dim):
    N, T, L, window = 4, 70, 400, (30, 0, 5)
    offsets, lengths = [200, 0, 330, 100], [270, 70, 400, 0]
    q, k, v, g = make(N, T, 4, 2, dim, L, dtype, seed=2)
    kw = dict(offsets=torch.tensor(offsets, device="cuda"), lengths=torch.tensor(lengths, device="cuda"))
    clean = run(q, k, v, g, *window, **kw)
    for n in range(N):
        unread = ~allowed_states(T, L, *window, offsets[n], lengths[n]).any(0)
        assert bool(unread.any())
        k[n, unread], v[n, unread] = math.nan, math.inf
    for a, b in zip(clean, run(q, k, v, g, *window, **kw)):
        assert torch.equal(a, b)
    for n in range(N):
        unread = ~allowed_states(T, L, *window, offsets[n], lengths[n]).any(0)
        assert not bool(clean[2][n, unread.cuda()].any()) and not bool(clean[3][n, unread.cuda()].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_a_window_over_everything_is_cross_attention(dtype):
    q, k, v, g = make(2, 150, 4, 2, 64, 333, dtype, seed=3)
    a = run(q, k, v, g, 400, 400)
    x = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = cross_attention(*x)
    for one, other in zip(a, (out,) + torch.autograd.grad(out, x, g.cuda())):
        bound = 16 * HALF[dtype] * float(other.abs().max()) + 64 * E  # (the same sums in another order)
        assert float((one - other).abs().max()) <= bound


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape,window", [((1, 5000, 2, 1, 64, 5000), (100, 0, 3)), ((1, 3000, 8, 1, 128, 3000), (700, 0, 1)),
                                          ((2, 2500, 1, 1, 32, 2500), (50, 50, 200)), ((1, 2600, 2, 2, 96, 2600), (2600, 0, 0))])
def test_long_sequences(shape, window, dtype):
    compare(shape, window, dtype, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_strides_and_scales(dtype):
    """Parts of a projection's rows, heads before tokens, expanded gradients, negative and other scales, rows that TMA cannot read."""
    N, T, H, Hk, D, window = 2, 140, 4, 2, 64, (37, 3, 2)
    gen = torch.Generator().manual_seed(5)
    rows = torch.randn(N, T, H + 2 * Hk, D, generator=gen).to(dtype)
    q, k, v = rows.split([H, Hk, Hk], 2)
    for scale in (0.3, -0.2, 0.0):
        res, bound = reference(q, k, v, torch.ones(N, T, H, D), *window, [0] * N, [T] * N, scale, dtype)
        a, b, c = (t.requires_grad_() for t in rows.cuda().split([H, Hk, Hk], 2))
        out = window_attention(a, b, c, *window, scale=scale)
        for name, x, y, z in zip(NAMES, (out,) + torch.autograd.grad(out, (a, b, c), torch.ones((), dtype=dtype, device="cuda").expand(N, T, H, D)), res, bound):
            check(x, y, z, name)
    res, bound = reference(q, k, v, q, *window, [0] * N, [T] * N, 0.125, dtype)
    turned = [t.transpose(1, 2).contiguous().cuda().transpose(1, 2).requires_grad_() for t in (q, k, v)]
    odd = [torch.cat([t.flatten(), t.flatten()[:1]]).cuda()[1:].view(t.shape) for t in (q.flatten().roll(1), k.flatten().roll(1), v.flatten().roll(1))]
    odd = [o.view(t.shape) for o, t in zip(odd, (q, k, v))]
    for x in (turned, [o.requires_grad_() for o in odd]):
        if x is not turned:
            assert all(t.data_ptr() % 16 for t in x)
            now = [t.detach().cpu() for t in x]
            res, bound = reference(*now, q, *window, [0] * N, [T] * N, 0.125, dtype)
        out = window_attention(*x, *window, scale=0.125)
        for name, y, z, w in zip(NAMES, (out,) + torch.autograd.grad(out, x, q.cuda()), res, bound):
            check(y, z, w, name)


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences of the float32 result along random directions: step 2^-6, whose square times the third derivative stays below
    1e-3 of the slope here, and rounding 2^-24 sqrt(values) / step."""
    q, k, v, g = (t.cuda() for t in make(1, 40, 2, 1, 16, 40, torch.float32, seed=6))
    window = (6, 1, 2)
    grads = run(q, k, v, g, *window)[1:]
    gen = torch.Generator("cuda").manual_seed(0)
    for i, x in enumerate((q, k, v)):
        d = torch.randn(x.shape, generator=gen, device="cuda")
        d = d / d.norm()
        f = lambda s: float((window_attention(*[t + s * d if t is x else t for t in (q, k, v)], *window).double() * g).sum())  # noqa: E731
        step = 2.0 ** -6
        slope = (f(step) - f(-step)) / (2 * step)
        want = float((grads[i].double() * d).sum())
        assert abs(slope - want) <= 1e-3 * float(grads[i].norm()) + 40 * E * float(g.norm()) / step


@pytest.mark.gpu
def test_repeatable_and_from_other_streams_and_devices_current():
    args = make(2, 700, 4, 2, 64, 700, torch.float16, seed=7)
    first = run(*args, 100, 0, 3)
    for a, b in zip(first, run(*args, 100, 0, 3)):
        assert torch.equal(a, b)
    q, k, v = (t.cuda() for t in args[:3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = window_attention(q, k, v, 100, 0, 3)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, first[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tokens", [(torch.bfloat16, 300), (torch.bfloat16, 1), (torch.float32, 300), (torch.float16, 300)])
def test_captured_calls_follow_their_inputs(dtype, tokens):
    """Two graphs of the same operator, replayed in turns; lengths and offsets are read at every replay."""
    shape = (2, tokens, 4, 2, 64, 300)
    graphs = []
    for seed in (8, 9):
        q, k, v, g = (t.cuda() for t in make(*shape, dtype, seed=seed))
        lengths, offsets = torch.tensor([300, 200], device="cuda"), torch.tensor([300 - tokens, 0], dtype=torch.int32, device="cuda")
        leaves = [t.requires_grad_() for t in (q, k, v)]

        def step(leaves=leaves, g=g, lengths=lengths, offsets=offsets):
            out = window_attention(*leaves, 60, 0, 2, offsets=offsets, lengths=lengths)
            return (out.detach(),) + torch.autograd.grad(out, leaves, g)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got, step, lengths))
    for length in (300, 150, 0):
        for graph, got, step, lengths in graphs:
            lengths[1] = length
            graph.replay()
        torch.cuda.synchronize()
        for graph, got, step, lengths in graphs:
            for a, b in zip(got, step()):
                assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_nothing_to_read_or_to_ask(dtype):
    for shape in ((0, 3, 2, 1, 32, 5), (2, 0, 2, 1, 32, 5), (2, 3, 2, 1, 32, 0)):
        q, k, v, g = make(*shape, dtype)
        for got, like in zip(run(q, k, v, g, 4, 0, 1), (q, q, k, v)):
            assert got.shape == like.shape and not bool(got.any())


@pytest.mark.gpu
def test_a_gradient_of_the_gradient_is_refused():
    q, k, v, g = (t.cuda().requires_grad_() for t in make(1, 8, 1, 1, 16, 8, torch.float32))
    grad, = torch.autograd.grad(window_attention(q, k, v, 2), q, g, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        grad.sum().backward()


def test_refusals():
    q, k, v, _ = make(2, 3, 4, 2, 16, 5, torch.float32)
    with pytest.raises(RuntimeError, match="window_attention is not implemented on CPU"):
        window_attention(q, k, v, 2)
    with pytest.raises(RuntimeError, match="not implemented for 'float64'"):
        window_attention(q.double(), k, v, 2)
    with pytest.raises(RuntimeError, match="expected scalar type"):
        window_attention(q, k.half(), v, 2)
    with pytest.raises(RuntimeError, match="expected query"):
        window_attention(q[0], k, v, 2)
    with pytest.raises(RuntimeError, match="same shape"):
        window_attention(q, k, v[:, 1:], 2)
    with pytest.raises(RuntimeError, match="same head size"):
        window_attention(q[..., :8], k, v, 2)
    with pytest.raises(RuntimeError, match="of the same sequences"):
        window_attention(q[:1], k, v, 2)
    with pytest.raises(RuntimeError, match="heads"):
        window_attention(q[:, :, :3], k, v, 2)
    with pytest.raises(RuntimeError, match="at most 256|head size"):
        window_attention(*(torch.zeros(2, 3, 2, 257) for _ in range(3)), 2)
    for bad in ((-1, 0, 0), (0, -1, 0), (0, 0, -1)):
        with pytest.raises(RuntimeError, match="must not be negative"):
            window_attention(q, k, v, *bad)
    with pytest.raises(TypeError):
        window_attention(q, k, v, 2.5)
    with pytest.raises(ValueError, match="64 bits"):
        window_attention(q, k, v, 2 ** 70)
    with pytest.raises(RuntimeError, match="scale must be finite"):
        window_attention(q, k, v, 2, scale=math.inf)
    for kw in (dict(lengths=torch.zeros(3, dtype=torch.int32)), dict(offsets=torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="one element per sequence"):
            window_attention(q, k, v, 2, **kw)
    for name in ("lengths", "offsets"):
        with pytest.raises(RuntimeError, match="must be int32 or int64"):
            window_attention(q, k, v, 2, **{name: torch.zeros(2)})


def test_the_library_refuses_before_it_launches():
    lib = _lib.lib
    a = _lib.Attention(dtype=0, R=2, T=3, Hq=4, Hk=2, N=2, L=5, D=16)
    w = _lib.Window(before=2)
    size = ctypes.c_int64()
    assert lib.mvr_window_attention_workspace(a, w, 0, size) == 0
    assert lib.mvr_window_attention_workspace(None, w, 0, size) == lib.mvr_window_attention_workspace(a, None, 0, size) == -6
    assert lib.mvr_window_attention_forward(a, w, None, 0, None, None) == -6
    for field, value, code in (("dtype", 2, -1), ("R", 1, -5), ("Hq", 3, -15), ("D", 257, -16), ("has_index", 1, -13), ("mask", 16, -13), ("L", 2 ** 40, -9)):
        b = _lib.Attention(dtype=0, R=2, T=3, Hq=4, Hk=2, N=2, L=5, D=16)
        setattr(b, field, value)
        assert lib.mvr_window_attention_workspace(b, w, 0, size) == code, field
    for field in ("before", "after", "sinks"):
        assert lib.mvr_window_attention_workspace(a, _lib.Window(**{field: -1}), 0, size) == -19
    assert "negative" in _lib.strerror(-19)
    big = _lib.Attention(dtype=0, R=1, T=4096, Hq=4, Hk=2, N=1, L=4096, D=32, q=16, k=16, v=16, out=16)
    assert lib.mvr_window_attention_workspace(big, _lib.Window(before=600), 0, size) == 0 and size.value > 0
    assert lib.mvr_window_attention_forward(big, _lib.Window(before=600), None, 0, None, None) == -14


def parts_of(case):
    """The host's cut of a call, restated: each (tile of states, part of rows) and (tile of rows, part of states) walked once."""
    T, G, L, before, after, sinks, offset, length, step, tile, parts, sink_parts, per = case
    token = lambda x: max(0, min(x, T))  # noqa: E731
    sink_tiles, seen = -(-min(sinks, L) // tile), set()
    for t in range(-(-L // tile)):
        j0, sink = t * tile, t < sink_tiles
        lo = token(j0 - after - offset) * G
        hi = (T if j0 < sinks else token(min(j0 + tile, length) - 1 + before + 1 - offset)) * G
        count = -(-max(0, hi - lo) // step)
        each = -(-count // sink_parts) if sink else per
        walked = [p * each + i for p in range(sink_parts if sink else parts) for i in range(max(0, min(each, count - p * each)))]
        assert walked == list(range(count)) and (sink or parts * per >= count)
        seen.update((t, row) for i in walked for row in range(lo + i * step, lo + (i + 1) * step))
    ok = allowed_states(T, L, before, after, sinks, offset, length)
    for i, j in ok.nonzero().tolist():
        for g in range(G):
            assert (j // tile, i * G + g) in seen
    return seen


@pytest.mark.parametrize("offset", [-20, 0, 7, 300])
@pytest.mark.parametrize("window", [(0, 0, 0), (9, 0, 3), (30, 12, 40), (500, 500, 1)])
def test_every_pair_is_walked_once(window, offset):
    """The index arithmetic of the gradients of keys and values, on the CPU: every row that reads a state is in exactly one part's walk."""
    before, after, sinks = window
    for T, L, G, length in ((60, 60, 1, 60), (90, 50, 3, 41), (1, 100, 4, 100), (64, 33, 2, 0)):
        reached = min(T, 16 + before + after) * G
        for step, tile in ((8, 16), (16, 16)):
            for parts in (1, 3):
                per = max(1, -(-min(-(-T * G // step), -(-reached // step) + 1) // parts))
                sink_parts = max(1, min(64, -(-(-(-T * G // step)) // per)))
                parts_of((T, G, L, before, after, sinks, offset, length, step, tile, parts, sink_parts, per))
