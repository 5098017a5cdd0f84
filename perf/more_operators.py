"""Operators of an encoder's blocks over channels-last states, as cases of one benchmark.

Families (key ``op``):
  norm     group norm with its activation over (images, states, channels): ops.group_norm
  rotary   rotary positions of several axes on queries and keys: ops.rotary_positions
  window   attention in a sliding window, with first states that stay visible: ops.window_attention

``own`` selects between the plain forms of this file (elementary torch operations in 32 bits, angles in 64) and the package's operators.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
INDEX = {"i32": torch.int32, "i64": torch.int64, "f32": torch.float32}


def listed():
    return [
        # inference on one region of interest: the coarsest map of an encoder; latency counts
        dict(name="coarse_map_norm", op="norm", dtype="f16", images=2, states=8 ** 3, channels=256, groups=32, activation="silu", train=False),
        # training step: a map in the middle of a 3D encoder
        dict(name="middle_map_norm", op="norm", dtype="f16", images=2, states=48 ** 3, channels=64, groups=16, activation="silu", train=True),
        # training step in single precision: 101 x 135 slices, channels and groups that are no powers of two
        dict(name="odd_map_norm", op="norm", dtype="f32", images=3, states=13635, channels=84, groups=7, activation="gelu", train=True),
        # training step: the finest map of a 3D network, larger than the L2 cache
        dict(name="fine_map_norm", op="norm", dtype="bf16", images=2, states=128 ** 3, channels=32, groups=8, activation="silu", train=True),
        # serving: queries and keys of one new token of every sequence
        dict(name="token_rotary", op="rotary", dtype="bf16", images=32, states=1, heads=32, kv_heads=8, dim=128, sections="24+20+20", base=1e4,
             interleaved=False, positions="i32", far=16384, train=False),
        # training step: queries and keys of a 16^3 map, three axes
        dict(name="volume_rotary", op="rotary", dtype="f16", images=2, states=16 ** 3, heads=8, kv_heads=8, dim=32, sections="6+5+5", base=1e4,
             interleaved=True, positions="f32", far=512, train=True),
        # training step: queries and shared keys of a batch of slices, rows and columns
        dict(name="slices_rotary", op="rotary", dtype="bf16", images=8, states=13635, heads=16, kv_heads=4, dim=64, sections="16+16", base=1e4,
             interleaved=False, positions="i64", far=1000000, train=True),
        # serving: one new token per sequence over a long cache, of which the last 2048 states and four first ones are read
        dict(name="token_window", op="window", dtype="bf16", sequences=32, tokens=1, states=16384, heads=32, kv_heads=8, dim=128, before=2047, after=0,
             sinks=4, ends="lengths", train=False),
        # training step on half a slice: neighbours on both sides of a scan line, in half precision
        dict(name="both_sides_window", op="window", dtype="f16", sequences=4, tokens=4096, states=4096, heads=8, kv_heads=8, dim=32, before=135, after=135,
             sinks=0, ends="all", train=True),
        # training step in single precision: sequences of different lengths, one of them empty
        dict(name="ragged_window", op="window", dtype="f32", sequences=3, tokens=2047, states=2047, heads=4, kv_heads=4, dim=64, before=300, after=0,
             sinks=1, ends="padded", train=True),
        # training step of a block over long sequences of slices, shared key heads
        dict(name="slices_window", op="window", dtype="bf16", sequences=2, tokens=8192, states=8192, heads=16, kv_heads=4, dim=64, before=1023, after=0,
             sinks=4, ends="all", train=True),
        # inference over whole studies: the largest product
        dict(name="study_window", op="window", dtype="bf16", sequences=2, tokens=32768, states=32768, heads=16, kv_heads=16, dim=128, before=4095, after=0,
             sinks=16, ends="all", train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "rotary", "window", "window", "window"])
    dtype = rng.choice(["f16", "bf16", "f32"])
    if op == "norm":
        while True:
            groups = rng.choice([1, 2, 4, 5, 7, 8, 16, 32])
            channels = groups * rng.choice([1, 2, 3, 4, 8, 12, 16, 32])
            train = rng.random() < 0.6
            # (where the derivative of a relu jumps, one rounding decides over a whole gradient: inference only)
            case = dict(op="norm", dtype=dtype, images=rng.randint(1, 8), states=_log(rng, 1, 2000000), channels=channels, groups=groups,
                        activation=rng.choice(["none", "silu", "gelu"] + ([] if train else ["relu"])), train=train)
            # (gradients of a group of a few values cancel to nothing)
            if train and case["states"] * channels < 16 * groups:
                continue
            if case["images"] * case["states"] * channels <= (6e7 if dtype == "f32" else 1.2e8):
                return case
    if op == "rotary":
        while True:
            kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4])
            dim = rng.choice([16, 24, 32, 33, 64, 64, 72, 96, 128, 128, 256])
            axes = rng.randint(1, 4)
            cut = sorted(rng.randint(0, dim // 2) for _ in range(axes)) if rng.random() < 0.5 else [dim // 2 * (i + 1) // axes for i in range(axes)]
            images = _log(rng, 1, 64)
            case = dict(op="rotary", dtype=dtype, images=images, states=rng.choice([1, _log(rng, 2, 20000), _log(rng, 2, 20000)]), heads=kv_heads * group,
                        kv_heads=kv_heads, dim=dim, sections="+".join(str(b - a) for a, b in zip([0] + cut, cut)), base=rng.choice([100.0, 1e4, 5e5]),
                        interleaved=rng.random() < 0.5, positions=rng.choice(["i32", "i64", "f32"]), far=_log(rng, 16, 1000000), train=rng.random() < 0.6)
            if images * case["states"] * (case["heads"] + kv_heads) * dim <= (6.5e7 if dtype == "f32" else 1.3e8):
                return case
    while True:
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4, 8])
        cache = rng.random() < 0.4
        states = _log(rng, 3, 32768)
        tokens = min(states, rng.choice([1, 1, 2, 5, 64])) if cache else states
        case = dict(op="window", dtype=dtype, sequences=_log(rng, 1, 48) if cache else rng.randint(1, 4), tokens=tokens, states=states, heads=kv_heads * group,
                    kv_heads=kv_heads, dim=rng.choice([16, 24, 32, 33, 64, 64, 80, 96, 128, 128]), before=_log(rng, 1, 8192) - 1,
                    after=rng.choice([0, 0, _log(rng, 1, 1000)]), sinks=rng.choice([0, 1, 4, 16, 130]),
                    ends="lengths" if cache else rng.choice(["all", "padded"]), train=not cache and rng.random() < 0.6)
        pairs = case["sequences"] * tokens * case["heads"] * min(states, case["before"] + 1 + case["after"] + case["sinks"])
        cost = pairs * case["dim"] * (14 if case["train"] else 4)
        if cost < (4e11 if dtype != "f32" else 1e11) and case["sequences"] * states * kv_heads * case["dim"] < 3e8:
            return case


# ---- what a case has beside its seed ------------------------------------------------------------------


def _sections(case):
    """Pairs of columns of every axis."""
    return [int(n) for n in case["sections"].split("+")]


def _lengths(case):
    """Valid states of every sequence: from all of them down to about half, unevenly; of three padded sequences or more one has none."""
    n, s = case["sequences"], case["states"]
    if case["ends"] == "all":
        return [s] * n
    lengths = [s - (s * ((5 * k) % n)) // (2 * n) for k in range(n)]
    if case["ends"] == "padded" and n >= 3:
        lengths[n - 2] = 0
    return lengths


def _offsets(case):
    """Place of the first token: a cache ends with the new tokens, a whole sequence begins with them."""
    if case["ends"] == "lengths":
        return [max(0, length - case["tokens"]) for length in _lengths(case)]
    return [0] * case["sequences"]


def _pairs(case):
    """Tokens and states that meet, and states that any token reads, over all sequences (of one head)."""
    pairs = states = 0
    before, after, sinks, tokens = case["before"], case["after"], case["sinks"], case["tokens"]
    for length, offset in zip(_lengths(case), _offsets(case)):
        place = torch.arange(offset, offset + tokens, dtype=torch.int64)
        end = torch.clamp(place + after + 1, max=length)
        begin = torch.clamp(place - before, min=0)
        first = torch.clamp(end, max=sinks)
        pairs += int((torch.clamp(end - begin, min=0) + first - torch.clamp(first - begin, min=0)).sum())
        lowest, highest = int(begin.min()), int(end.max())
        head = min(sinks, highest)
        states += max(0, highest - lowest) + head - max(0, head - lowest) if highest > lowest else head
    return pairs, states


# ---- inputs -------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]

    def normal(*shape, dtype=t):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    state = dict(case)
    if case["op"] == "norm":
        n, s, c = case["images"], case["states"], case["channels"]
        x = torch.randn(n, s, c, generator=g, device="cuda")
        # what a convolution leaves: every channel with a mean and a spread of its own
        x.mul_(torch.rand(c, generator=g, device="cuda") * 1.5 + 0.5).add_(torch.randn(c, generator=g, device="cuda"))
        state["x"] = x.to(t)
        state["weight"] = 1 + 0.2 * torch.randn(c, generator=g, device="cuda")
        state["bias"] = 0.2 * torch.randn(c, generator=g, device="cuda")
        if case["train"]:
            state["grad"] = normal(n, s, c)
            for k in ("x", "weight", "bias"):
                state[k].requires_grad_(True)
    elif case["op"] == "rotary":
        n, s, d = case["images"], case["states"], case["dim"]
        # queries and keys as a projection leaves them: parts of the same rows
        rows = normal(n, s, case["heads"] + case["kv_heads"], d)
        state["query"], state["key"] = rows.split([case["heads"], case["kv_heads"]], 2)
        at = torch.rand(n, s, len(_sections(case)), generator=g, device="cuda") * case["far"]
        state["at"] = at.to(INDEX[case["positions"]])
        if case["train"]:
            state["grads"] = [normal(*state["query"].shape), normal(*state["key"].shape)]
            for k in ("query", "key"):
                state[k].requires_grad_(True)
    else:
        n, s, d = case["sequences"], case["states"], case["dim"]
        state["query"] = normal(n, case["tokens"], case["heads"], d)
        state["key"], state["value"] = normal(n, s, case["kv_heads"], d), normal(n, s, case["kv_heads"], d)
        state["lengths"] = state["offsets"] = None
        if case["ends"] != "all":
            state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        if case["ends"] == "lengths":
            state["offsets"] = torch.tensor(_offsets(case), dtype=torch.int32, device="cuda")
        if case["train"]:
            state["grad"] = normal(n, case["tokens"], case["heads"], d)
            for k in ("query", "key", "value"):
                state[k].requires_grad_(True)
    return state


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "rotary": _plain_rotary, "window": _plain_window}[state["op"]](state)


def _own(state):
    from medvision_b200 import ops
    if state["op"] == "norm":
        inputs = state["x"], state["weight"], state["bias"]
        activation = None if state["activation"] == "none" else state["activation"]
        out = ops.group_norm(state["x"], state["groups"], state["weight"], state["bias"], eps=1e-5, activation=activation)
        if not state["train"]:
            return out
        return (out.detach(),) + torch.autograd.grad(out, inputs, state["grad"])
    if state["op"] == "rotary":
        out = ops.rotary_positions(state["query"], state["at"], key=state["key"], sections=_sections(state), base=state["base"],
                                   interleaved=state["interleaved"])
        if not state["train"]:
            return out
        return tuple(o.detach() for o in out) + torch.autograd.grad(out, (state["query"], state["key"]), state["grads"])
    inputs = state["query"], state["key"], state["value"]
    out = ops.window_attention(*inputs, before=state["before"], after=state["after"], sinks=state["sinks"], offsets=state["offsets"],
                               lengths=state["lengths"])
    if not state["train"]:
        return out
    return (out.detach(),) + torch.autograd.grad(out, inputs, state["grad"])


# ---- plain forms --------------------------------------------------------------------------------------


def _plain_norm(st):
    """act((x - mean) / sqrt(var + eps) weight + bias) with mean and variance of an image's group of channels, and its gradients."""
    x = st["x"]
    n, s, c = x.shape
    k = st["groups"]
    values = x.float().reshape(n, s, k, c // k)
    mean = values.mean((1, 3), keepdim=True)
    centred = values - mean
    inverse = 1.0 / torch.sqrt((centred * centred).mean((1, 3), keepdim=True) + 1e-5)
    xhat = centred * inverse
    weight, bias = st["weight"].reshape(k, -1), st["bias"].reshape(k, -1)
    z = xhat * weight + bias
    kind = st["activation"]
    if kind == "silu":
        gate = 1.0 / (1.0 + torch.exp(-z))
        out, slope = z * gate, gate * (1.0 + z * (1.0 - gate))
    elif kind == "gelu":
        gate = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        out, slope = z * gate, gate + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    else:
        out, slope = (torch.where(z > 0, z, 0.0), None) if kind == "relu" else (z, torch.ones_like(z))
    out = out.reshape(n, s, c).to(x.dtype)
    if not st["train"]:
        return out
    grad = st["grad"].float().reshape(n, s, k, c // k) * slope
    grad_bias, grad_weight = grad.sum((0, 1)).reshape(c), (grad * xhat).sum((0, 1)).reshape(c)
    grad = grad * weight
    grad_x = inverse * (grad - grad.mean((1, 3), keepdim=True) - xhat * (grad * xhat).mean((1, 3), keepdim=True))
    return out, grad_x.reshape(n, s, c).to(x.dtype), grad_weight, grad_bias


def _plain_rotary(st):
    """Pair i of an axis with n pairs turns by position times base^(-i / n); pairs are neighbours, or a half of the turned columns apart."""
    sections = _sections(st)
    pairs = sum(sections)
    angle = torch.cat([st["at"][..., a, None].double() * st["base"] ** (-torch.arange(n, device="cuda", dtype=torch.float64) / max(n, 1))
                       for a, n in enumerate(sections)], -1)[:, :, None, :]
    cos, sin = angle.cos().float(), angle.sin().float()

    def turn(x, sin):
        y = x.float()
        a, b = (y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]) if st["interleaved"] else (y[..., :pairs], y[..., pairs:2 * pairs])
        a, b = a * cos - b * sin, a * sin + b * cos
        turned = torch.stack((a, b), -1).flatten(-2) if st["interleaved"] else torch.cat((a, b), -1)
        return torch.cat((turned, y[..., 2 * pairs:]), -1).to(x.dtype)

    out = turn(st["query"], sin), turn(st["key"], sin)
    if not st["train"]:
        return out
    return out + (turn(st["grads"][0], -sin), turn(st["grads"][1], -sin))


def _plain_window(st):
    """Block by block of the tokens: softmax over the first states and the band of states that the block may read."""
    t = st["query"].dtype
    n, tokens, heads, d = st["query"].shape
    states, kv = st["key"].shape[1:3]
    group, before, after, sinks = heads // kv, st["before"], st["after"], min(st["sinks"], st["states"])
    ends = torch.full((n,), states, device="cuda") if st["lengths"] is None else st["lengths"].long()
    offsets = torch.zeros(n, dtype=torch.long, device="cuda") if st["offsets"] is None else st["offsets"].long()
    block = max(1, min(tokens, max(before + after, 128), 2 ** 28 // (n * heads * min(states, before + after + 128))))
    span = min(states, block + before + after)
    key, value = st["key"].float().reshape(n * states, kv, d), st["value"].float().reshape(n * states, kv, d)
    out = torch.zeros(n, tokens, heads, d, device="cuda")
    grad_query = torch.zeros_like(out)
    grad_key, grad_value = torch.zeros_like(key), torch.zeros_like(value)
    first = torch.arange(sinks, device="cuda").expand(n, sinks)
    for t0 in range(0, tokens, block):
        rows = min(block, tokens - t0)
        place = offsets[:, None] + t0 + torch.arange(rows, device="cuda")                              # n, rows
        band = (offsets[:, None] + t0 - before).clamp(max=states - span).clamp(min=0) + torch.arange(span, device="cuda")
        at = torch.cat((first, band), 1)                                                                # n, j
        seen = (at[:, None] <= place[:, :, None] + after) & (at < ends[:, None])[:, None]
        seen[:, :, sinks:] &= (band >= sinks)[:, None] & (band[:, None] >= place[:, :, None] - before)
        at = at + states * torch.arange(n, device="cuda")[:, None]
        k, v = key[at].permute(0, 2, 1, 3), value[at].permute(0, 2, 1, 3)                               # n, kv, j, d

        def split(x):  # n, kv, rows * group, d
            return x[:, t0:t0 + rows].float().reshape(n, rows, kv, group, d).permute(0, 2, 1, 3, 4).reshape(n, kv, rows * group, d)

        def merge(x):
            return x.reshape(n, kv, rows, group, d).permute(0, 2, 1, 3, 4).reshape(n, rows, heads, d)

        q = split(st["query"])
        closed = ~seen[:, None, :, None].expand(n, 1, rows, group, seen.shape[-1]).reshape(n, 1, rows * group, -1)
        p = (q @ k.transpose(2, 3)).mul_(d ** -0.5).masked_fill_(closed, -math.inf)
        top = p.amax(-1, keepdim=True)
        p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
        total = p.sum(-1, keepdim=True)
        p = p.div_(torch.where(total == 0, 1.0, total))
        o = p @ v
        out[:, t0:t0 + rows] = merge(o)
        if st["train"]:
            g = split(st["grad"])
            ds = (g @ v.transpose(2, 3)).sub_((g * o).sum(-1, keepdim=True)).mul_(p).mul_(d ** -0.5)
            grad_query[:, t0:t0 + rows] = merge(ds @ k)
            grad_key.index_add_(0, at.reshape(-1), (ds.transpose(2, 3) @ q).permute(0, 2, 1, 3).reshape(-1, kv, d))
            grad_value.index_add_(0, at.reshape(-1), (p.transpose(2, 3) @ g).permute(0, 2, 1, 3).reshape(-1, kv, d))
    if not st["train"]:
        return out.to(t)
    return out.to(t), grad_query.to(t), grad_key.reshape(n, states, kv, d).to(t), grad_value.reshape(n, states, kv, d).to(t)


# ---- the definitions in 64 bits -----------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "window": _exact_window}[case["op"]](state)


def _exact_norm(st):
    leaves = [st[k].detach().double().requires_grad_(st["train"]) for k in ("x", "weight", "bias")]
    x, weight, bias = leaves
    n, s, c = x.shape
    with torch.set_grad_enabled(st["train"]):
        parts = []
        for i in range(n):  # an image's groups as rows
            rows = x[i].reshape(s, st["groups"], -1).transpose(0, 1).flatten(1)
            variance, mean = torch.var_mean(rows, 1, correction=0)
            rows = (rows - mean[:, None]) * (variance[:, None] + 1e-5).rsqrt()
            parts.append(rows.reshape(st["groups"], s, -1).transpose(0, 1).reshape(s, c) * weight + bias)
        z = torch.stack(parts)
        out = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[st["activation"]](z)
        if not st["train"]:
            return out
        return (out.detach(),) + torch.autograd.grad(out, leaves, st["grad"].double())


def _exact_rotary(st):
    pairs = [(axis, st["base"] ** (-i / n)) for axis, n in enumerate(_sections(st)) for i in range(n)]
    count = len(pairs)

    def turn(x, sign):
        y = x.detach().double().clone()
        for i, (axis, frequency) in enumerate(pairs):
            angle = sign * frequency * st["at"][..., axis].double()[..., None]
            a, b = (2 * i, 2 * i + 1) if st["interleaved"] else (i, i + count)
            turned = torch.polar(torch.ones_like(angle), angle) * torch.complex(y[..., a], y[..., b])
            y[..., a], y[..., b] = turned.real, turned.imag
        return y

    out = turn(st["query"], 1), turn(st["key"], 1)
    return out + (turn(st["grads"][0], -1), turn(st["grads"][1], -1)) if st["train"] else out


def _exact_window(st):
    query, key, value = (st[k].detach().double() for k in ("query", "key", "value"))
    n, tokens, heads, d = query.shape
    states, group = st["states"], heads // st["kv_heads"]
    out, gq, gk, gv = torch.zeros_like(query), torch.zeros_like(query), torch.zeros_like(key), torch.zeros_like(value)
    state = torch.arange(states, device="cuda")
    for i, (length, offset) in enumerate(zip(_lengths(st), _offsets(st))):
        for t0 in range(0, tokens, 4096):
            t1 = min(tokens, t0 + 4096)
            place = torch.arange(offset + t0, offset + t1, device="cuda")[:, None]
            allowed = (state < length) & (state <= place + st["after"]) & ((state >= place - st["before"]) | (state < st["sinks"]))
            for h in range(heads):
                q, k, v = query[i, t0:t1, h], key[i, :, h // group], value[i, :, h // group]
                logits = torch.where(allowed, q @ k.T / math.sqrt(d), -math.inf)
                w = torch.nan_to_num(torch.softmax(logits, 1), nan=0.0)  # (rows that read nothing)
                out[i, t0:t1, h] = w @ v
                if st["train"]:
                    g = st["grad"][i, t0:t1, h].double()
                    dw = g @ v.T
                    dx = w * (dw - (w * dw).sum(1, keepdim=True)) / math.sqrt(d)
                    gq[i, t0:t1, h] = dx @ k
                    gk[i, :, h // group] += dx.T @ q
                    gv[i, :, h // group] += w.T @ g
    return (out, gq, gk, gv) if st["train"] else out


# ---- what a pass cannot do without --------------------------------------------------------------------


def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "norm":
        n = case["images"] * case["states"] * case["channels"]
        small = 4 * case["channels"] * (4 if case["train"] else 2)
        # x in, y out; with gradients the gradient in and that of x out (x, kept or read again, counts once)
        return {"bytes": b * n * (4 if case["train"] else 2) + small, "flops": n * (25 if case["train"] else 8)}
    if case["op"] == "rotary":
        rows = case["images"] * case["states"]
        n = rows * (case["heads"] + case["kv_heads"]) * case["dim"]
        at = rows * len(_sections(case)) * (8 if case["positions"] == "i64" else 4)
        passes = 2 if case["train"] else 1
        turned = rows * (case["heads"] + case["kv_heads"]) * sum(_sections(case))
        return {"bytes": 2 * b * n * passes + at, "flops": 6 * turned * passes}
    pairs, states = _pairs(case)
    rows = case["sequences"] * case["tokens"] * case["heads"] * case["dim"]
    read = states * case["kv_heads"] * case["dim"]
    whole = case["sequences"] * case["states"] * case["kv_heads"] * case["dim"]
    pairs *= case["heads"] * case["dim"]
    if case["train"]:
        # query, output and gradient in, gradient of the query out; states that are read in, gradients of all states out
        return {"bytes": b * (4 * rows + 2 * read + 2 * whole), "flops": 14 * pairs}
    return {"bytes": b * (2 * rows + 2 * read), "flops": 4 * pairs}
