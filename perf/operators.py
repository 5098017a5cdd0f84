"""Operators of the layers behind the roi modules, as cases of one benchmark.

Families (key ``op``):
  attention   regions (or any queries) read an encoder's states of another length: ops.cross_attention
  dropout     dropout from a counter-based generator, alone or with the residual's addition: ops.dropout
  labels      log-probabilities of given labels, entropy, best alternatives and the gradient of the logits: ops.label_log_probs

``own`` selects between the plain forms of this file (elementary torch operations in 32 bits) and the package's operators.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # inference of a detection head on a handful of proposals: one query per region, a small feature map; latency counts
        dict(name="regions_infer", op="attention", dtype="f16", regions=16, tokens=1, images=2, heads=8, kv_heads=8, dim=32,
             states=1024, valid="all", indexed=True, train=False),
        # training step: the 7x7 bins that RoIAlign pools for every region read the states of a 16^3 encoder map
        dict(name="bins_train", op="attention", dtype="f16", regions=128, tokens=49, images=2, heads=8, kv_heads=8, dim=32,
             states=4096, valid="all", indexed=True, train=True),
        # training step in single precision: regions read a 101x135 map of which a body mask leaves a part, and in one image nothing
        dict(name="masked_map_train", op="attention", dtype="f32", regions=200, tokens=1, images=3, heads=4, kv_heads=4, dim=64,
             states=13635, valid="mask", indexed=True, train=True),
        # training step of a decoder block: many queries, shared key heads, images with different numbers of states
        dict(name="queries_train", op="attention", dtype="bf16", regions=2, tokens=2048, images=2, heads=16, kv_heads=4, dim=64,
             states=8191, valid="lengths", indexed=False, train=True),
        # serving: one new token per sequence over long states, shared key heads
        dict(name="single_tokens", op="attention", dtype="bf16", regions=32, tokens=1, images=32, heads=32, kv_heads=8, dim=128,
             states=16384, valid="lengths", indexed=False, train=False),
        # inference of a decoder block over a large map: the largest product
        dict(name="large_infer", op="attention", dtype="bf16", regions=2, tokens=4096, images=2, heads=16, kv_heads=16, dim=128,
             states=8192, valid="all", indexed=False, train=False),
        # training step of a head's hidden features: the smallest dropout
        dict(name="features_dropout", op="dropout", dtype="f32", rows=128, cols=256, p=0.5, residual=False, train=True),
        # training step of a decoder block: a branch joins the residual stream
        dict(name="residual_dropout", op="dropout", dtype="bf16", rows=8 * 13635, cols=256, p=0.1, residual=True, train=True),
        # augmentation: voxels dropped out of a batch of volumes
        dict(name="voxel_dropout", op="dropout", dtype="f16", rows=16 * 128, cols=128 * 128, p=0.25, residual=False, train=False),
        # inference of a classification head: class of a few regions with its alternatives; latency counts
        dict(name="regions_labels", op="labels", dtype="f32", batch=16, classes=81, space=1, top=5, train=False),
        # training step of a segmentation network: one label per voxel, a part of them not given
        dict(name="voxels_train", op="labels", dtype="f16", batch=2, classes=14, space=96 * 96 * 96, top=2, train=True),
        # training step over a long list of labels
        dict(name="long_list_train", op="labels", dtype="bf16", batch=2000, classes=32001, space=1, top=8, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "dropout", "labels", "labels"])
    if op == "attention":
        while True:
            indexed = rng.random() < 0.5
            images = rng.randint(1, 4) if indexed else _log(rng, 1, 48)
            regions = _log(rng, 1, 512) if indexed else images
            tokens = rng.choice([1, 1, 4, 9, 49]) if indexed else rng.choice([1, _log(rng, 2, 4096), _log(rng, 2, 4096)])
            kv_heads, group = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 1, 1, 2, 4, 8])
            case = dict(op="attention", dtype=rng.choice(["f16", "f16", "bf16", "bf16", "f32"]), regions=regions, tokens=tokens,
                        images=images, heads=kv_heads * group, kv_heads=kv_heads, dim=rng.choice([16, 24, 32, 32, 64, 64, 72, 96, 128, 128, 20, 33]),
                        states=_log(rng, 7, 16384), valid=rng.choice(["all", "lengths", "mask"]), indexed=indexed,
                        train=rng.random() < 0.5)
            scores = regions * tokens * case["heads"] * case["states"]
            gathered = regions * case["states"] * kv_heads * case["dim"]
            if scores < 3e8 and gathered < 5e8 and scores * case["dim"] * (14 if case["train"] else 4) < 3e11 / (4 if case["dtype"] == "f32" else 1):
                return case
    dtype = rng.choice(["f16", "bf16", "f32"])
    if op == "dropout":
        return dict(op="dropout", dtype=dtype, rows=_log(rng, 1, 20000), cols=_log(rng, 8, 1500), p=round(rng.uniform(0.02, 0.7), 3),
                    residual=rng.random() < 0.5, train=rng.random() < 0.6)
    if rng.random() < 0.5:
        classes, space, batch = _log(rng, 2, 160), _log(rng, 100, 400000), rng.randint(1, 3)
        batch = batch if batch * classes * space < 6e7 else 1
        return dict(op="labels", dtype=dtype, batch=batch, classes=classes, space=space, top=min(classes, rng.choice([0, 1, 2, 3])),
                    train=rng.random() < 0.7)
    classes = _log(rng, 2, 120000)
    return dict(op="labels", dtype=dtype, batch=_log(rng, 1, min(4000, 6e7 / classes)), classes=classes, space=1,
                top=min(classes, rng.choice([0, 1, 5, 8, 16])), train=rng.random() < 0.6)


# ---- what a case has beside its seed ------------------------------------------------------------------


def _lengths(case):
    """Valid states of every image: from all of them down to about half, unevenly."""
    n, s = case["images"], case["states"]
    return [s - (s * ((5 * k) % n)) // (2 * n) for k in range(n)]


def _mask(case):
    """A body mask over the map (as rows of about square-root length) of every image; of three images or more, one has no body at all."""
    n, s = case["images"], case["states"]
    width = max(1, math.isqrt(s))
    k = np.arange(s)
    y, x = (k // width + 0.5) * width / s * 2 - 1, (k % width + 0.5) / width * 2 - 1
    body = [((x / 0.9) ** 2 + (y / (0.55 + 0.4 * i / n)) ** 2 <= 1) for i in range(n)]
    if n >= 3:
        body[n - 2][:] = False
    return np.stack(body)


def _valid_counts(case):
    if case["valid"] == "lengths":
        return _lengths(case)
    if case["valid"] == "mask":
        return [int(v) for v in _mask(case).sum(1)]
    return [case["states"]] * case["images"]


def _image_of_region(case, seed):
    return np.random.default_rng(seed).integers(0, case["images"], case["regions"])


# ---- inputs -------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]

    def normal(*shape, dtype=t, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    state = dict(case)
    if case["op"] == "attention":
        r, n, s, d = case["regions"], case["images"], case["states"], case["dim"]
        state["query"] = normal(r, case["tokens"], case["heads"], d)
        state["key"], state["value"] = normal(n, s, case["kv_heads"], d), normal(n, s, case["kv_heads"], d)
        state["index"] = state["lengths"] = state["mask"] = None
        if case["indexed"]:
            # the first column of the regions' rois: the image as a floating number
            state["index"] = torch.tensor(_image_of_region(case, seed), dtype=torch.float32, device="cuda")
        if case["valid"] == "lengths":
            state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        if case["valid"] == "mask":
            state["mask"] = torch.tensor(_mask(case), device="cuda")
        if case["train"]:
            state["grad"] = normal(r, case["tokens"], case["heads"], d)
            for k in ("query", "key", "value"):
                state[k].requires_grad_(True)
    elif case["op"] == "dropout":
        shape = case["rows"], case["cols"]
        state["x"] = normal(*shape)
        state["add"] = normal(*shape) if case["residual"] else None
        state["key64"] = random.Random(seed).getrandbits(63)
        if case["train"]:
            state["grad"] = normal(*shape)
            state["x"].requires_grad_(True)
            if case["residual"]:
                state["add"].requires_grad_(True)
    else:
        b, c, s = case["batch"], case["classes"], case["space"]
        shape = (b, c) if s == 1 else (b, c, s)
        state["logits"] = normal(*shape, scale=2.0)
        label = torch.randint(0, c, (b,) if s == 1 else (b, s), generator=g, device="cuda", dtype=torch.int32)
        state["label"] = torch.where(torch.rand(label.shape, generator=g, device="cuda") < 0.1, -1, label)
        if case["train"]:
            state["grad_log_prob"] = normal(*label.shape, dtype=torch.float32)
            state["grad_entropy"] = normal(*label.shape, dtype=torch.float32, scale=0.1)
            state["logits"].requires_grad_(True)
    return state


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"attention": _plain_attention, "dropout": _plain_dropout, "labels": _plain_labels}[state["op"]](state)


def _own(state):
    from medvision_b200 import ops
    if state["op"] == "attention":
        inputs = state["query"], state["key"], state["value"]
        out = ops.cross_attention(*inputs, batch_index=state["index"], lengths=state["lengths"], mask=state["mask"])
        if not state["train"]:
            return out
        return (out.detach(),) + torch.autograd.grad(out, inputs, state["grad"])
    if state["op"] == "dropout":
        out = ops.dropout(state["x"], state["p"], seed=state["key64"], residual=state["add"])
        if not state["train"]:
            return out
        inputs = [v for v in (state["x"], state["add"]) if v is not None]
        return (out.detach(),) + torch.autograd.grad(out, inputs, state["grad"])
    got = ops.label_log_probs(state["logits"], state["label"], top=state["top"])
    outputs = [got.log_prob.detach(), got.entropy.detach()]
    if state["top"]:
        outputs += [got.top_log_prob, got.top_label]
    if state["train"]:
        outputs += torch.autograd.grad((got.log_prob, got.entropy), (state["logits"],),
                                       (state["grad_log_prob"], state["grad_entropy"]))
    return tuple(outputs)


# ---- plain forms --------------------------------------------------------------------------------------


def _plain_attention(st):
    """softmax(Q K^T / sqrt(d)) V over the states that are valid; a query with none reads zeros."""
    t = st["query"].dtype
    r, q, h, d = st["query"].shape
    n, s, hk, _ = st["key"].shape
    allowed = torch.ones(n, s, dtype=torch.bool, device="cuda")
    if st["lengths"] is not None:
        allowed = torch.arange(s, device="cuda") < st["lengths"][:, None]
    if st["mask"] is not None:
        allowed = st["mask"]
    key, value = st["key"].float(), st["value"].float()
    if st["index"] is not None:
        at = st["index"].long()
        key, value, allowed = key[at], value[at], allowed[at]
    key, value = key.permute(0, 2, 1, 3), value.permute(0, 2, 1, 3)                                  # r, hk, s, d
    query = st["query"].float().reshape(r, q, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(r, hk, -1, d)  # r, hk, q * group, d
    closed = ~allowed[:, None, None, :]
    p = (query @ key.transpose(2, 3)).mul_(d ** -0.5).masked_fill_(closed, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    out = p @ value

    def rows(x):
        return x.reshape(r, hk, q, h // hk, d).permute(0, 2, 1, 3, 4).reshape(r, q, h, d).to(t)

    if not st["train"]:
        return rows(out)
    grad = st["grad"].float().reshape(r, q, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(r, hk, -1, d)
    grad_value = p.transpose(2, 3) @ grad
    ds = grad @ value.transpose(2, 3)
    ds = ds.sub_((grad * out).sum(-1, keepdim=True)).mul_(p).mul_(d ** -0.5)
    grad_query = ds @ key
    grad_key = ds.transpose(2, 3) @ query

    def states(x):
        x = x.permute(0, 2, 1, 3)
        if st["index"] is not None:
            x = torch.zeros(n, s, hk, d, device="cuda").index_add_(0, at, x)
        return x.to(t)

    return rows(out), rows(grad_query), states(grad_key), states(grad_value)


def _random_words(key64, groups):
    """Philox 4x32-10 (Salmon, Moraes, Dror, Shaw 2011) of the counters (i, 0, 0, 0), i < groups: (groups, 4) words of 32 bits as int64."""
    low = 0xFFFFFFFF
    i = torch.arange(groups, device="cuda")
    a, b, c, d = i & low, i >> 32, torch.zeros_like(i), torch.zeros_like(i)
    k0, k1 = key64 & low, key64 >> 32
    for _ in range(10):
        first, second = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = ((second >> 32) & low) ^ b ^ k0, second & low, ((first >> 32) & low) ^ d ^ k1, first & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((a, b, c, d), 1)


def _plain_dropout(st):
    """Element e takes 16 bits of word (e % 8) / 2 of counter e / 8, the low half first, and stays when they are not below
    round(65536 p); what stays is scaled by the inverse of the probability of staying."""
    x, n = st["x"], st["x"].numel()
    cut = math.floor(st["p"] * 65536 + 0.5)
    words = _random_words(st["key64"], (n + 7) // 8)
    bits = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n].reshape(x.shape)
    kept, scale = bits >= cut, 65536.0 / (65536 - cut)
    out = torch.where(kept, x.float() * scale, 0.0)
    if st["add"] is not None:
        out = out + st["add"].float()
    out = out.to(x.dtype)
    if not st["train"]:
        return out
    grads = (torch.where(kept, st["grad"].float() * scale, 0.0).to(x.dtype),)
    return (out,) + grads + ((st["grad"],) if st["add"] is not None else ())


def _plain_labels(st):
    """Log-softmax over the classes at the given labels (0 where none is given), entropy, the largest log-probabilities (ties to
    the lowest class) and the gradient of the logits."""
    x = st["logits"].float()
    label = st["label"].long()
    given = label >= 0
    at = torch.where(given, label, 0).unsqueeze(1)
    top = x.amax(1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(1, keepdim=True)
    logs = x - top - total.log()
    p = e / total
    log_prob = torch.where(given, logs.gather(1, at).squeeze(1), 0.0)
    entropy = -(p * logs).sum(1)
    outputs = [log_prob, entropy]
    if st["top"]:
        best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :st["top"]]
        outputs += [logs.gather(1, best), best.int()]
    if st["train"]:
        a = torch.where(given, st["grad_log_prob"], 0.0).unsqueeze(1)
        grad = -p * (a + st["grad_entropy"].unsqueeze(1) * (logs + entropy.unsqueeze(1)))
        outputs.append(grad.scatter_add(1, at, a).to(st["logits"].dtype))
    return tuple(outputs)


# ---- the definitions in 64 bits -----------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return {"attention": _exact_attention, "dropout": _exact_dropout, "labels": _exact_labels}[case["op"]](state)


def _exact_attention(st):
    query, key, value = (st[k].detach().double() for k in ("query", "key", "value"))
    group = st["heads"] // st["kv_heads"]
    image = list(range(st["images"])) if st["index"] is None else [int(v) for v in st["index"].tolist()]
    out = torch.zeros_like(query)
    gq, gk, gv = torch.zeros_like(query), torch.zeros_like(key), torch.zeros_like(value)
    for n in range(st["images"]):
        mine = [r for r, i in enumerate(image) if i == n]
        s = torch.arange(st["states"], device="cuda")
        if st["lengths"] is not None:
            s = s[:int(st["lengths"][n])]
        if st["mask"] is not None:
            s = s[st["mask"][n]]
        if not mine or not len(s):
            continue
        for h in range(st["heads"]):
            k, v = key[n, s, h // group], value[n, s, h // group]
            x = query[mine, :, h].reshape(-1, st["dim"])
            w = torch.softmax(torch.einsum("id,jd->ij", x, k) / math.sqrt(st["dim"]), 1)
            o = torch.einsum("ij,jd->id", w, v)
            out[mine, :, h] = o.reshape(len(mine), -1, st["dim"])
            if st["train"]:
                g = st["grad"][mine, :, h].double().reshape(-1, st["dim"])
                dw = torch.einsum("id,jd->ij", g, v)
                dx = w * (dw - torch.einsum("ij,ij->i", w, dw)[:, None]) / math.sqrt(st["dim"])
                gq[mine, :, h] = torch.einsum("ij,jd->id", dx, k).reshape(len(mine), -1, st["dim"])
                gk[n, s, h // group] += torch.einsum("ij,id->jd", dx, x)
                gv[n, s, h // group] += torch.einsum("ij,id->jd", w, g)
    return (out, gq, gk, gv) if st["train"] else out


def _exact_dropout(st):
    n = st["x"].numel()
    i = np.arange((n + 7) // 8, dtype=np.uint64)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    counter = [i & low, i >> half, np.zeros_like(i), np.zeros_like(i)]
    keys = [st["key64"] % 2 ** 32, st["key64"] // 2 ** 32]
    for turn in range(10):
        a, b = counter[0] * np.uint64(0xD2511F53), counter[2] * np.uint64(0xCD9E8D57)
        k = [np.uint64((keys[0] + turn * 0x9E3779B9) % 2 ** 32), np.uint64((keys[1] + turn * 0xBB67AE85) % 2 ** 32)]
        counter = [(b >> half) ^ counter[1] ^ k[0], b & low, (a >> half) ^ counter[3] ^ k[1], a & low]
    halves = np.stack([c.astype(np.uint32) for c in counter], 1).astype("<u4").view("<u2").reshape(-1)[:n]
    cut = math.floor(st["p"] * 65536 + 0.5)
    factor = torch.tensor(np.where(halves < cut, 0.0, 65536 / (65536 - cut))).to("cuda").reshape(st["x"].shape)
    out = st["x"].detach().double() * factor
    if st["add"] is not None:
        out = out + st["add"].detach().double()
    if not st["train"]:
        return out
    grads = (st["grad"].double() * factor,)
    return (out,) + grads + ((st["grad"].double(),) if st["add"] is not None else ())


def _exact_labels(st):
    leaf = st["logits"].detach().double().requires_grad_(True)
    logs = torch.log_softmax(leaf, 1)
    label = st["label"].long()
    log_prob = logs.gather(1, label.clamp(min=0).unsqueeze(1)).squeeze(1) * (label >= 0)
    entropy = -(logs.exp() * logs).sum(1)
    outputs = [log_prob.detach(), entropy.detach()]
    if st["top"]:
        outputs += [logs.detach().topk(st["top"], 1).values, None]
    if st["train"]:
        outputs += torch.autograd.grad((log_prob, entropy), (leaf,), (st["grad_log_prob"].double(), st["grad_entropy"].double()))
    return tuple(outputs)


# ---- what a pass cannot do without --------------------------------------------------------------------


def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "attention":
        rows = case["regions"] * case["tokens"] * case["heads"]
        counts = _valid_counts(case)
        # scores of all rows: an image's rows times its valid states (an indexed region reads any image as likely as another)
        pairs = rows * sum(counts) / case["images"]
        states = sum(counts) * case["kv_heads"] * case["dim"]
        whole = case["images"] * case["states"] * case["kv_heads"] * case["dim"]
        if case["train"]:
            # query, output and gradient in, gradient of the query out; valid states in, gradients of all states out
            return {"bytes": b * (4 * rows * case["dim"] + 2 * states + 2 * whole), "flops": 14 * pairs * case["dim"]}
        return {"bytes": b * (2 * rows * case["dim"] + 2 * states), "flops": 4 * pairs * case["dim"]}
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": b * n * (2 + case["residual"] + 2 * case["train"]), "flops": n * (1 + case["residual"] + case["train"])}
    rows = case["batch"] * case["space"]
    small = rows * (4 + 8 + 8 * case["top"] + 8 * case["train"])
    return {"bytes": b * rows * case["classes"] * (2 if case["train"] else 1) + small,
            "flops": rows * case["classes"] * (10 if case["train"] else 5)}
