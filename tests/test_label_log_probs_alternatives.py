"""ops.label_log_probs: alternatives of positions with few classes of any probability, with NaN and infinities, in every kernel.

Order: NaN first, then the larger score, equal ones by class.  The alternatives' log-probabilities are compared where they are finite:
a difference of two floats and a logarithm of a sum of K exponentials (8 sqrt(K) e and a rounding of the difference)."""
import math

import pytest
import torch

from medvision_b200.ops import label_log_probs

E = 2.0 ** -24


def scores(shape, dtype, kind, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g) * 4).round() / 2                      # many equal ones
    share = torch.rand((shape[0], 1) + shape[2:], generator=g) * 1.2           # classes without probability: from none to all
    x[torch.rand(shape, generator=g) < share] = -float("inf")
    if kind != "finite":
        few = torch.rand(shape, generator=g) < 0.6 / shape[1]
        x[few] = float(kind)
    return x.to(dtype)


def check(x, top):
    labels = torch.zeros((x.shape[0],) + tuple(x.shape[2:]), dtype=torch.int32, device="cuda")
    leaf = x.cuda().requires_grad_()
    got = label_log_probs(leaf, labels, top)
    key = x.float().nan_to_num(nan=1e30, posinf=1e20, neginf=-1e30)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_label.cpu().long(), order)
    logs = torch.log_softmax(x.double(), 1).gather(1, order)
    empty = (x == -float("inf")).all(1, keepdim=True).expand_as(logs)          # all -inf: -inf
    logs = torch.where(empty, -float("inf"), logs)
    value = got.top_log_prob.cpu().double()
    assert torch.equal(value.isnan(), logs.isnan()) and torch.equal(value == -float("inf"), logs == -float("inf"))
    fine = logs.isfinite()
    bound = (8 * math.sqrt(x.shape[1]) + 4 + 6 * logs.abs()) * E
    assert bool(((value - logs).abs() <= bound)[fine].all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["finite", "nan", "inf"])
@pytest.mark.parametrize("K", [1, 3, 8, 14, 16, 40])
@pytest.mark.parametrize("space", [(2, 30), (1, 33), (7, 1, 37)])
def test_maps(space, K, kind, dtype):
    for top in sorted({min(K, t) for t in (1, 2, 3, 5, 8, 16)}):
        x = scores((3, K) + space, dtype, kind, top)
        check(x, top)
        check(x.movedim(1, -1).contiguous().movedim(-1, 1), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["finite", "nan", "inf"])
@pytest.mark.parametrize("K", [2, 50, 129, 700, 1025, 1700, 5001, 20000, 70001])
def test_rows(K, kind, dtype):
    for top in sorted({min(K, t) for t in (1, 3, 16)}):
        check(scores((12, K), dtype, kind, top), top)
