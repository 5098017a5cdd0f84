"""ops.dropout: results that lie over x or over the residual."""
import ctypes

import pytest
import torch

from medvision_b200 import _lib
from medvision_b200.ops import dropout


def test_nothing_is_copied_where_the_result_is_the_residual():
    """p = 1 leaves the residual: with the result over it there is nothing to do, and no copy of memory onto itself."""
    assert _lib.lib.mvr_dropout(16, 32, 32, 0, 4, 1.0, 1, None, 0, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.3, 1.0])
def test_results_over_x_and_over_the_residual(p):
    x, r = torch.randn(1000, device="cuda"), torch.randn(1000, device="cuda")
    want, alone = dropout(x, p, 5, residual=r), dropout(x, p, 5)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    at = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    for residual, over, expected in ((r, "r", want), (r, "x", want), (None, "x", alone)):
        a, b = x.clone(), r.clone()
        out = a if over == "x" else b
        assert _lib.lib.mvr_dropout(at(a), None if residual is None else at(b), at(out), 0, 1000, p, 5, None, 0, stream) == 0
        assert torch.equal(out, expected), (p, over)
