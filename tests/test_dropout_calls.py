"""ops.dropout: evaluation takes the residuals that training takes; a seed that is not given; results that lie over x or over the residual."""
import ctypes

import pytest
import torch

from medvision_b200 import _lib
from medvision_b200.ops import Dropout, dropout


def test_evaluation_refuses_the_residuals_that_training_refuses():
    x = torch.zeros(4, 3)
    layer = Dropout(0.5).eval()
    for residual, words in ((torch.zeros(3), "same shape"), (torch.zeros(4, 1), "same shape"), (torch.zeros(2, 4, 3), "same shape"),
                            (torch.zeros(4, 3).half(), "expected scalar type torch.float32 but found torch.float16"),
                            (torch.zeros(4, 3).double(), "expected scalar type torch.float32 but found torch.float64"),
                            (torch.zeros(4, 3, device="meta"), "same CUDA device")):
        for call in (lambda: dropout(x, 0.5, 1, residual=residual), lambda: dropout(x, 0.5, training=False, residual=residual),
                     lambda: layer(x, residual)):
            with pytest.raises(RuntimeError, match=words):
                call()
    for training in (True, False):
        with pytest.raises(TypeError, match="residual must be a Tensor, not float"):
            dropout(x, 0.5, 1, residual=1.0, training=training)
    assert layer(x) is x and torch.equal(layer(x, x + 1), x + 1)


def test_a_seed_that_is_not_given_is_drawn_on_the_cpu():
    """Also where tensors are made on another device by default: its generator could not be asked while a graph is captured."""
    x = torch.zeros(4)
    torch.manual_seed(3)
    torch.randint(2 ** 63 - 1, ())
    after = torch.rand(())
    torch.manual_seed(3)
    with torch.device("meta"), pytest.raises(RuntimeError, match="dropout is not implemented on CPU"):
        dropout(x, 0.5)
    assert torch.equal(torch.rand(()), after)


@pytest.mark.gpu
def test_a_default_device_changes_no_mask_and_no_capture():
    x = torch.randn(1000, device="cuda")
    torch.manual_seed(4)
    want = dropout(x, 0.5)
    torch.manual_seed(4)
    with torch.device("cuda"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = dropout(x, 0.5)
    graph.replay()
    assert torch.equal(out, want)


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
