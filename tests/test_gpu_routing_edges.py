"""
The operators over the top-K lists where one pixel or Gaussian could disturb another of its patch (8x8 pixels): against the float64 oracle
with the tolerances of test_gpu_routing.py.
"""
import numpy as np
import pytest
import torch

from igs_b200 import _lib, ops
from oracle import routing
from test_gpu_routing import check_balance_grad, check_dropout, to_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("others", [0, 45])
def test_large_values_stay_where_they_belong(others, device):
    """A colour of 1e32 (an importance gradient of 1e36) beside a pixel of the same patch that does not name its Gaussian, whose weights sum
    to 1e-8 so that the gate's denominator is eps: their product is past float32's range there, and counts zero times. others: further
    Gaussians in the patch, one row each; with 45 it has more rows than a group."""
    h, w, n = 8, 8, 2 + others
    rng = np.random.default_rng(91)
    xys, conics = np.zeros((n, 2)), np.tile([0.5, 0.1, 0.4], (n, 1))
    lists = np.full((h, w, 10), -1, np.int32)
    xys[0], lists[0, 0, 2] = (-6.0, 0.0), 0  # sigma 18 + 0.36 at (0, 0)
    conics[0] = (1.02, 0.0, 1.0)
    xys[1], lists[7, 7, 4] = (6.3, 7.4), 1
    for i in range(others):
        y, x = divmod(10 + i, w)
        xys[2 + i], lists[y, x, 1] = (x + 0.3, y - 0.2), 2 + i
    xys, conics = np.float32(xys), np.float32(conics)
    alpha = np.float32(rng.standard_normal(n))
    alpha[1] = 1e36
    x, k, t = to_gpu(device, xys, conics, lists)
    _, counts, _, totals = ops.topk_balance_forward(h, w, x, k, t)
    got = ops.topk_balance_backward(h, w, x, k, t, counts, totals, None, torch.from_numpy(alpha).to(device))
    _, o_counts, _, o_totals, g = routing.balance(h, w, xys, conics, lists)
    check_balance_grad(got, g, o_counts, o_totals, 0.0, alpha)
    colors, v = rng.standard_normal((n, 3)), rng.standard_normal((3, h, w))
    colors[1], v[:, 0, 0], v[:, 7, 7] = 1e32, 1e4, 1e-20
    check_dropout(h, w, xys, conics, colors, lists, 0.0, (1, 1), v, device)


def test_stream_handles_are_the_public_ones(device):
    side = torch.cuda.Stream(device)
    for stream in (torch.cuda.current_stream(device), side):
        with torch.cuda.stream(stream):
            for d in (device, device.index, "cuda:0", None):
                assert (_lib.stream_of(d).value or 0) == torch.cuda.current_stream(d).cuda_stream == stream.cuda_stream
