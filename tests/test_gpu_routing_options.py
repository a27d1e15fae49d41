"""
RasterStep's routing options: inputs that the caller changes in place between steps, and the kernels a step launches.
"""
import pytest
import torch

from common import make_case, to_dev
from igs_b200 import ops, pipeline

pytestmark = pytest.mark.gpu


def build(device, h=40, w=56, n=150, seed=41, **options):
    _, inp = make_case(h, w, n, seed=seed)
    d = to_dev(inp, device)
    return pipeline.RasterStep(d["means"], d["scales"], d["rotations"], d["features"], d["target"], **options)


@pytest.mark.parametrize("replayed", [False, True])
@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8])
@pytest.mark.parametrize("layout", ["contiguous", "transposed", "every second column", "one row for all"])
def test_mask_is_read_anew_by_every_step(layout, dtype, replayed, device):
    """A mask of any strides that the caller changes in place: each step equals the operator's result under the mask of the moment."""
    h, w = 40, 56
    mask = {"contiguous": lambda: torch.ones(h, w, dtype=dtype, device=device),
            "transposed": lambda: torch.ones(w, h, dtype=dtype, device=device).t(),
            "every second column": lambda: torch.ones(h, 2 * w, dtype=dtype, device=device)[:, ::2],
            "one row for all": lambda: torch.ones(w, dtype=dtype, device=device).expand(h, w)}[layout]()
    base = mask[0] if layout == "one row for all" else mask
    step = build(device, h, w, balance=dict(factor=0.05, mask=mask))
    seen = []
    for keep in (1.0, 0.6, 0.2):
        base.copy_(torch.rand(base.shape, device=device) < keep)
        step.replay() if replayed else step.launch()
        want = ops.topk_balance_forward(h, w, step.xys, step.conics, step.pixel_topk, mask.contiguous())
        for a, b in zip((step.balance_loss, step.counts, step.importance, step.totals), want):
            assert torch.equal(a, b)
        seen.append(int(step.totals[0]))
    assert seen[0] > seen[1] > seen[2]
