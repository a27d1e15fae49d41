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


def kernel_nodes(issue):
    """How many kernels issue() launches: the kernel nodes of a graph captured from it."""
    from cuda.bindings import driver

    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        issue()
    raw = driver.CUgraph(graph.raw_cuda_graph())
    error, _, count = driver.cuGraphGetNodes(raw)
    assert error == driver.CUresult.CUDA_SUCCESS
    error, nodes, count = driver.cuGraphGetNodes(raw, count)
    assert error == driver.CUresult.CUDA_SUCCESS and len(nodes) == count
    kinds = [driver.cuGraphNodeGetType(node) for node in nodes]
    assert all(error == driver.CUresult.CUDA_SUCCESS for error, _ in kinds)
    return sum(kind == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL for _, kind in kinds)


@pytest.mark.parametrize("n", [1, 400, 401, 900])
@pytest.mark.parametrize("options", ["balance", "balance, strided mask", "dropout", "both"])
def test_kernels_per_step_are_those_that_a_step_launches(options, n, device):
    """On both sides of the Gaussians that the last CTA finishes."""
    h, w = 48, 64
    kw = {}
    if options != "dropout":
        mask = torch.ones(w, h, dtype=torch.bool, device=device).t() if "strided" in options else None
        kw["balance"] = dict(factor=0.05, mask=mask)
    if options in ("dropout", "both"):
        kw["gate_dropout"] = dict(p=0.1, rng_state=torch.zeros(2, dtype=torch.int64, device=device))
    step = build(device, h, w, n, **kw)
    step.launch()  # outside a capture first
    torch.cuda.synchronize()
    routing = [s for s in step.STAGES if s in ("_lists_forward", "_dropout_forward", "_image_loss", "_lists_backward", "_balance_term",
                                               "_next_mask")]
    assert {s: step.kernels_of(s) for s in routing} == {s: kernel_nodes(getattr(step, s)) for s in routing}
    assert step.kernels_per_step == sum(step.kernels_of(s) for s in step.STAGES) == kernel_nodes(step.launch)


def test_kernels_per_step_without_the_options(device):
    for fused in (True, False):
        step = build(device, 48, 64, 200, fused=fused)
        step.launch()
        torch.cuda.synchronize()
        assert step.kernels_per_step == kernel_nodes(step.launch)
