"""
RasterStep's routing options: inputs that the caller changes in place between steps, the kernels a step launches, and the options beside the
quantizer, the loss-space transform, the rate term and packed inputs.
"""
import pytest
import torch

from common import make_case, to_dev
from igs_b200 import autograd as ag
from igs_b200 import ops, pipeline, workloads
from test_gpu_ops import py_fixture
from test_gpu_routing_step import close, lists_of

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


def yuv_step(device, pack=False, **options):
    """The 480p YUV step (quantizer, loss-space transform, rate term) with the options, the settings, and the inputs."""
    z = py_fixture("cfg2_480p_yuv")
    wl = workloads.get_workload("cfg2_480p_yuv")
    d = to_dev(workloads.make_inputs(wl), device)
    q, transform = workloads.quant_settings(wl, device), workloads.loss_transform_yuv().to(device)
    rate = dict(model=workloads.RateModelTensors(z, device), inv_rot_step=float(z["inv_rot_step"]), factor=float(z["factor"]))
    step = pipeline.RasterStep(d["means"], d["scales"], d["rotations"], d["features"], d["loss_target"], quant=q, loss_transform=transform,
                               rate=rate, **options)
    if pack:
        step.pack_inputs()
    return step, wl, d, q, transform, rate


@pytest.mark.parametrize("p,factor,pack", [(0.15, None, False), (None, 0.02, True), (0.15, 0.02, True)])
def test_step_with_quantizer_transform_and_rate_term_matches_autograd(p, factor, pack, device):
    """Both options in the 480p YUV step, graph-captured, its inputs in one packed buffer or not, against the same step composed from the
    autograd operators; the quantities and tolerances of the step's own test without the options."""
    rng = torch.tensor([31, 4], dtype=torch.int64, device=device)
    options = {} if p is None else dict(gate_dropout=dict(p=p, rng_state=rng))
    if factor is not None:
        options["balance"] = dict(factor=factor)
    step, wl, d, q, transform, rate = yuv_step(device, pack, **options)
    step.replay()
    torch.cuda.synchronize()
    offset = int(rng[1]) - (p is not None)  # that of the replay: the step behind it has moved on
    h, w = wl.height, wl.width
    raw = [d[key].clone().requires_grad_(True) for key in ("means", "scales", "rotations", "features")]
    m, s, r, f = ag.quantize_ste(*raw, q["pos_steps"], q["scale_step"], q["rot_step"], q["feat_steps"])
    ft = f @ transform.T
    topk = lists_of(m.detach(), s.detach(), r.detach(), ft.detach(), h, w)
    xys, _, conics, _ = ag.project_gaussians_2d_scale_rot(m, s, r, h, w, ops.tile_grid(h, w))
    state = torch.tensor([31, offset], dtype=torch.int64, device=device)
    img = ag.rasterize_topk_dropout(xys, conics, ft, topk, h, w, p or 0.0, state)
    l1 = ag.l1_loss(img.permute(2, 0, 1), d["loss_target"])
    rate_term = ag.rate_loss(raw[3], raw[2], l1, rate["model"], rate["inv_rot_step"], 1.0, rate["factor"])
    balance = ag.topk_balance(xys, conics, topk, h, w)[0]
    (l1 + rate_term + (factor or 0.0) * balance).backward()
    l1, rate_term, balance = l1.detach(), rate_term.detach(), balance.detach()
    assert torch.equal(step.pixel_topk, topk)
    assert abs(float(step.loss) - float(l1)) <= 1e-5 * float(l1)
    assert abs(float(step.rate_loss) - float(rate_term)) <= 1e-5 * abs(float(rate_term))
    if factor is not None:
        assert abs(float(step.balance_loss) - float(balance)) <= 1e-5 * float(balance)
    close(step.v_mean2d, raw[0].grad, "means", 1e-3)
    close(step.v_scale, raw[1].grad, "scales", 1e-3)
    close(step.v_rot.view(-1) + step.rate_grad_rot, raw[2].grad.view(-1), "rotations", 1e-3)
    close(step.v_feat, raw[3].grad, "features", 1e-3)
