"""
The training step with the routing regularizers: RasterStep with gate dropout and with the balance term against the same operators called
one by one through autograd, replayed as a CUDA graph, and behind the straight-through quantizer.
"""
import pytest
import torch

from common import make_case, to_dev
from igs_b200 import autograd as ag
from igs_b200 import ops, pipeline, workloads

pytestmark = pytest.mark.gpu


def lists_of(means, scales, rotations, features, h, w):
    tb = ops.tile_grid(h, w)
    n = means.shape[0]
    xys, radii, conics, hits = ops.project_gaussians_2d_scale_rot_forward(n, means, scales, rotations, h, w, tb)
    cum, total = ops.cumulative_intersects(hits)
    ids, bins = ops.sort_intersects_by_tile(n, int(total.item()), xys, radii, cum, tb)
    return ops.nd_rasterize_forward_topk_norm(tb, (16, 16, 1), (w, h, 1), ids, bins, xys, conics, features)[1]


def autograd_step(d, h, w, p=None, state=None, factor=0.0, mask=None, l1_ratio=1.0):
    """(loss, balance loss, image, gradients of means, scales, rotations, features)."""
    leaves = [d[k].clone().requires_grad_(True) for k in ("means", "scales", "rotations", "features")]
    topk = lists_of(*(t.detach() for t in leaves), h, w)
    xys, _, conics, _ = ag.project_gaussians_2d_scale_rot(*leaves[:3], h, w, ops.tile_grid(h, w))
    rng = torch.tensor(state or (0, 0), dtype=torch.int64, device=xys.device)
    image = ag.rasterize_topk_dropout(xys, conics, leaves[3], topk, h, w, p or 0.0, rng).permute(2, 0, 1)
    loss = l1_ratio * ag.l1_loss(image, d["target"])
    balance = ag.topk_balance(xys, conics, topk, h, w, mask)[0]
    (loss + factor * balance).backward()
    return loss.detach(), balance.detach(), image.detach(), [t.grad for t in leaves]


def close(a, b, what, rtol=1e-4):
    # Sums of the same terms by atomics in other orders: a few dozen roundings of 2^-24 of the terms' magnitudes, which the projection's
    # backward pass combines with factors of order 1. The terms of an L1 gradient cancel, by a factor of 250 at most where the value is
    # above 1e-3 of the largest (the floor): 64 * 2^-24 * 250 = 1e-3 for gradients.
    err = (a - b).abs() / torch.clamp(b.abs(), min=1e-3 * float(b.abs().max()) + 1e-30)
    assert float(err.max()) <= rtol, f"{what}: {float(err.max()):.3g}"


@pytest.mark.parametrize("p,factor,masked", [(0.2, None, False), (None, 0.05, False), (0.3, 0.05, True), (0.0, 0.02, False)])
def test_step_matches_autograd(p, factor, masked, device):
    h, w, n = 100, 152, 500
    _, inp = make_case(h, w, n, seed=21)
    d = to_dev(inp, device)
    mask = torch.rand(h, w, device=device) > 0.3 if masked else None
    rng = torch.tensor([12, 7], dtype=torch.int64, device=device)
    step = pipeline.RasterStep(d["means"], d["scales"], d["rotations"], d["features"], d["target"], l1_ratio=0.8,
                               balance=None if factor is None else dict(factor=factor, mask=mask),
                               gate_dropout=None if p is None else dict(p=p, rng_state=rng))
    step.launch()
    loss, balance, image, grads = autograd_step(d, h, w, p, (12, 7), factor or 0.0, mask, 0.8)
    if p is not None:
        assert torch.equal(step.image, image) and rng.tolist() == [12, 8]
    close(step.image, image, "image", 1e-5 / 0.05)  # the render's own bound where it is the rasterizer's
    assert abs(float(step.loss) - float(loss)) <= 2e-6 * float(loss)
    if factor is not None:
        assert float(step.balance_loss) == float(balance) and int(step.totals[0]) == int(step.counts.sum())
    for a, b, name in zip((step.v_mean2d, step.v_scale, step.v_rot, step.v_colors), grads, ("means", "scales", "rotations", "features")):
        close(a, b, name, 1e-3)


def test_replayed_step_draws_a_new_mask(device):
    h, w, n = 96, 120, 400
    _, inp = make_case(h, w, n, seed=22)
    d = to_dev(inp, device)
    rng = torch.tensor([5, 0], dtype=torch.int64, device=device)
    step = pipeline.RasterStep(d["means"], d["scales"], d["rotations"], d["features"], d["target"], balance=dict(factor=0.01),
                               gate_dropout=dict(p=0.25, rng_state=rng))
    step.replay()  # captures (after a launch outside the capture) and replays
    images = []
    for _ in range(3):
        offset = int(rng[1])
        step.replay()
        assert int(rng[1]) == offset + 1
        assert torch.equal(step.image, autograd_step(d, h, w, 0.25, (5, offset))[2])
        images.append(step.image.clone())
    assert not torch.equal(images[0], images[1])


def test_step_behind_the_quantizer(device):
    h, w, n = 64, 80, 200
    wl, inp = make_case(h, w, n, seed=23)
    d = to_dev(inp, device)
    quant = workloads.quant_settings(wl, device)
    rng = torch.tensor([9, 9], dtype=torch.int64, device=device)
    step = pipeline.RasterStep(d["means"], d["scales"], d["rotations"], d["features"], d["target"], quant=quant, balance=dict(factor=0.03),
                               gate_dropout=dict(p=0.1, rng_state=rng))
    step.launch()
    q = dict(zip(("means", "scales", "rotations", "features"),
                 ag.quantize_ste(d["means"], d["scales"], d["rotations"], d["features"], quant["pos_steps"], quant["scale_step"],
                                 quant["rot_step"], quant["feat_steps"])))
    loss, balance, image, grads = autograd_step(dict(q, target=d["target"]), h, w, 0.1, (9, 9), 0.03)
    assert torch.equal(step.image, image) and float(step.balance_loss) == float(balance)
    for a, b, name in zip((step.v_mean2d, step.v_scale, step.v_rot, step.v_colors), grads, ("means", "scales", "rotations", "features")):
        close(a, b, name, 1e-3)


def test_step_refuses(device):
    _, inp = make_case(32, 32, 20, seed=1)
    d = to_dev(inp, device)
    args = (d["means"], d["scales"], d["rotations"], d["features"], d["target"])
    rng = torch.zeros(2, dtype=torch.int64, device=device)
    with pytest.raises(ValueError, match=r"\[0, 1\]"):
        pipeline.RasterStep(*args, gate_dropout=dict(p=1.5, rng_state=rng))
    with pytest.raises(ValueError, match="rng_state"):
        pipeline.RasterStep(*args, gate_dropout=dict(p=0.5, rng_state=rng.int()))
    with pytest.raises(ValueError, match="mask"):
        pipeline.RasterStep(*args, balance=dict(factor=0.1, mask=torch.ones(4, 4, dtype=torch.bool, device=device)))
