"""
The operators over the top-K lists on the GPU against the float64 oracle: counts, importance, the balance loss and its gradient; the render
under gate dropout and its gradients.

Tolerances, with u = 2^-24 (half a float32 step, relative) and M the largest sum of sigma's terms' magnitudes in the case:
  weight  sigma's terms round at most 6 times each and are added twice: 8 u M; __expf is off by at most 2 + 1.173 sigma steps of 2 u, and
          sigma <= M: E = (11 M + 8) u relative
  gate    w / (sum w + eps): 2 E, at most 32 roundings of sums, reciprocal and product: G = 2 E + 32 u
  sums    of m values in any order: m u of the sum of their magnitudes
  gradient  dL/dsigma is a gate times a difference of two values that each carry a gate's error, all of it relative to the terms'
          magnitudes; the geometric factors and the scores round at most 64 times: 2 G + (64 + m) u of the sum of the magnitudes
"""
import numpy as np
import pytest
import torch

from common import make_case, np_, ours_stages, to_dev
from igs_b200 import _lib, ops
from igs_b200 import autograd as ag
from oracle import routing
from test_cpu_routing import lists_case

pytestmark = pytest.mark.gpu
U = 2.0**-24


def gate_tolerance(g):
    return 2 * (11 * g.magnitude + 8) * U + 32 * U


def check_sums(actual, expected, sizes, rel, what, floor=0.0):
    """|actual - expected| <= rel * sizes (+ floor) elementwise; infinite or missing values are failures."""
    a = np_(actual).astype(np.float64)
    assert a.shape == expected.shape, f"{what}: {a.shape} != {expected.shape}"
    excess = np.abs(a - expected) - rel * sizes - floor
    assert np.all(np.isfinite(a)) and np.all(excess <= 0), f"{what}: {np.nanmax(excess):.3g} over its bound"


def check_balance(got, h, w, xys, conics, lists, mask=None):
    loss, counts, importance, totals = got
    o_loss, o_counts, o_importance, o_totals, g = routing.balance(h, w, xys, conics, lists, mask)
    assert np.array_equal(np_(counts), o_counts) and tuple(totals.tolist()) == o_totals
    rel = gate_tolerance(g) + 64 * U
    check_sums(importance, o_importance, o_importance, rel, "importance", floor=1e-9)
    assert abs(float(loss) - o_loss) <= rel * o_loss + 1e-9
    return g, o_counts, o_totals


def check_balance_grad(got, g, counts, totals, v_loss, v_importance):
    v_xy, v_conic, m_xy, m_conic = routing.balance_grad(g, counts, totals, v_loss, v_importance)
    rel = 2 * gate_tolerance(g) + (64 + counts.max(initial=0)) * U
    check_sums(got[0], v_xy, m_xy, rel, "v_xy", floor=1e-30)
    check_sums(got[1], v_conic, m_conic, rel, "v_conic", floor=1e-30)


def check_dropout(h, w, xys, conics, colors, lists, p, state, v_out, device):
    d = lambda a, dt=np.float32: torch.from_numpy(np.ascontiguousarray(a, dt)).to(device)  # noqa: E731
    args = (d(xys), d(conics), d(colors))
    rng = torch.tensor(state, dtype=torch.int64, device=device)
    image, used = ops.topk_dropout_forward(h, w, *args, d(lists, np.int32), p, rng)
    grads = ops.topk_dropout_backward(h, w, *args, d(v_out), d(lists, np.int32), p, used)
    assert used.tolist() == list(state)
    kept = routing.keep_mask(h * w, p, *state)
    o_image, size, g = routing.dropout(h, w, np.float32(xys), np.float32(conics), np.float32(colors), lists, kept)
    gate = gate_tolerance(g)
    check_sums(image, o_image, size, gate + 32 * U, "image", floor=1e-30)
    v_xy, v_conic, v_colors, m_xy, m_conic, m_colors = routing.dropout_grad(g, np.float32(colors), np.float32(v_out))
    m = np.bincount(g.ids[g.live].ravel(), minlength=1).max(initial=0)
    rel = 2 * gate + (64 + m) * U
    for a, b, size, what in zip(grads, (v_xy, v_conic, v_colors), (m_xy, m_conic, m_colors), ("v_xy", "v_conic", "v_colors")):
        check_sums(a, b, size, rel, what, floor=1e-30)
    return image, grads


def to_gpu(device, xys, conics, lists):
    return (torch.from_numpy(np.float32(xys)).to(device), torch.from_numpy(np.float32(conics)).to(device),
            torch.from_numpy(np.ascontiguousarray(lists, np.int32)).to(device))


# one pixel, single rows and columns, partial tiles and patches; few Gaussians and, with 300 in random lists, hundreds in one patch
SIZES = [(1, 1, 1), (1, 17, 5), (23, 1, 12), (4, 8, 9), (16, 16, 40), (33, 47, 90), (19, 26, 300)]


@pytest.mark.parametrize("h,w,n", SIZES)
def test_balance_matches_oracle(h, w, n, device):
    xys, conics, lists = lists_case(h, w, n, 100 * h + w)
    xys, conics = np.float32(xys), np.float32(conics)
    x, k, t = to_gpu(device, xys, conics, lists)
    got = ops.topk_balance_forward(h, w, x, k, t)
    g, counts, totals = check_balance(got, h, w, xys, conics, lists)
    v_loss = torch.tensor(0.7, device=device)
    v_imp = np.float32(np.random.default_rng(1).standard_normal(n))
    for vl, vi in ((v_loss, None), (None, torch.from_numpy(v_imp).to(device)), (v_loss, torch.from_numpy(v_imp).to(device)), (None, None)):
        grads = ops.topk_balance_backward(h, w, x, k, t, got[1], got[3], vl, vi)
        check_balance_grad(grads, g, counts, totals, 0.0 if vl is None else np.float64(np.float32(0.7)), None if vi is None else v_imp)


@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8])
def test_balance_mask(dtype, device):
    h, w, n = 21, 35, 60
    xys, conics, lists = lists_case(h, w, n, 5)
    xys, conics = np.float32(xys), np.float32(conics)
    x, k, t = to_gpu(device, xys, conics, lists)
    rng = np.random.default_rng(2)
    for mask in (rng.random((h, w)) > 0.4, np.zeros((h, w), bool), np.ones((h, w), bool)):
        mask = mask.copy()
        mask[7:12] = False  # whole rows left out
        m = torch.from_numpy(mask).to(device)
        m = m if dtype == torch.bool else m.to(torch.uint8) * 255
        got = ops.topk_balance_forward(h, w, x, k, t, m)
        g, counts, totals = check_balance(got, h, w, xys, conics, lists, mask)
        grads = ops.topk_balance_backward(h, w, x, k, t, got[1], got[3], torch.tensor(1.0, device=device), None, m)
        check_balance_grad(grads, g, counts, totals, 1.0, None)


def hostile_lists(lists, n, seed):
    """IDs out of range, the lowest and highest int32, and a Gaussian in two slots of one pixel."""
    rng = np.random.default_rng(seed)
    lists = lists.copy()
    at = rng.random(lists.shape)
    lists[at < 0.04] = n
    lists[(at > 0.04) & (at < 0.08)] = np.iinfo(np.int32).max
    lists[(at > 0.08) & (at < 0.12)] = np.iinfo(np.int32).min
    lists[::3, :, 7] = lists[::3, :, 2]
    return lists


def test_lists_with_ids_out_of_range_and_repeats(device):
    h, w, n = 18, 29, 50
    xys, conics, lists = lists_case(h, w, n, 8)
    xys, conics, lists = np.float32(xys), np.float32(conics), hostile_lists(lists, n, 9)
    x, k, t = to_gpu(device, xys, conics, lists)
    got = ops.topk_balance_forward(h, w, x, k, t)
    g, counts, totals = check_balance(got, h, w, xys, conics, lists)
    grads = ops.topk_balance_backward(h, w, x, k, t, got[1], got[3], torch.tensor(1.0, device=device))
    check_balance_grad(grads, g, counts, totals, 1.0, None)
    rng = np.random.default_rng(3)
    check_dropout(h, w, xys, conics, rng.standard_normal((n, 3)), lists, 0.25, (77, 0), rng.standard_normal((3, h, w)), device)


def test_broken_gaussians_weigh_nothing(device):
    """NaN, infinite and negative-sigma parameters: the slot counts, its weight and its gradients are zero, and no other Gaussian feels it."""
    h, w, n = 20, 24, 30
    xys, conics, lists = lists_case(h, w, n, 12)
    xys, conics = np.float32(xys), np.float32(conics)
    xys[3], xys[4, 0], conics[5, 1], conics[6] = np.nan, np.inf, np.nan, np.inf
    conics[7] = -conics[7]
    colors = np.float32(np.random.default_rng(1).standard_normal((n, 3)))
    x, k, t = to_gpu(device, xys, conics, lists)
    got = ops.topk_balance_forward(h, w, x, k, t)
    g, counts, totals = check_balance(got, h, w, xys, conics, lists)
    grads = ops.topk_balance_backward(h, w, x, k, t, got[1], got[3], torch.tensor(1.0, device=device))
    check_balance_grad(grads, g, counts, totals, 1.0, None)
    for i in (3, 4, 5, 6, 7):
        assert int(got[1][i]) > 0 and float(got[2][i]) == 0 and not grads[0][i].any() and not grads[1][i].any()
    check_dropout(h, w, xys, conics, colors, lists, 0.25, (5, 6), np.random.default_rng(2).standard_normal((3, h, w)), device)


def test_empty_inputs(device):
    f, i32 = dict(device=device), dict(device=device, dtype=torch.int32)
    rng = torch.tensor([1, 2], device=device)
    for h, w, n in ((0, 5, 4), (6, 0, 4), (5, 6, 0), (0, 0, 0)):
        x, k, t = torch.rand(n, 2, **f), torch.rand(n, 3, **f), torch.zeros(h, w, 10, **i32)
        loss, counts, importance, totals = ops.topk_balance_forward(h, w, x, k, t)
        assert float(loss) == 0 and not counts.any() and not importance.any() and totals.tolist() == [0, 0]
        grads = ops.topk_balance_backward(h, w, x, k, t, counts, totals, torch.ones((), **f))
        image, used = ops.topk_dropout_forward(h, w, x, k, torch.rand(n, 3, **f), t, 0.5, rng)
        grads += ops.topk_dropout_backward(h, w, x, k, torch.rand(n, 3, **f), torch.rand(3, h, w, **f), t, 0.5, used)
        assert used.tolist() == [1, 2] and image.shape == (3, h, w) and not image.any()
        assert all(not v.any() for v in grads)
    x, k, t = torch.rand(7, 2, **f), torch.rand(7, 3, **f), torch.full((9, 11, 10), -1, **i32)  # lists without a slot
    loss, counts, importance, totals = ops.topk_balance_forward(9, 11, x, k, t)
    assert float(loss) == 0 and not counts.any() and totals.tolist() == [0, 0]
    assert all(not v.any() for v in ops.topk_balance_backward(9, 11, x, k, t, counts, totals, torch.ones((), **f)))


@pytest.mark.parametrize("h,w,n", SIZES)
@pytest.mark.parametrize("p", [0.0, 0.3, 1.0])
def test_dropout_matches_oracle(h, w, n, p, device):
    xys, conics, lists = lists_case(h, w, n, 7 * h + w)
    rng = np.random.default_rng(h + w)
    image, grads = check_dropout(h, w, xys, conics, rng.standard_normal((n, 3)), lists, p, (1 << 40 | 12345, 9), rng.standard_normal((3, h, w)),
                                 device)
    if p == 1.0:
        assert not image.any() and all(not v.any() for v in grads)


@pytest.mark.parametrize("c", range(1, 13))
def test_dropout_channels(c, device):
    h, w, n = 13, 22, 35
    xys, conics, lists = lists_case(h, w, n, 40 + c)
    rng = np.random.default_rng(c)
    check_dropout(h, w, xys, conics, rng.standard_normal((n, c)), lists, 0.2, (3, 1 << 33), rng.standard_normal((c, h, w)), device)


@pytest.mark.parametrize("state", [(0, 0), (-1, -1), (-(1 << 63), (1 << 63) - 1), (0xFFFFFFFF, 0x100000000)])
def test_dropout_mask_of_any_state(state, device):
    """The mask itself: with ten Gaussians of weight 1 and one-hot colours, a pixel's channels show which of its slots were kept."""
    h, w = 6, 11
    xys = np.zeros((10, 2))
    conics = np.full((10, 3), 0.0)  # sigma 0: every weight is 1
    lists = np.broadcast_to(np.arange(10, dtype=np.int32), (h, w, 10))
    kept = routing.keep_mask(h * w, 0.5, *state)
    x, k, t = to_gpu(device, xys, conics, lists)
    rng = torch.tensor(state, dtype=torch.int64, device=device)
    image, _ = ops.topk_dropout_forward(h, w, x, k, torch.eye(10, device=device), t, 0.5, rng)
    assert np.array_equal(np_(image).reshape(10, -1).T > 0, kept)


def test_dropout_of_nothing_is_the_render(device):
    """p = 0 on the rasterizer's own lists: its render and the gradients of its backward pass."""
    h, w, n = 88, 120, 300
    _, inp = make_case(h, w, n, seed=11)
    d = to_dev(inp, device)
    s = ours_stages(d, h, w)
    rng = torch.tensor([5, 5], device=device)
    image, used = ops.topk_dropout_forward(h, w, s["xys"], s["conics"], d["features"], s["pixel_topk"], 0.0, rng)
    # both renders are within their gates' error of the same value
    g = routing.Gates(h, w, np_(s["xys"]), np_(s["conics"]), np_(s["pixel_topk"]))
    size = np.moveaxis((g.gate[..., None] * abs(np_(inp["features"])[g.ids])).sum(1), 1, 0).reshape(3, h, w)
    check_sums(image, np_(s["image"]).astype(np.float64), size, 2 * (gate_tolerance(g) + 32 * U), "image", floor=1e-30)
    grads = ops.topk_dropout_backward(h, w, s["xys"], s["conics"], d["features"], s["v_output"], s["pixel_topk"], 0.0, used)
    *_, m_xy, m_conic, m_colors = routing.dropout_grad(g, np_(inp["features"]), np_(s["v_output"]))
    m = np.bincount(g.ids[g.live].ravel()).max()
    for a, b, size in zip(grads, (s["v_xy"], s["v_conic"], s["v_colors"]), (m_xy, m_conic, m_colors)):
        check_sums(a, np_(b).astype(np.float64), size, 2 * (2 * gate_tolerance(g) + (64 + m) * U), "gradient", floor=1e-30)


def test_dropped_colors_are_not_read_into_the_sums(device):
    """Infinite and NaN colours of Gaussians that only dropped or empty slots name leave no trace."""
    h, w, n = 8, 9, 12
    xys, conics, lists = lists_case(h, w, n, 21)
    colors = np.random.default_rng(1).standard_normal((n, 3))
    kept = routing.keep_mask(h * w, 0.5, 4, 4).reshape(h, w, 10)
    lists = np.where(kept, lists % 10, np.random.default_rng(2).integers(10, 12, lists.shape))  # 10 and 11 in dropped slots only
    lists[0, 0] = -1
    colors[10], colors[11] = np.inf, np.nan
    image, grads = check_dropout(h, w, xys, conics, colors, lists, 0.5, (4, 4), np.random.default_rng(3).standard_normal((3, h, w)), device)
    assert not grads[2][10:].any() and not image[:, 0, 0].any()


def test_balance_repeats_bit_for_bit(device):
    h, w, n = 64, 96, 50
    xys, conics, lists = lists_case(h, w, n, 6)
    x, k, t = to_gpu(device, xys, conics, lists)
    first = ops.topk_balance_forward(h, w, x, k, t)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.topk_balance_forward(h, w, x, k, t)))


def test_autograd_balance(device):
    h, w, n = 30, 41, 70
    xys, conics, lists = lists_case(h, w, n, 14)
    x, k, t = to_gpu(device, xys, conics, lists)
    mask = torch.rand(h, w, device=device) > 0.3
    weight = torch.randn(n, device=device)
    x.requires_grad_(True), k.requires_grad_(True)
    loss, counts, importance, totals = ag.topk_balance(x, k, t, h, w, mask)
    assert not counts.requires_grad and not totals.requires_grad
    got = torch.autograd.grad(0.5 * loss + (weight * importance).sum(), (x, k))
    g, o_counts, o_totals = check_balance((loss.detach(), counts, importance.detach(), totals), h, w, np_(x), np_(k), lists, np_(mask))
    check_balance_grad(got, g, o_counts, o_totals, 0.5, np_(weight))
    only = torch.autograd.grad((weight * ag.topk_balance(x, k, t, h, w, mask)[2]).sum(), (x, k))
    check_balance_grad(only, g, o_counts, o_totals, 0.0, np_(weight))
    # layouts that are not contiguous give the same
    wide = torch.zeros(n, 5, device=device)
    wide[:, :2], wide[:, 2:] = x.detach(), k.detach()
    other = ag.topk_balance(wide[:, :2], wide[:, 2:], t.permute(2, 0, 1).contiguous().permute(1, 2, 0), h, w, mask.t().contiguous().t())
    assert all(torch.equal(a, b) for a, b in zip(other, (loss.detach(), counts, importance.detach(), totals)))
    with pytest.raises(RuntimeError):  # once differentiable
        gx, = torch.autograd.grad(ag.topk_balance(x, k, t, h, w)[0], x, create_graph=True)
        gx.sum().backward()


def test_autograd_dropout_keeps_its_mask_when_the_state_moves(device):
    h, w, n = 30, 41, 70
    xys, conics, lists = lists_case(h, w, n, 15)
    x, k, t = to_gpu(device, xys, conics, lists)
    f = torch.randn(n, 4, device=device)
    rng = torch.tensor([10, 20], device=device)
    v = torch.randn(h, w, 4, device=device)
    want_image, used = ops.topk_dropout_forward(h, w, x, k, f, t, 0.4, rng)
    want = ops.topk_dropout_backward(h, w, x, k, f, v.permute(2, 0, 1).contiguous(), t, 0.4, used)
    leaves = [a.clone().requires_grad_(True) for a in (x, k, f)]
    image = ag.rasterize_topk_dropout(*leaves, t, h, w, 0.4, rng)
    rng[1] += 1
    assert torch.equal(image.detach().permute(2, 0, 1), want_image)
    (image * v).sum().backward()
    for a, b in zip(leaves, want):
        torch.testing.assert_close(a.grad, b, rtol=1e-4, atol=1e-5 * float(b.abs().max()))  # the order of the atomics alone
    assert not torch.equal(ops.topk_dropout_forward(h, w, x, k, f, t, 0.4, rng)[0], want_image)


def test_captured_step_draws_a_new_mask_each_replay(device):
    """Both operators forward and backward in one captured graph whose last node moves the offset: each replay equals the eager call at
    that offset, with new inputs written in place."""
    h, w, n = 40, 56, 80
    xys, conics, lists = lists_case(h, w, n, 16)
    x, k, t = to_gpu(device, xys, conics, lists)
    f, v = torch.randn(n, 3, device=device), torch.randn(3, h, w, device=device)
    rng, one = torch.tensor([3, 100], device=device), torch.ones((), device=device)

    def step(state):
        image, used = ops.topk_dropout_forward(h, w, x, k, f, t, 0.3, state)
        grads = ops.topk_dropout_backward(h, w, x, k, f, v, t, 0.3, used)
        loss, counts, importance, totals = ops.topk_balance_forward(h, w, x, k, t)
        return (image, loss, counts, importance, totals), grads + ops.topk_balance_backward(h, w, x, k, t, counts, totals, one)

    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        step(rng)
    torch.cuda.current_stream(device).wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        exact, sums = step(rng)
        rng[1:].add_(1)
    rng.copy_(torch.tensor([3, 100]))
    images = []
    for i in range(3):
        graph.replay()
        want_exact, want_sums = step(torch.tensor([3, 100 + i], device=device))
        assert all(torch.equal(a, b) for a, b in zip(exact, want_exact))
        for a, b in zip(sums, want_sums):
            torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5 * float(b.abs().max()))
        images.append(exact[0].clone())
        x += 0.25  # new inputs in place
    assert rng.tolist() == [3, 103]
    assert not torch.equal(images[0], images[1])


def test_python_layer_refuses(device):
    h, w, n = 4, 6, 5
    x, k = torch.rand(n, 2, device=device), torch.rand(n, 3, device=device)
    t = torch.zeros(h, w, 10, dtype=torch.int32, device=device)
    f, rng, v = torch.rand(n, 3, device=device), torch.zeros(2, dtype=torch.int64, device=device), torch.rand(3, h, w, device=device)
    counts, totals = torch.zeros(n, dtype=torch.int32, device=device), torch.zeros(2, dtype=torch.int64, device=device)
    fwd, bwd = ops.topk_balance_forward, ops.topk_balance_backward
    drop, back = ops.topk_dropout_forward, ops.topk_dropout_backward
    for call, words in ((lambda: fwd(h, w, x.double(), k, t), "xys"), (lambda: fwd(h, w, x, k[:4], t), "conics"),
                        (lambda: fwd(h, w, x, k, t.long()), "pixel_topk"), (lambda: fwd(h, w + 1, x, k, t), "pixel_topk"),
                        (lambda: fwd(h, w, x, k, t[..., :9]), "contiguous"), (lambda: fwd(h, w, x[:, :1], k, t), "contiguous"),
                        (lambda: fwd(h, w, x, k, t, torch.zeros(h, w, device=device)), "pixel_mask"),
                        (lambda: fwd(h, w, x, k, t, torch.zeros(h, dtype=torch.bool, device=device)), "pixel_mask"),
                        (lambda: bwd(h, w, x, k, t, counts.long(), totals), "counts"), (lambda: bwd(h, w, x, k, t, counts[:3], totals), "counts"),
                        (lambda: bwd(h, w, x, k, t, counts, totals, torch.ones(2, device=device)), "grad_loss"),
                        (lambda: bwd(h, w, x, k, t, counts, totals, torch.ones((), dtype=torch.float64, device=device)), "grad_loss"),
                        (lambda: bwd(h, w, x, k, t, counts, totals, None, torch.ones(3, device=device)), "grad_importance"),
                        (lambda: drop(h, w, x, k, f[:4], t, 0.1, rng), "colors"), (lambda: drop(h, w, x, k, f.half(), t, 0.1, rng), "colors"),
                        (lambda: drop(h, w, x, k, torch.rand(n, 13, device=device), t, 0.1, rng), "channels"),
                        (lambda: drop(h, w, x, k, f, t, 0.1, rng.int()), "rng_state"), (lambda: drop(h, w, x, k, f, t, 0.1, rng[:1]), "rng_state"),
                        (lambda: drop(h, w, x, k, f, t, 0.1, rng.cpu()), "CUDA tensor|must be on"),
                        (lambda: back(h, w, x, k, f, v[:2], t, 0.1, rng), "v_output")):
        with pytest.raises(RuntimeError, match=words):
            call()
    for p in (-0.5, 1.5, float("nan")):
        with pytest.raises(ValueError, match=r"\[0, 1\]"):
            drop(h, w, x, k, f, t, p, rng)
    flat = torch.zeros(h * w * 10 + 1, dtype=torch.int32, device=device)
    with pytest.raises(_lib.IgsError, match="aligned"):  # lists that start on an odd 4-byte word
        fwd(h, w, x, k, flat[1:].view(h, w, 10))


def test_operators_on_a_side_stream(device):
    h, w, n = 50, 70, 100
    xys, conics, lists = lists_case(h, w, n, 31)
    x, k, t = to_gpu(device, xys, conics, lists)
    f, rng = torch.rand(n, 3, device=device), torch.tensor([1, 1], device=device)
    want = ops.topk_balance_forward(h, w, x, k, t), ops.topk_dropout_forward(h, w, x, k, f, t, 0.2, rng)
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        got = ops.topk_balance_forward(h, w, x, k, t), ops.topk_dropout_forward(h, w, x, k, f, t, 0.2, rng)
    stream.synchronize()
    assert all(torch.equal(a, b) for s, u in zip(want, got) for a, b in zip(s, u))


def test_values_that_are_not_finite_stay_where_they_belong(device):
    """A NaN or infinite image gradient, colour or importance gradient reaches the Gaussians of the pixels concerned, and no other: not
    those of neighbouring pixels, and nothing at a pixel without a slot."""
    h, w, n = 16, 40, 60
    xys, conics, lists = lists_case(h, w, n, 51, empty=0.5)
    lists[2, 5] = -1
    x, k, t = to_gpu(device, xys, conics, lists)
    rng = torch.tensor([1, 1], device=device)
    f, v = torch.randn(n, 3, device=device), torch.randn(3, h, w, device=device)
    used = ops.topk_dropout_forward(h, w, x, k, f, t, 0.0, rng)[1]
    g = routing.Gates(h, w, np_(x), np_(k), lists)
    holds = lambda i, j: set(g.ids.reshape(h, w, 10)[i, j][g.weight.reshape(h, w, 10)[i, j] > 1e-37])  # noqa: E731
    clean = ops.topk_dropout_backward(h, w, x, k, f, v, t, 0.0, used)

    def compare(got, want, touched):
        others = np.setdiff1d(np.arange(n), list(touched))
        assert len(others) > 10
        for a, b in zip(got, want):
            a, b = np_(a)[others], np_(b)[others]
            assert np.all(np.isfinite(a)) and np.all(abs(a - b) <= 1e-4 * abs(b) + 1e-5 * abs(b).max())  # paths that sum in other orders

    bad = v.clone()
    bad[1, 2, 5], bad[0, 9, 33] = float("nan"), float("inf")  # (2, 5) has no slot
    got = ops.topk_dropout_backward(h, w, x, k, f, bad, t, 0.0, used)
    compare(got, clean, holds(9, 33))
    assert all(not torch.isfinite(got[2][i]).all() for i in holds(9, 33))

    alpha = torch.randn(n, device=device)
    alpha[7] = float("nan")
    _, counts, _, totals = ops.topk_balance_forward(h, w, x, k, t)
    want = ops.topk_balance_backward(h, w, x, k, t, counts, totals, None, torch.where(torch.isnan(alpha), 0.0, alpha))
    got = ops.topk_balance_backward(h, w, x, k, t, counts, totals, None, alpha)
    together = set().union(*(holds(i, j) for i in range(h) for j in range(w) if 7 in holds(i, j)))
    apart = np.setdiff1d(np.arange(n), list(together))
    if len(apart) > 10:
        compare(got, want, together)
    one = torch.full((h, w, 10), -1, dtype=torch.int32, device=device)  # each Gaussian alone in its pixel: only the broken one is touched
    one.view(-1, 10)[:n, 4] = torch.arange(n, device=device, dtype=torch.int32)
    _, counts, _, totals = ops.topk_balance_forward(h, w, x, k, one)
    got = ops.topk_balance_backward(h, w, x, k, one, counts, totals, None, alpha)
    want = ops.topk_balance_backward(h, w, x, k, one, counts, totals, None, torch.where(torch.isnan(alpha), 0.0, alpha))
    compare(got, want, {7})
    f2 = f.clone()
    f2[7] = float("inf")
    compare(ops.topk_dropout_backward(h, w, x, k, f2, v, one, 0.0, used), ops.topk_dropout_backward(h, w, x, k, f, v, one, 0.0, used), {7})


@pytest.mark.parametrize("h,w,n,log_scale", [(120, 168, 900, 1.1), (90, 75, 2500, 0.2)])
def test_rasterizer_lists(h, w, n, log_scale, device):
    """The rasterizer's own lists, with more Gaussians than the last CTA finishes, sparse and dense enough that patches overflow their rows."""
    _, inp = make_case(h, w, n, log_scale_mean=log_scale, seed=31)
    d = to_dev(inp, device)
    s = ours_stages(d, h, w)
    xys, conics, lists = np_(s["xys"]), np_(s["conics"]), np_(s["pixel_topk"])
    x, k, t = s["xys"], s["conics"], s["pixel_topk"]
    got = ops.topk_balance_forward(h, w, x, k, t)
    g, counts, totals = check_balance(got, h, w, xys, conics, lists)
    grads = ops.topk_balance_backward(h, w, x, k, t, got[1], got[3], torch.tensor(1.0, device=device))
    check_balance_grad(grads, g, counts, totals, 1.0, None)
    rng = np.random.default_rng(7)
    check_dropout(h, w, xys, conics, rng.standard_normal((n, 3)), lists, 0.15, (1, 2), rng.standard_normal((3, h, w)), device)


def test_thin_gaussians(device):
    """Axes from 1:1 to 3000:1 at all angles, and conics that are not positive definite: where rounding decides sigma's sign, the weight is 0
    or the bound is as wide as sigma's rounding."""
    h, w, n = 24, 40, 80
    rng = np.random.default_rng(61)
    xys, _, lists = lists_case(h, w, n, 62)
    ratio, theta = np.geomspace(1, 3000, n), rng.uniform(0, np.pi, n)
    i0, i1 = np.full(n, 1 / 6.0**2), (ratio / 6.0) ** 2 / np.maximum(1, ratio / 300) ** 2
    cos, sin = np.cos(theta), np.sin(theta)
    conics = np.float32(np.stack([cos**2 * i0 + sin**2 * i1, cos * sin * (i0 - i1), sin**2 * i0 + cos**2 * i1], 1))
    conics[5], conics[9], conics[13] = (0.1, 0.2, 0.1), (-0.1, 0.0, 0.1), (0.0, 0.0, 0.0)
    xys = np.float32(xys)
    x, k, t = to_gpu(device, xys, conics, lists)
    got = ops.topk_balance_forward(h, w, x, k, t)
    _, counts, importance, totals, g = routing.balance(h, w, xys, conics, lists)
    assert np.array_equal(np_(got[1]), counts) and tuple(got[3].tolist()) == totals
    # sigma may be off by 8 u of its terms' magnitude, a weight by a factor exp of that (a weight whose sigma's sign that decides: by 1 at
    # most): per slot, with the oracle's magnitudes
    magnitude = 0.5 * (abs(g.a) * g.dx**2 + abs(g.c) * g.dy**2) + abs(g.b * g.dx * g.dy)
    sigma = 0.5 * (g.a * g.dx**2 + g.c * g.dy**2) + g.b * g.dx * g.dy
    off = 11 * U * magnitude + 8 * U
    decided = sigma > off
    wide = np.where(decided, np.expm1(np.minimum(off, 50.0)) * g.weight, 1.0) * g.filled
    bound = wide.sum(1, keepdims=True) / (np.maximum(g.weight.sum(1, keepdims=True) - wide.sum(1, keepdims=True), 0) + 1e-4) * g.gate + \
        wide / (np.maximum(g.weight.sum(1, keepdims=True) - wide.sum(1, keepdims=True), 0) + 1e-4) + 64 * U * g.gate
    lists_flat = lists.reshape(h * w, 10)
    sums = np.zeros(n)
    np.add.at(sums, np.where(g.filled, lists_flat, 0)[g.filled], np.minimum(bound, 1.0)[g.filled])
    check_sums(got[2], importance, np.ones(n), 0.0, "importance", floor=sums + 1e-6)
    assert torch.isfinite(got[2]).all()
    grads = ops.topk_balance_backward(h, w, x, k, t, got[1], got[3], torch.tensor(1.0, device=device))
    assert all(torch.isfinite(v).all() for v in grads)


def test_unaligned_parameters(device):
    """xys, conics and colours that start on any 4-byte word."""
    h, w, n = 21, 26, 60
    xys, conics, lists = lists_case(h, w, n, 71)
    x, k, t = to_gpu(device, xys, conics, lists)
    f, v, rng = torch.randn(n, 5, device=device), torch.randn(5, h, w, device=device), torch.tensor([4, 4], device=device)

    def shifted(a):
        flat = torch.empty(a.numel() + 1, device=device)
        flat[1:] = a.reshape(-1)
        return flat[1:].view(a.shape)

    want = ops.topk_balance_forward(h, w, x, k, t) + ops.topk_dropout_forward(h, w, x, k, f, t, 0.2, rng)
    got = ops.topk_balance_forward(h, w, shifted(x), shifted(k), t) + ops.topk_dropout_forward(h, w, shifted(x), shifted(k), shifted(f), t, 0.2, rng)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    grads = ops.topk_dropout_backward(h, w, shifted(x), shifted(k), shifted(f), shifted(v), t, 0.2, rng)
    for a, b in zip(grads, ops.topk_dropout_backward(h, w, x, k, f, v, t, 0.2, rng)):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5 * float(b.abs().max()))


@pytest.mark.parametrize("c", [3, 12])
def test_captured_autograd_step(c, device):
    """Both operators through autograd, forward and backward, captured in one graph (after a warm-up on the capturing stream), with eager
    steps of the same leaves before and after: the replayed gradients equal the eager ones at the same offset."""
    h, w, n = 48, 64, 600
    xys, conics, lists = lists_case(h, w, n, 17)
    x, k, t = to_gpu(device, xys, conics, lists)
    leaves = [a.requires_grad_(True) for a in (x, k, torch.randn(n, c, device=device))]
    target, rng = torch.rand(h, w, c, device=device), torch.tensor([8, 40], device=device)

    def step():
        image = ag.rasterize_topk_dropout(*leaves, t, h, w, 0.2, rng)
        loss = (image - target).square().mean() + 0.1 * ag.topk_balance(leaves[0], leaves[1], t, h, w)[0]
        return loss, torch.autograd.grad(loss, leaves)

    # The eager graph is gone before the capture: a live one ties the leaves to its stream, which ends the capture, whatever the operators
    eager = float(step()[0])
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream(device).wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        loss, grads = step()
        rng[1:].add_(1)
    rng.copy_(torch.tensor([8, 40]))
    for _ in range(2):
        offset = rng.tolist()
        graph.replay()
        rng_after = rng.tolist()
        rng.copy_(torch.tensor(offset))
        want_loss, want = step()
        rng.copy_(torch.tensor(rng_after))
        assert float(loss) == float(want_loss) and rng_after[1] == offset[1] + 1
        for a, b in zip(grads, want):
            torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-5 * float(b.abs().max()))  # the order of the atomics alone
    assert eager != float(loss)


def test_two_streams_at_once(device):
    """Calls of different sizes running at once on two streams share nothing."""
    cases = []
    for h, w, n, seed in ((300, 260, 350, 81), (200, 333, 1500, 82)):
        rng = np.random.default_rng(seed)
        xys = np.float32(rng.uniform(0, [w, h], (n, 2)))
        conics = np.tile(np.float32([0.05, 0.01, 0.04]), (n, 1))
        near = ((np.arange(h)[:, None] // 8) * (w // 8 + 1) + np.arange(w)[None] // 8) % n
        lists = (near[..., None] + np.arange(10)) % n
        cases.append((h, w) + to_gpu(device, xys, conics, lists) + (torch.randn(n, 3, device=device), torch.randn(3, h, w, device=device)))
    state = torch.tensor([3, 3], device=device)

    def run(h, w, x, k, t, f, v):
        got = ops.topk_balance_forward(h, w, x, k, t)
        image, used = ops.topk_dropout_forward(h, w, x, k, f, t, 0.3, state)
        return got + (image,), ops.topk_dropout_backward(h, w, x, k, f, v, t, 0.3, used)

    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in cases]
    results = [[], []]
    for _ in range(20):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                results[i].append(run(*c))
    torch.cuda.synchronize()
    for (exact, sums), got in zip(want, results):
        for e, g in got:
            assert all(torch.equal(a, b) for a, b in zip(exact, e))
            for a, b in zip(sums, g):
                torch.testing.assert_close(b, a, rtol=1e-3, atol=1e-5 * float(a.abs().max()))
