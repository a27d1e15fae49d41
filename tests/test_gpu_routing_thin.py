"""
The operators over the top-K lists for thin Gaussians and conics that are not positive definite, weights and gradients, against the float64
oracle with a bound per slot. The kernels weigh a patch (8x8 pixels) by rows where each of its conics' determinants is at least 2^-16 of a c
and slot by slot otherwise; the cases say which patches do what.

With u = 2^-24 and S the sum of the magnitudes of sigma's terms at a slot, sigma is off by at most 8 u S and a weight by a factor of
exp((11 S + 8) u) (test_gpu_routing.py), e_k = expm1 of that times w_k. Then with D = eps + sum w, E = sum e:
  gate n_k         (w_k + e_k) / (D - E) - w_k / D, and 32 roundings
  t_k = dL/dsigma  n_k (mean - s_k), mean = sum n s: each gate's error times the magnitudes of the scores it meets, once directly and once in
                   the mean
  sums of m terms  those of the terms' errors, and 64 + m roundings of the terms' magnitudes
A slot whose sigma is within 11 u S of zero could be weighed or left out; the cases have none.
"""
import numpy as np
import pytest
import torch

from common import np_
from igs_b200 import ops
from oracle import routing
from test_cpu_routing import lists_case

pytestmark = pytest.mark.gpu
U = 2.0**-24
H, W = 24, 40  # 3 x 5 patches


def thin_case(kind, n, seed):
    """float32 xys, conics and the lists; the patches that name a conic the row path does not take, as a [3, 5] bool array. kind "rows": axis
    ratios of 50 to 480 at any angle, "slots": 640 to 3000 at 30 to 60 degrees to the axes, "few": as "rows", with invalid conics (indefinite,
    negative, NaN, zero) in two patches."""
    rng = np.random.default_rng(seed)
    xys, _, lists = lists_case(H, W, n, seed)
    short = rng.uniform(1.0, 2.0, n)
    if kind == "slots":
        ratio, theta = np.geomspace(640, 3000, n), np.pi / 180 * (rng.uniform(30, 60, n) + 90 * rng.integers(0, 2, n))
    else:
        ratio, theta = np.geomspace(50, 480, n), rng.uniform(0, np.pi, n)
    i0, i1 = (ratio * short) ** -2.0, short**-2.0
    cos, sin = np.cos(theta), np.sin(theta)
    conics = np.stack([cos**2 * i0 + sin**2 * i1, cos * sin * (i0 - i1), sin**2 * i0 + cos**2 * i1], 1)
    if kind == "few":
        xys = np.concatenate([xys, rng.uniform(0, [W, H], (4, 2))])
        conics = np.concatenate([conics, [(0.1, 0.2, 0.1), (-0.1, 0.02, -0.1), (np.nan, 0.0, 0.1), (0.0, 0.0, 0.0)]])
        lists[0:8:3, 0:8:2, 6] = n + np.arange(4)
        lists[9:16:2, 17:24:3, 0] = n + np.arange(3)[None]
    xys, conics = np.float32(xys), np.float32(conics)
    lists[sign_undecided(xys, conics, lists)] = -1
    a, b, c = conics.astype(np.float64).T
    share = np.where((a > 0) & (c > 0), a * c - b * b, -1.0) / np.where(a * c > 0, a * c, 1.0)
    share = np.where(np.isfinite(share), share, -1.0)
    assert np.all(np.abs(share / 2.0**-16 - 1) > 0.05)  # no conic so near the border that its rounding decides
    named = np.where(lists >= 0, share[np.clip(lists, 0, len(share) - 1)] < 2.0**-16, False).any(-1)
    return xys, conics, lists, named.reshape(3, 8, 5, 8).any((1, 3))


def sign_undecided(xys, conics, lists):
    """The slots [H, W, 10] whose sigma lies within its rounding of zero, and is not zero exactly."""
    ids = np.where(lists >= 0, lists, 0)
    y, x = np.mgrid[:H, :W]
    (a, b, c), dx, dy = np.moveaxis(conics[ids].astype(np.float64), -1, 0), xys[ids, 0] - x[..., None], xys[ids, 1] - y[..., None]
    sigma = 0.5 * (a * dx**2 + c * dy**2) + b * dx * dy
    size = 0.5 * (abs(a) * dx**2 + abs(c) * dy**2) + abs(b * dx * dy)
    return (abs(sigma) <= 11 * U * size) & (size > 0) & (lists >= 0)


def gate_errors(g):
    size = 0.5 * (abs(g.a) * g.dx**2 + abs(g.c) * g.dy**2) + abs(g.b * g.dx * g.dy)
    e = np.expm1(np.minimum((11 * size + 8) * U, 50.0)) * g.weight
    total, off = g.weight.sum(1, keepdims=True) + routing.EPS, e.sum(1, keepdims=True)
    assert np.all(off < 0.5 * total)
    return (g.weight + e) / (total - off) - g.gate + 32 * U * g.gate


def within(actual, expected, bound, what, tight=0.02):
    """Within the bound, which is not a wide one: below `tight` of the value's magnitude for most."""
    a = np_(actual).astype(np.float64)
    assert a.shape == expected.shape and np.all(np.isfinite(a)), what
    over = abs(a - expected) - bound
    assert np.all(over <= 0), f"{what}: {over.max():.3g} over its bound"
    some = abs(expected) > 1e-3 * abs(expected).max()
    assert np.median(bound[some] / abs(expected[some])) < tight, what


def gradient_bounds(g, score, score_size):
    """t, and its error and magnitude, from the scores [P, 10] and the magnitudes of their terms."""
    n_err = gate_errors(g)
    mean = (g.gate * score).sum(1, keepdims=True)
    mean_size, mean_err = ((x * score_size).sum(1, keepdims=True) for x in (g.gate, n_err))
    err = n_err * (mean_size + mean_err + score_size) + g.gate * mean_err
    return g.gate * (mean - score), err, g.gate * (mean_size + score_size)


def check_geometry(got, g, score, score_size):
    t, err, size = gradient_bounds(g, score, score_size)
    v_xy, v_conic, err_xy, err_conic = g.geometry(t, err)
    *_, size_xy, size_conic = g.geometry(t, size)
    m = np.bincount(g.ids[g.live].ravel(), minlength=1).max(initial=0)
    within(got[0], v_xy, err_xy + (64 + m) * U * size_xy + 1e-30, "v_xy", 0.1)
    within(got[1], v_conic, err_conic + (64 + m) * U * size_conic + 1e-30, "v_conic", 0.1)


CASES = [("rows", 12), ("rows", 24), ("rows", 80), ("slots", 12), ("slots", 80), ("few", 20), ("few", 80)]


def check_paths(kind, by_slots):
    want = {"rows": np.zeros((3, 5), bool), "slots": np.ones((3, 5), bool), "few": np.zeros((3, 5), bool)}[kind]
    if kind == "few":
        want[0, 0] = want[1, 2] = True
    assert np.array_equal(by_slots, want)


def on(device, *arrays):
    return tuple(torch.from_numpy(np.ascontiguousarray(a)).to(device) for a in arrays)


@pytest.mark.parametrize("kind,n", CASES)
def test_balance_of_thin_gaussians(kind, n, device):
    xys, conics, lists, by_slots = thin_case(kind, n, 100 + n)
    check_paths(kind, by_slots)
    x, k, t = on(device, xys, conics, lists)
    loss, counts, importance, totals = ops.topk_balance_forward(H, W, x, k, t)
    o_loss, o_counts, o_importance, o_totals, g = routing.balance(H, W, xys, conics, lists)
    assert np.array_equal(np_(counts), o_counts) and tuple(totals.tolist()) == o_totals
    bound = g.add(gate_errors(g)) + 64 * U * o_importance + 1e-9
    within(importance, o_importance, bound, "importance")
    factor = len(xys) / (o_totals[0] * o_totals[1])
    assert abs(float(loss) - o_loss) <= factor * float((o_counts * bound).sum()) + 64 * U * o_loss
    v_imp = np.float32(np.random.default_rng(n).standard_normal(len(xys)))
    got = ops.topk_balance_backward(H, W, x, k, t, counts, totals, torch.tensor(0.5, device=device), on(device, v_imp)[0])
    alpha = (0.5 * factor * o_counts + v_imp)[g.ids]
    check_geometry(got, g, alpha, abs(alpha))


@pytest.mark.parametrize("kind,n", CASES)
def test_dropout_of_thin_gaussians(kind, n, device):
    xys, conics, lists, by_slots = thin_case(kind, n, 200 + n)
    check_paths(kind, by_slots)
    rng = np.random.default_rng(n)
    colors, v = np.float32(rng.standard_normal((len(xys), 3))), np.float32(rng.standard_normal((3, H, W)))
    x, k, t, f, v_out = on(device, xys, conics, lists, colors, v)
    image, used = ops.topk_dropout_forward(H, W, x, k, f, t, 0.2, torch.tensor([6, 2], device=device))
    got = ops.topk_dropout_backward(H, W, x, k, f, v_out, t, 0.2, used)
    kept = routing.keep_mask(H * W, 0.2, 6, 2)
    o_image, size, g = routing.dropout(H, W, xys, conics, colors, lists, kept)
    slot_f = np.where(g.live[..., None], colors[g.ids], 0).astype(np.float64)
    n_err = gate_errors(g)
    within(image, o_image, np.moveaxis((n_err[..., None] * abs(slot_f)).sum(1), 1, 0).reshape(size.shape) + 32 * U * size + 1e-30, "image")
    slot_v = np.moveaxis(v.reshape(3, -1), 0, 1).astype(np.float64)[:, None, :]
    check_geometry(got, g, (slot_f * slot_v).sum(-1), abs(slot_f * slot_v).sum(-1))
    v_colors, sizes, errors = (g.add(x) for x in (g.gate[..., None] * slot_v, g.gate[..., None] * abs(slot_v), n_err[..., None] * abs(slot_v)))
    m = np.bincount(g.ids[g.live].ravel(), minlength=1).max(initial=0)
    within(got[2], v_colors, errors + (64 + m) * U * sizes + 1e-30, "v_colors", 0.1)
