"""
The operators over the top-K lists where one pixel or Gaussian could disturb another of its patch (8x8 pixels): against the float64 oracle
with the tolerances of test_gpu_routing.py.
"""
import numpy as np
import pytest
import torch

from igs_b200 import _lib, ops
from oracle import routing
from test_gpu_routing import U, check_balance, check_balance_grad, check_dropout, check_sums, gate_tolerance, to_gpu

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


def neighbour_lists(cells_y, cells_x, cell):
    """Gaussians one per cell of `cell` pixels a side; every pixel names its own cell's and the eight around it."""
    y, x = np.mgrid[:cells_y * cell, :cells_x * cell] // cell
    lists = np.full((cells_y * cell, cells_x * cell, 10), -1, np.int32)
    for k, (dy, dx) in enumerate((a, b) for a in (-1, 0, 1) for b in (-1, 0, 1)):
        inside = (0 <= y + dy) & (y + dy < cells_y) & (0 <= x + dx) & (x + dx < cells_x)
        lists[..., k] = np.where(inside, (y + dy) * cells_x + x + dx, -1)
    return lists


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_value_that_is_not_finite_reaches_those_that_share_a_pixel_alone(value, device):
    """Lists of nine Gaussians: one that is not finite leaves the gradients of all that share no pixel with it, of its own patches too."""
    cell, cells_y, cells_x, bad = 4, 4, 12, 13  # cell (1, 1): named by rows and columns 0 to 11, half of the patches beside the first
    lists = neighbour_lists(cells_y, cells_x, cell)
    h, w, n = lists.shape[0], lists.shape[1], cells_y * cells_x
    rng = np.random.default_rng(17)
    at = np.arange(n)
    xys = np.float32(np.stack([at % cells_x, at // cells_x], 1) * cell + rng.uniform(0, cell, (n, 2)))
    conics = np.tile(np.float32([0.11, 0.02, 0.09]), (n, 1))
    holds = (lists == bad).any(-1)
    together = set(lists[holds].ravel()) - {-1}
    apart = np.setdiff1d(at, list(together))
    patch = lambda m: m.reshape(h // 8, 8, w // 8, 8).any((1, 3))  # noqa: E731
    same_patch = [i for i in apart if (patch((lists == i).any(-1)) & patch(holds)).any()]
    assert len(apart) > 20 and len(same_patch) > 3

    def compare(got, want, sizes, rel):
        for a, b, size in zip(got, want, sizes):
            a = a.cpu().numpy().astype(np.float64)
            assert not np.isfinite(a[bad]).all()
            assert np.all(abs(a[apart] - b[apart]) <= rel * size[apart] + 1e-30)

    x, k, t = to_gpu(device, xys, conics, lists)
    _, counts, _, totals = ops.topk_balance_forward(h, w, x, k, t)
    alpha = np.float32(rng.standard_normal(n))
    _, o_counts, _, o_totals, g = routing.balance(h, w, xys, conics, lists)
    v_xy, v_conic, *sizes = routing.balance_grad(g, o_counts, o_totals, 0.0, alpha)
    alpha[bad] = value
    got = ops.topk_balance_backward(h, w, x, k, t, counts, totals, None, torch.from_numpy(alpha).to(device))
    rel = 2 * gate_tolerance(g) + (64 + o_counts.max()) * U
    compare(got, (v_xy, v_conic), sizes, rel)

    colors, v = np.float32(rng.standard_normal((n, 3))), np.float32(rng.standard_normal((3, h, w)))
    v_xy, v_conic, v_colors, *sizes = routing.dropout_grad(g, colors, v)
    colors[bad, 1] = value
    state = torch.tensor([2, 2], device=device)
    f, v_out = torch.from_numpy(colors).to(device), torch.from_numpy(v).to(device)
    image = ops.topk_dropout_forward(h, w, x, k, f, t, 0.0, state)[0]
    assert torch.isfinite(image[0]).all() and torch.equal(~torch.isfinite(image[1]).cpu(), torch.from_numpy(holds))
    got = ops.topk_dropout_backward(h, w, x, k, f, v_out, t, 0.0, state)
    compare(got[:2], (v_xy, v_conic), sizes[:2], rel)
    a = got[2].cpu().numpy().astype(np.float64)  # the colours' gradients hold no colour
    assert np.all(abs(a - v_colors) <= rel * sizes[2] + 1e-30)


ROWS = 28  # of a group


@pytest.mark.parametrize("ids,repeats", [(15, 0), (16, 0), (17, 0), (ROWS - 1, 0), (ROWS, 0), (ROWS + 1, 0), (2 * ROWS, 0), (2 * ROWS + 1, 0),
                                         (ROWS - 1, 1), (ROWS, 1), (ROWS + 1, 1), (ROWS, 9), (2 * ROWS, 1)])
def test_rows_at_the_border_of_a_group(ids, repeats, device):
    """One patch whose lists name just as many Gaussians as half a warp or a group of rows takes, one fewer and one more; and with the last of
    a group's IDs in 1 + repeats slots of one pixel, each a row of its own, so that the same ID lies on both sides of the border."""
    h = w = 8
    rng = np.random.default_rng(1000 * ids + repeats)
    lists = np.full((h * w, 10), -1, np.int32)
    for p in range(h * w):
        lists[p, :7] = (p * 5 + np.arange(7)) % ids  # every ID in some pixels
    if repeats:
        lists[11] = -1
        lists[11, rng.permutation(10)[:1 + repeats]] = min(ROWS, ids) - 1
    lists = rng.permuted(lists, axis=1).reshape(h, w, 10)
    assert len(np.unique(lists[lists >= 0])) == ids
    n = ids + 3  # some that nothing names
    xys, conics = np.float32(rng.uniform(0, 8, (n, 2))), np.tile(np.float32([0.2, 0.05, 0.3]), (n, 1))
    x, k, t = to_gpu(device, xys, conics, lists)
    got = ops.topk_balance_forward(h, w, x, k, t)
    g, counts, totals = check_balance(got, h, w, xys, conics, lists)
    v_imp = np.float32(rng.standard_normal(n))
    grads = ops.topk_balance_backward(h, w, x, k, t, got[1], got[3], torch.tensor(1.0, device=device), torch.from_numpy(v_imp).to(device))
    check_balance_grad(grads, g, counts, totals, 1.0, v_imp)
    for p, c in ((0.0, 3), (0.2, 1), (0.2, 9)):
        check_dropout(h, w, xys, conics, rng.standard_normal((n, c)), lists, p, (ids, repeats), rng.standard_normal((c, h, w)), device)


@pytest.mark.slow
def test_largest_image(device):
    """The tallest image of the operators' limits, 214 million pixels, with slots in its first and last rows alone: lists of 8.6 GB, and twelve
    channels, whose planes pass 2^31 values."""
    h, w, c, half = 65535 * 16, 204, 12, 20
    top, bottom = 2, 5
    rng = np.random.default_rng(77)
    n = 2 * half
    xys = rng.uniform(0, [w, 5], (n, 2))
    xys[half:, 1] += h - bottom
    xys, conics = np.float32(xys), np.tile(np.float32([0.02, 0.003, 0.1]), (n, 1))
    lists = torch.full((h, w, 10), -1, dtype=torch.int32, device=device)
    ends = [rng.permuted(np.broadcast_to(np.arange(half), (rows, w, half)), axis=2)[..., :10] for rows in (top, bottom)]
    ends[1] = ends[1] + half
    lists[:top], lists[-bottom:] = torch.from_numpy(ends[0]).to(device), torch.from_numpy(ends[1]).to(device)
    x, k = torch.from_numpy(xys).to(device), torch.from_numpy(conics).to(device)

    def at_the_ends(what):  # what(rows, xys of these rows, lists, first pixel) at both ends; the halves of the Gaussians are apart
        shifted = xys.astype(np.float64)
        shifted[:, 1] -= h - bottom
        return what(top, xys, ends[0], 0), what(bottom, shifted, ends[1], (h - bottom) * w)

    loss, counts, importance, totals = ops.topk_balance_forward(h, w, x, k, lists)
    both = at_the_ends(lambda rows, at, ids, _: routing.balance(rows, w, at, conics, ids))
    o_counts, o_importance = (sum(b[i] for b in both) for i in (1, 2))
    o_totals = tuple(sum(b[3][i] for b in both) for i in (0, 1))
    assert np.array_equal(counts.cpu().numpy(), o_counts) and tuple(totals.tolist()) == o_totals == ((top + bottom) * w * 10, (top + bottom) * w)
    gate = max(gate_tolerance(b[4]) for b in both)
    check_sums(importance, o_importance, o_importance, gate + 64 * U, "importance", floor=1e-8)  # 2^-34 in each of some 52 patches
    factor = n / (o_totals[0] * o_totals[1])
    o_loss = factor * float((o_counts * o_importance).sum())
    assert abs(float(loss) - o_loss) <= (gate + 64 * U) * o_loss + factor * float(o_counts.sum()) * 1e-8
    grads = ops.topk_balance_backward(h, w, x, k, lists, counts, totals, torch.tensor(1.0, device=device))
    alpha = factor * o_counts  # as an importance gradient, the counts and totals of one end being its own
    parts = [routing.balance_grad(b[4], b[1], b[3], 0.0, alpha) for b in both]
    v_xy, v_conic, m_xy, m_conic = (sum(p[i] for p in parts) for i in range(4))
    rel = 2 * gate + (64 + o_counts.max()) * U
    check_sums(grads[0], v_xy, m_xy, rel, "v_xy", floor=1e-30)
    check_sums(grads[1], v_conic, m_conic, rel, "v_conic", floor=1e-30)

    p, seed, offset = 0.3, 5, 6
    colors = np.float32(rng.standard_normal((n, c)))
    f = torch.from_numpy(colors).to(device)
    image, used = ops.topk_dropout_forward(h, w, x, k, f, lists, p, torch.tensor([seed, offset], device=device))
    assert not image[:, top:-bottom].any()
    v = [np.float32(rng.standard_normal((c, rows, w))) for rows in (top, bottom)]
    image_ends = image[:, :top].clone(), image[:, -bottom:].clone()
    v_output = image.fill_(1.0)  # (10 GB: in place)
    v_output[:, :top], v_output[:, -bottom:] = torch.from_numpy(v[0]).to(device), torch.from_numpy(v[1]).to(device)
    grads = ops.topk_dropout_backward(h, w, x, k, f, v_output, lists, p, used)

    def render(rows, at, ids, first):
        words = [[routing.philox4x32((i, j, offset, 0), (seed, 0)) for j in (0, 1)] for i in range(first, first + rows * w)]
        words = np.array(words, np.int64).reshape(-1, 8)
        low = words & 255
        tail = np.stack([low[:, i] << 16 | low[:, i + 1] << 8 | low[:, i + 2] for i in (0, 3)], 1)
        kept = np.concatenate([words >> 8, tail], 1) >= int(np.rint(p * 2.0**24))
        return routing.dropout(rows, w, at, conics, colors, ids, kept)

    both = at_the_ends(render)
    gate = max(gate_tolerance(g) for *_, g in both)
    for got, (want, size, _) in zip(image_ends, both):
        check_sums(got, want, size, gate + 32 * U, "image", floor=1e-30)
    parts = [routing.dropout_grad(g, colors, v_end) for (*_, g), v_end in zip(both, v)]
    sums = [sum(part[i] for part in parts) for i in range(6)]
    for got, want, size, what in zip(grads, sums[:3], sums[3:], ("v_xy", "v_conic", "v_colors")):
        check_sums(got, want, size, 2 * gate + (64 + o_counts.max()) * U, what, floor=1e-30)
