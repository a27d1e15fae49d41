"""
The operators over the top-K lists without a GPU: the oracle's generator against the published test vectors, its gradients against
differences in float64, its edge cases, and the refusals of the C ABI and the Python layer.
"""
import ctypes

import numpy as np
import pytest
import torch

from igs_b200 import _lib, ops
from igs_b200 import autograd as ag
from oracle import routing


def lists_case(h, w, n, seed, empty=0.2):
    rng = np.random.default_rng(seed)
    xys = rng.uniform(0, [w, h], (n, 2))
    theta, s = rng.uniform(0, np.pi, n), rng.uniform(1.0, 3.0, (n, 2))
    cos, sin, i = np.cos(theta), np.sin(theta), 1 / s**2
    conics = np.stack([cos**2 * i[:, 0] + sin**2 * i[:, 1], cos * sin * (i[:, 0] - i[:, 1]), sin**2 * i[:, 0] + cos**2 * i[:, 1]], 1)
    lists = np.full((h, w, 10), -1, np.int32)
    for p in range(h * w):
        k = min(10, n)
        lists[p // w, p % w, :k] = rng.permutation(n)[:k]
    lists[rng.random(lists.shape) < empty] = -1
    return xys, conics, lists


def test_philox_known_answers():
    # the known-answer vectors published with the generator
    for counter, key, want in (((0,) * 4, (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                               ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                               ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                                (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(routing.philox4x32(counter, key)) == want


def test_draws_are_uniform_and_distinct():
    d = routing.draws(400, 1234567, 3)
    assert d.min() >= 0 and d.max() < 1 << 24
    # 4000 uniform draws: mean within 5 standard deviations (2^24 / sqrt(12 * 4000)), per-slot means of 400 likewise
    sd = 2.0**24 / np.sqrt(12)
    assert abs(d.mean() - 2.0**23) < 5 * sd / np.sqrt(d.size)
    assert np.all(abs(d.mean(0) - 2.0**23) < 5 * sd / np.sqrt(400))
    assert not np.array_equal(d, routing.draws(400, 1234567, 4)) and not np.array_equal(d, routing.draws(400, 1234568, 3))
    assert routing.keep_mask(50, 0.0, 1, 2).all() and not routing.keep_mask(50, 1.0, 1, 2).any()


def test_balance_of_an_even_spread_is_one():
    # every pixel on its own Gaussian, on its centre: gates 1 / (1 + eps), counts 1
    h, w = 4, 6
    xys = np.stack([np.tile(np.arange(w), h), np.repeat(np.arange(h), w)], 1).astype(float)
    lists = np.full((h, w, 10), -1, np.int32)
    lists[..., 3] = np.arange(h * w).reshape(h, w)
    loss, counts, importance, totals, _ = routing.balance(h, w, xys, np.tile([1.0, 0.0, 1.0], (h * w, 1)), lists)
    assert totals == (24, 24) and (counts == 1).all()
    assert np.allclose(importance, 1 / 1.0001) and abs(loss - 1 / 1.0001) < 1e-12
    lists[:] = -1
    assert routing.balance(h, w, xys, np.ones((h * w, 3)), lists)[0] == 0.0


def differences(f, x, step=1e-6):
    out = np.empty(x.size)
    for i in range(x.size):
        up, down = x.copy(), x.copy()
        up.flat[i] += step
        down.flat[i] -= step
        out[i] = (f(up) - f(down)) / (2 * step)
    return out.reshape(x.shape)


def test_oracle_gradients_match_differences():
    # central differences of functions of order 1 in float64: truncation step^2 = 1e-12, rounding 2^-53 / step = 1e-10, both times the
    # third derivative and the value (below 100)
    h, w, n, c = 5, 7, 9, 2
    xys, conics, lists = lists_case(h, w, n, 3)
    rng = np.random.default_rng(4)
    v_imp = rng.standard_normal(n)
    mask = rng.random((h, w)) > 0.2
    loss, counts, importance, totals, g = routing.balance(h, w, xys, conics, lists, mask)
    factor = n / (totals[0] * totals[1])
    f = lambda x, k: float(((1.5 * factor * counts + v_imp) * routing.balance(h, w, x, k, lists, mask)[2]).sum())  # noqa: E731
    v_xy, v_conic, _, _ = routing.balance_grad(g, counts, totals, 1.5, v_imp)
    np.testing.assert_allclose(v_xy, differences(lambda x: f(x, conics), xys), rtol=0, atol=1e-8)
    np.testing.assert_allclose(v_conic, differences(lambda k: f(xys, k), conics), rtol=0, atol=1e-8)

    colors, v_out = rng.standard_normal((n, c)), rng.standard_normal((c, h, w))
    kept = routing.keep_mask(h * w, 0.3, 11, 5)
    render = lambda x, k, f: float((routing.dropout(h, w, x, k, f, lists, kept)[0] * v_out).sum())  # noqa: E731
    _, _, g = routing.dropout(h, w, xys, conics, colors, lists, kept)
    v_xy, v_conic, v_colors = routing.dropout_grad(g, colors, v_out)[:3]
    np.testing.assert_allclose(v_xy, differences(lambda x: render(x, conics, colors), xys), rtol=0, atol=1e-8)
    np.testing.assert_allclose(v_conic, differences(lambda k: render(xys, k, colors), conics), rtol=0, atol=1e-8)
    np.testing.assert_allclose(v_colors, differences(lambda f: render(xys, conics, f), colors), rtol=0, atol=1e-8)


def refused(status, words):
    message = _lib.load().igs_last_error().decode()
    assert status == 1 and words in message, (status, message)


def test_entry_points_refuse_invalid_arguments():
    lib = _lib.load()
    null, fake, odd = None, ctypes.c_void_p(256), ctypes.c_void_p(260)  # never dereferenced: the host checks come first
    big = 1 << 30
    fwd = lambda h=4, w=4, n=3, xys=fake, topk=fake, loss=fake, ws=fake, size=big: lib.igs_topk_balance_fwd(  # noqa: E731
        h, w, n, xys, fake, topk, null, loss, fake, fake, fake, ws, size, null)
    refused(fwd(h=-1), "negative")
    refused(fwd(n=-1), "negative")
    refused(fwd(h=1 << 15, w=1 << 15), "pixels")
    refused(fwd(h=1, w=(1 << 24) + 1), "pixels")
    refused(fwd(loss=null), "null output")
    refused(fwd(ws=null), "workspace")
    refused(fwd(size=lib.igs_topk_balance_workspace(3) - 1), "workspace")
    refused(fwd(ws=odd), "aligned")
    refused(fwd(topk=null), "null")
    refused(fwd(h=0, xys=null), "null")  # the Gaussians are read without pixels too
    refused(fwd(topk=ctypes.c_void_p(260)), "aligned")
    bwd = lambda h=4, n=3, counts=fake, ws=fake, size=big: lib.igs_topk_balance_bwd(  # noqa: E731
        h, 4, n, fake, fake, fake, null, counts, fake, null, null, 0, fake, fake, ws, size, null)
    refused(bwd(h=-1), "negative")
    refused(bwd(counts=null), "null")
    refused(bwd(ws=odd), "aligned")
    refused(bwd(size=lib.igs_topk_balance_workspace(3) - 1), "workspace")
    assert lib.igs_topk_balance_bwd(0, 4, 3, null, fake, null, null, fake, fake, null, null, 0, fake, fake, fake, big, null) == 1
    assert bwd(n=0) == 0
    drop = lambda h=4, c=3, n=3, p=0.1, topk=fake, rng=fake: lib.igs_topk_dropout_fwd(  # noqa: E731
        h, 4, c, n, fake, fake, fake, topk, p, rng, fake, fake, null)
    refused(drop(h=-1), "negative")
    refused(drop(c=0), "channels")
    refused(drop(c=13), "channels")
    for p in (-0.1, 1.1, float("nan")):
        refused(drop(p=p), "[0, 1]")
    refused(drop(rng=null), "rng")
    refused(drop(topk=null), "null")
    refused(drop(topk=odd), "aligned")
    back = lambda c=3, n=3, p=0.1, v=fake, ws=fake, size=big: lib.igs_topk_dropout_bwd(  # noqa: E731
        4, 4, c, n, fake, fake, fake, fake, fake, p, fake, v, fake, fake, ws, size, null)
    refused(back(c=13), "channels")
    refused(back(p=2.0), "[0, 1]")
    refused(back(v=null), "null output")
    refused(back(ws=null), "workspace")
    refused(back(size=lib.igs_topk_dropout_workspace(3, 3) - 1), "workspace")
    assert lib.igs_topk_dropout_bwd(0, 4, 3, 3, null, fake, fake, fake, fake, 0.1, fake, fake, fake, fake, fake, big, null) == 1
    assert back(n=0) == 0


def test_python_layer_refuses_cpu_tensors():
    xys, conics, topk = torch.zeros(3, 2), torch.zeros(3, 3), torch.zeros(4, 4, 10, dtype=torch.int32)
    rng = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.topk_balance_forward(4, 4, xys, conics, topk)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ag.topk_balance(xys, conics, topk, 4, 4)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.topk_dropout_forward(4, 4, xys, conics, torch.zeros(3, 3), topk, 0.1, rng)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ag.rasterize_topk_dropout(xys, conics, torch.zeros(3, 3), topk, 4, 4, 0.1, rng)
