"""
The operators over the routing lists of the top-K rasterizer, as they are measured: every pixel is routed to at most ten Gaussians
(pixel_topk [H, W, 10] int32, -1 for an empty slot) with the gates n_k = w_k / (sum_j w_j + 1e-4), w_k = exp(-sigma_k).

  balance   how the pixels spread over the Gaussians: per-Gaussian counts, importance (the sum of the gates) and the balance loss
            N / (A T) * sum_g counts_g importance_g (A filled slots, T pixels with one), and its gradients for the Gaussians' geometry
  dropout   the render with gates dropped before the normalization, drawn by a counter-based generator (Philox4x32-10), and its
            gradients for the geometry and the colours

`own` false computes both with elementary torch operations; true calls igs_b200.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TOP_K = 10
EPS = 1e-4
MAX_PIXELS = 2160 * 3840
MAX_VALUES = 9 * 2048 * 2048  # pixels times channels of the largest listed render


def _case(name, op, h, w, n, c=3, grads=True, masked=False, v_importance=False, p=0.0):
    return dict(name=name, op=op, h=h, w=w, n=n, c=c, grads=grads, masked=masked, v_importance=v_importance, p=p)


def listed():
    return [
        # the smallest image that is trained, a thumbnail or one crop of a batch: launch latency
        _case("balance_64", "balance", 64, 64, 100),
        # a ragged crop with a region of interest: partial tiles, pixels outside the mask; the counts alone, as density control reads them
        _case("balance_120x88_masked", "balance", 88, 120, 300, grads=False, masked=True),
        # the loss term of a 480p step with a region of interest, and a term on the importance as well
        _case("balance_480p_masked", "balance", 480, 854, 4000, masked=True, v_importance=True),
        # the loss term of the 1080p training step
        _case("balance_1080p", "balance", 1080, 1920, 20000),
        # density control of one texture stack: counts and importance, no gradient
        _case("balance_2048_counts", "balance", 2048, 2048, 50000, grads=False),
        # the loss term of the 2160p training step
        _case("balance_2160p", "balance", 2160, 3840, 80000),
        # one small render under dropout, no gradient (Monte Carlo spread of a thumbnail)
        _case("dropout_64", "dropout", 64, 64, 100, grads=False, p=0.1),
        # a ragged one-channel crop: odd width, partial tiles
        _case("dropout_333x187_gray", "dropout", 187, 333, 700, c=1, p=0.3),
        # training steps of the 256x256, 1080p and nine-channel texture workloads under dropout
        _case("dropout_256", "dropout", 256, 256, 1000, p=0.1),
        _case("dropout_1080p", "dropout", 1080, 1920, 20000, p=0.1),
        _case("dropout_2048_tex9", "dropout", 2048, 2048, 50000, c=9, p=0.2),
        # a full render of the 2160p image under dropout
        _case("dropout_2160p_render", "dropout", 2160, 3840, 80000, grads=False, p=0.1),
    ]


def draw(rng):
    """A case of the listed ranges: images of 16 to 3840 pixels a side, 25 to 250 pixels per Gaussian, 1 to 12 channels."""
    side = lambda hi: round(math.exp(rng.uniform(math.log(16), math.log(hi))))  # noqa: E731
    h, w = side(2160), side(3840)
    op = rng.choice(["balance", "dropout"])
    n = max(1, min(80000, round(h * w / math.exp(rng.uniform(math.log(25), math.log(250))))))
    c = rng.choice([1, 2, 3, 3, 3, 4, 5, 6, 8, 9, 12])
    if op == "dropout":
        c = max(1, min(c, MAX_VALUES // (h * w)))
    return dict(op=op, h=h, w=w, n=n, c=c if op == "dropout" else 3, grads=rng.random() < 0.7,
                masked=op == "balance" and rng.random() < 0.4, v_importance=op == "balance" and rng.random() < 0.4,
                p=rng.choice([0.0, 0.05, 0.1, 0.2, 0.5, 0.9, 1.0]) if op == "dropout" else 0.0)


def work(case):
    pixels, n, c = case["h"] * case["w"], case["n"], case["c"]
    lists, geometry = 4 * TOP_K * pixels, 20 * n
    if case["op"] == "balance":
        # the lists and the geometry in; counts and importance (and the geometry's gradients) out
        total = lists + geometry + 8 * n + (pixels if case["masked"] else 0)
        if case["grads"]:
            total += geometry + (4 * n if case["v_importance"] else 0)
        # per slot: sigma 9, exp 1, the sums 4; backward: dL/dsigma 4, the five sums 12
        flops = TOP_K * pixels * (14 + (16 if case["grads"] else 0))
    else:
        colors, image = 4 * c * n, 4 * c * pixels
        total = lists + geometry + colors + image
        if case["grads"]:
            total += image + geometry + colors
        # per slot: sigma 9, exp 1, the sum 1, the blend 2c; backward: the score 2c, dL/dsigma 4, the five sums 12, the colour sums 2c
        flops = TOP_K * pixels * (11 + 2 * c + (16 + 4 * c if case["grads"] else 0))
    return {"bytes": total, "flops": flops}


# ---- inputs ----------------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    """Gaussians spread over the image on a jittered grid with IDs in random order, as a trained model's lie, and every pixel's ten
    largest weights among the 25 nearest cells; one patch of the image holds none. Empty slots come last, as the rasterizer leaves them."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    h, w, n, c = case["h"], case["w"], case["n"], case["c"]
    rand = lambda *s: torch.rand(*s, generator=gen, device=dev)  # noqa: E731
    randn = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    gx = max(1, min(n, round(math.sqrt(n * w / h))))
    gy = -(-n // gx)
    cell_w, cell_h = w / gx, h / gy
    cells = torch.arange(n, device=dev)
    xy = torch.stack([((cells % gx) + rand(n)) * cell_w, ((cells // gx) + rand(n)) * cell_h], 1)
    scale = 0.35 * math.sqrt(cell_w * cell_h) * torch.exp(0.4 * randn(n, 2))
    theta = math.pi * rand(n)
    cos, sin = torch.cos(theta), torch.sin(theta)
    i0, i1 = 1 / scale[:, 0]**2, 1 / scale[:, 1]**2
    conic = torch.stack([cos * cos * i0 + sin * sin * i1, cos * sin * (i0 - i1), sin * sin * i0 + cos * cos * i1], 1)
    id_of_cell = torch.randperm(n, generator=gen, device=dev)
    xys, conics = torch.empty_like(xy), torch.empty_like(conic)
    xys[id_of_cell], conics[id_of_cell] = xy, conic
    topk = torch.empty(h, w, TOP_K, dtype=torch.int32, device=dev)
    off = torch.arange(-2, 3, device=dev)
    px = torch.arange(w, device=dev)
    cx = (px.float() / cell_w).long().clamp_(max=gx - 1)
    rows = max(1, (1 << 21) // w)
    for r in range(0, h, rows):
        py = torch.arange(r, min(h, r + rows), device=dev)
        cy = (py.float() / cell_h).long().clamp_(max=gy - 1)
        y, x = cy[:, None, None, None] + off[:, None], cx[None, :, None, None] + off
        cell = (y * gx + x).expand(len(py), w, 5, 5).reshape(len(py), w, 25)
        there = ((y >= 0) & (x >= 0) & (x < gx)).expand(len(py), w, 5, 5).reshape(len(py), w, 25) & (cell < n)
        g = id_of_cell[cell.clamp(0, n - 1)]
        d = xys[g] - torch.stack(torch.broadcast_tensors(px.float()[None, :, None], py.float()[:, None, None]), -1)
        k = conics[g]
        sigma = 0.5 * (k[..., 0] * d[..., 0]**2 + k[..., 2] * d[..., 1]**2) + k[..., 1] * d[..., 0] * d[..., 1]
        sigma = torch.where(there & (sigma < 30), sigma, math.inf)
        best, at = torch.topk(sigma, TOP_K, dim=-1, largest=False)
        topk[r:r + len(py)] = torch.where(best < math.inf, g.gather(-1, at), -1).to(torch.int32)
    topk[h // 3:h // 3 + max(1, h // 10), w // 2:w // 2 + max(1, w // 10)] = -1
    state = dict(case=case, xys=xys, conics=conics, pixel_topk=topk, mask=None)
    if case["op"] == "balance":
        if case["masked"]:  # a region of interest with specks left out
            mask = rand(h, w) > 0.02
            mask[:h // 8], mask[:, w - w // 6:] = False, False
            state["mask"] = mask
        state["grad_loss"] = torch.full((), 0.01, device=dev)
        state["v_importance"] = randn(n) / (h * w) if case["v_importance"] else None
    else:
        state["colors"] = 0.5 + 0.2 * randn(n, c)
        state["v_output"] = torch.sign(randn(c, h, w)) / (c * h * w)  # the gradient of a mean absolute error
        state["rng_state"] = torch.tensor([seed * 2654435761 % (1 << 62), seed % 1000], dtype=torch.int64, device=dev)
    return state


# ---- the operators ---------------------------------------------------------------------------------------------------------------------

def _ops():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "image-gs_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from igs_b200 import ops

    return ops


def run(state):
    if own:
        return _run_own(state)
    return _balance(state) if state["case"]["op"] == "balance" else _dropout(state)


def _run_own(s):
    ops, case = _ops(), s["case"]
    h, w = case["h"], case["w"]
    if case["op"] == "balance":
        loss, counts, importance, totals = ops.topk_balance_forward(h, w, s["xys"], s["conics"], s["pixel_topk"], s["mask"])
        out = dict(loss=loss, counts=counts, importance=importance, totals=totals)
        if case["grads"]:
            out["v_xy"], out["v_conic"] = ops.topk_balance_backward(h, w, s["xys"], s["conics"], s["pixel_topk"], counts, totals,
                                                                    s["grad_loss"], s["v_importance"], s["mask"])
        return out
    image, used = ops.topk_dropout_forward(h, w, s["xys"], s["conics"], s["colors"], s["pixel_topk"], case["p"], s["rng_state"])
    out = dict(image=image)
    if case["grads"]:
        out["v_xy"], out["v_conic"], out["v_colors"] = ops.topk_dropout_backward(h, w, s["xys"], s["conics"], s["colors"], s["v_output"],
                                                                                 s["pixel_topk"], case["p"], used)
    return out


def _slots(s, kept=None):
    """Per slot [P, 10]: the ID (0 where empty), whether it is filled, dx, dy, the conic, the weight, the gate."""
    h, w, n = s["case"]["h"], s["case"]["w"], s["case"]["n"]
    ids = s["pixel_topk"].reshape(-1, TOP_K)
    filled = (ids >= 0) & (ids < n)
    if s["mask"] is not None:
        filled = filled & s["mask"].reshape(-1, 1)
    ids = torch.where(filled, ids, 0).long()
    p = torch.arange(h * w, device=ids.device)[:, None]
    xy, conic = s["xys"][ids], s["conics"][ids]
    dx, dy = xy[..., 0] - (p % w).float(), xy[..., 1] - (p // w).float()
    sigma = 0.5 * (conic[..., 0] * dx * dx + conic[..., 2] * dy * dy) + conic[..., 1] * dx * dy
    counted = filled & (sigma >= 0) & (sigma < math.inf)
    if kept is not None:
        counted = counted & kept
    weight = torch.where(counted, torch.exp(-sigma), 0.0)
    gate = weight / (weight.sum(1, keepdim=True) + EPS)
    return ids, filled, dx, dy, conic, gate


def _geometry_gradients(s, ids, dx, dy, conic, t):
    """v_xy [N, 2] and v_conic [N, 3] from dL/dsigma [P, 10]."""
    values = torch.stack([t * (conic[..., 0] * dx + conic[..., 1] * dy), t * (conic[..., 1] * dx + conic[..., 2] * dy),
                          0.5 * t * dx * dx, t * dx * dy, 0.5 * t * dy * dy], -1)
    sums = torch.zeros(s["case"]["n"], 5, device=t.device).index_add_(0, ids.reshape(-1), values.reshape(-1, 5))
    return sums[:, :2].contiguous(), sums[:, 2:].contiguous()


def _balance(s):
    n = s["case"]["n"]
    ids, filled, dx, dy, conic, gate = _slots(s)
    counts = torch.zeros(n, dtype=torch.int32, device=ids.device).index_add_(0, ids.reshape(-1), filled.reshape(-1).int())
    importance = torch.zeros(n, dtype=torch.float64, device=ids.device).index_add_(0, ids.reshape(-1), gate.reshape(-1).double())
    totals = torch.stack([counts.sum(), filled.any(1).sum()])
    scale = torch.where(totals[0] > 0, n / (totals[0].double() * totals[1].double()), 0.0)
    out = dict(loss=(scale * (counts * importance).sum()).float(), counts=counts, importance=importance.float(), totals=totals)
    if s["case"]["grads"]:
        alpha = s["grad_loss"] * (scale * counts).float()
        if s["v_importance"] is not None:
            alpha = alpha + s["v_importance"]
        a = alpha[ids]
        t = gate * ((gate * a).sum(1, keepdim=True) - a)
        out["v_xy"], out["v_conic"] = _geometry_gradients(s, ids, dx, dy, conic, t)
    return out


def _philox(counter, key):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011) on int64 tensors holding 32-bit words: counter of four, key of two."""
    low = 0xFFFFFFFF
    c0, c1, c2, c3 = counter
    k0, k1 = key
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the 64-bit products' bits, whatever their sign
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c0, c1, c2, c3


def _kept(s):
    """Whether each slot [P, 10] is kept: its 24-bit draw is at least rint(p 2^24)."""
    h, w = s["case"]["h"], s["case"]["w"]
    low = 0xFFFFFFFF
    seed, offset = s["rng_state"][0], s["rng_state"][1]
    pixel = torch.arange(h * w, device=s["xys"].device)
    zero = torch.zeros_like(pixel)
    key = (seed & low, (seed >> 32) & low)
    words = [_philox((pixel, zero + j, zero + (offset & low), zero + ((offset >> 32) & low)), key) for j in (0, 1)]
    w = torch.stack(words[0] + words[1], 1)
    b = w & 0xFF
    tail = torch.stack([(b[:, 0] << 16) | (b[:, 1] << 8) | b[:, 2], (b[:, 3] << 16) | (b[:, 4] << 8) | b[:, 5]], 1)
    return torch.cat([w >> 8, tail], 1) >= round(s["case"]["p"] * (1 << 24))


def _dropout(s):
    h, w, n, c = s["case"]["h"], s["case"]["w"], s["case"]["n"], s["case"]["c"]
    ids, _, dx, dy, conic, gate = _slots(s, _kept(s))
    colors = s["colors"][ids]
    out = dict(image=(gate[..., None] * colors).sum(1).t().reshape(c, h, w).contiguous())
    if s["case"]["grads"]:
        v = s["v_output"].reshape(c, -1).t().contiguous()
        score = (colors * v[:, None, :]).sum(-1)
        t = gate * ((gate * score).sum(1, keepdim=True) - score)
        out["v_xy"], out["v_conic"] = _geometry_gradients(s, ids, dx, dy, conic, t)
        out["v_colors"] = torch.zeros(n, c, device=v.device).index_add_(0, ids.reshape(-1), (gate[..., None] * v[:, None, :]).reshape(-1, c))
    return out


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    h, w, n, c = case["h"], case["w"], case["n"], case["c"]
    dev = s["xys"].device
    f8 = lambda t: t.to(torch.float64)  # noqa: E731
    lists = s["pixel_topk"].reshape(h * w, TOP_K)
    x = torch.arange(w, device=dev, dtype=torch.float64).repeat(h)
    y = torch.arange(h, device=dev, dtype=torch.float64).repeat_interleave(w)
    inside = torch.ones(h * w, dtype=torch.bool, device=dev) if s["mask"] is None else s["mask"].reshape(-1)
    keep = None
    if case["op"] == "dropout":
        keep = torch.from_numpy(_draws_64(h * w, *s["rng_state"].tolist()) >= int(np.rint(case["p"] * 2.0**24))).to(dev)
    slots, total = [], torch.zeros(h * w, dtype=torch.float64, device=dev)
    for k in range(TOP_K):
        there = inside & (lists[:, k] >= 0) & (lists[:, k] < n)
        g = lists[:, k].long().clamp(0, n - 1)
        a, b, q = f8(s["conics"][g]).unbind(1)
        u, v = f8(s["xys"][g, 0]) - x, f8(s["xys"][g, 1]) - y
        sigma = a * u * u / 2 + b * u * v + q * v * v / 2
        live = there & (sigma >= 0) & torch.isfinite(sigma)
        if keep is not None:
            live &= keep[:, k]
        e = torch.where(live, torch.exp(-sigma), torch.zeros_like(sigma))
        total += e
        slots.append((g, there, u, v, a, b, q, e))
    inverse = 1 / (total + EPS)
    add = lambda g, v: torch.zeros(n, dtype=torch.float64, device=dev).index_add_(0, g, v)  # noqa: E731
    out, scores = {}, None
    if case["op"] == "balance":
        counts = sum(add(g, f8(there)) for g, there, *_ in slots)
        importance = sum(add(sl[0], sl[7] * inverse) for sl in slots)
        filled, routed = counts.sum(), torch.stack([sl[1] for sl in slots]).any(0).sum()
        factor = n / (float(filled) * float(routed)) if filled > 0 else 0.0
        out = dict(loss=factor * (counts * importance).sum(), counts=counts.to(torch.int32), importance=importance,
                   totals=torch.stack([filled.long(), routed.long()]))
        alpha = float(s["grad_loss"]) * factor * counts + (0 if s["v_importance"] is None else f8(s["v_importance"]))
        scores = [alpha[sl[0]] for sl in slots]
    else:
        colors, v_out = f8(s["colors"]), f8(s["v_output"]).reshape(c, -1)
        image = torch.zeros(c, h * w, dtype=torch.float64, device=dev)
        for sl in slots:
            for ch in range(c):
                image[ch] += sl[7] * inverse * colors[sl[0], ch]
        out = dict(image=image.reshape(c, h, w))
        scores = [sum(colors[sl[0], ch] * v_out[ch] for ch in range(c)) for sl in slots]
    if not case["grads"]:
        return out
    mean = sum(sl[7] * inverse * sc for sl, sc in zip(slots, scores))
    v_xy, v_conic = torch.zeros(n, 2, dtype=torch.float64, device=dev), torch.zeros(n, 3, dtype=torch.float64, device=dev)
    for (g, _, u, v, a, b, q, e), sc in zip(slots, scores):
        t = -e * inverse * (sc - mean)
        v_xy[:, 0] += add(g, t * (a * u + b * v))
        v_xy[:, 1] += add(g, t * (b * u + q * v))
        v_conic[:, 0] += add(g, t * u * u / 2)
        v_conic[:, 1] += add(g, t * u * v)
        v_conic[:, 2] += add(g, t * v * v / 2)
    out["v_xy"], out["v_conic"] = v_xy, v_conic
    if case["op"] == "dropout":
        out["v_colors"] = torch.stack([sum(add(sl[0], sl[7] * inverse * v_out[ch]) for sl in slots) for ch in range(c)], 1)
    return out


def _draws_64(pixels, seed, offset):
    """The 24-bit draws [P, 10], the generator's arithmetic on numpy's unsigned 64-bit integers."""
    word = np.uint64(0xFFFFFFFF)
    eight = []
    for block in range(2):
        state = [np.arange(pixels, dtype=np.uint64), np.full(pixels, block, np.uint64), np.full(pixels, offset & 0xFFFFFFFF, np.uint64),
                 np.full(pixels, (offset >> 32) & 0xFFFFFFFF, np.uint64)]
        for r in range(10):
            key0, key1 = np.uint64((seed + r * 0x9E3779B9) & 0xFFFFFFFF), np.uint64(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
            first, second = state[0] * np.uint64(0xD2511F53), state[2] * np.uint64(0xCD9E8D57)
            state = [(second >> np.uint64(32)) ^ state[1] ^ key0, second & word, (first >> np.uint64(32)) ^ state[3] ^ key1, first & word]
        eight += state
    low = [v & np.uint64(0xFF) for v in eight]
    tails = [low[i] << np.uint64(16) | low[i + 1] << np.uint64(8) | low[i + 2] for i in (0, 3)]
    return np.stack([v >> np.uint64(8) for v in eight] + tails, 1).astype(np.int64)
