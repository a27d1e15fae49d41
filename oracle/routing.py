"""
ORACLE (test infrastructure): the operators over the top-K lists in float64 on the CPU, from their definitions: per-Gaussian counts,
importance and the balance loss with its gradient, and the render under gate dropout with its gradients, with the published Philox4x32-10
generator on Python integers. Beside each gradient stands the sum of the magnitudes of its terms, for error bounds.
"""
import numpy as np

EPS = 1e-4


def philox4x32(counter, key):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): four 32-bit words from a counter of four and a key of two (Python integers)."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def draws(pixels, seed, offset):
    """[P, 10] 24-bit draws: slot k < 8 the upper 24 bits of word k, slots 8 and 9 the low bytes of words 0-2 and 3-5."""
    seed, offset = seed & (1 << 64) - 1, offset & (1 << 64) - 1
    key = (seed & 0xFFFFFFFF, seed >> 32)
    out = np.empty((pixels, 10), np.int64)
    for p in range(pixels):
        w = [v for j in (0, 1) for v in philox4x32((p, j, offset & 0xFFFFFFFF, offset >> 32), key)]
        out[p, :8] = [v >> 8 for v in w]
        b = [v & 255 for v in w]
        out[p, 8:] = (b[0] << 16 | b[1] << 8 | b[2], b[3] << 16 | b[4] << 8 | b[5])
    return out


def keep_mask(pixels, p, seed, offset):
    """[P, 10] bool: whether each slot is kept."""
    return draws(pixels, seed, offset) >= int(np.rint(p * 2.0**24))


class Gates:
    """The slots [P, 10] of the lists: ids (0 where empty), filled, dx, dy, conic a, b, c, weight and gate; kept [P, 10] and mask [P] leave
    slots out. magnitude is the largest sum of sigma's terms' magnitudes over the slots whose weight float32 can hold (sigma < 104): the
    size that sigma's rounding has."""

    def __init__(self, h, w, xys, conics, pixel_topk, mask=None, kept=None):
        xys, conics = np.asarray(xys, np.float64).reshape(-1, 2), np.asarray(conics, np.float64).reshape(-1, 3)
        self.n = n = len(xys)
        lists = np.asarray(pixel_topk).reshape(h * w, 10).astype(np.int64)
        self.filled = (lists >= 0) & (lists < n)
        if mask is not None:
            self.filled = self.filled & (np.asarray(mask).reshape(-1, 1) != 0)
        live = self.filled if kept is None else self.filled & kept
        self.ids = np.where(live, lists, 0)
        p = np.arange(h * w)
        if n == 0:
            xys, conics = np.zeros((1, 2)), np.zeros((1, 3))
        with np.errstate(all="ignore"):
            self.dx, self.dy = xys[self.ids, 0] - (p % max(w, 1))[:, None], xys[self.ids, 1] - (p // max(w, 1))[:, None]
            self.a, self.b, self.c = (conics[self.ids, j] for j in range(3))
            square = 0.5 * (self.a * self.dx**2 + self.c * self.dy**2)
            sigma = square + self.b * self.dx * self.dy
            live = live & (sigma >= 0) & np.isfinite(sigma)
            self.weight = np.where(live, np.exp(-np.where(live, sigma, 0)), 0)
            self.magnitude = float(np.max(np.where(live & (sigma < 104), square + np.abs(self.b * self.dx * self.dy), 0), initial=0.0))
        for name in ("dx", "dy", "a", "b", "c"):  # a Gaussian without a weight contributes nothing, whatever its parameters hold
            setattr(self, name, np.where(live, getattr(self, name), 0))
        self.live = live
        self.gate = self.weight / (self.weight.sum(1, keepdims=True) + EPS)

    def add(self, values):
        """[N, ...] sums of per-slot values [P, 10, ...]."""
        out = np.zeros((self.n,) + values.shape[2:])
        np.add.at(out, self.ids[self.live], values[self.live])
        return out

    def geometry(self, t, t_abs):
        """v_xy, v_conic of dL/dsigma t, and the same sums over the terms' magnitudes with t_abs in place of |t|."""
        dx, dy, a, b, c = self.dx, self.dy, self.a, self.b, self.c
        v = np.stack([t * (a * dx + b * dy), t * (b * dx + c * dy), t * dx * dx / 2, t * dx * dy, t * dy * dy / 2], -1)
        m = np.stack([t_abs * (abs(a * dx) + abs(b * dy)), t_abs * (abs(b * dx) + abs(c * dy)), t_abs * dx * dx / 2,
                      t_abs * abs(dx * dy), t_abs * dy * dy / 2], -1)
        v, m = self.add(v), self.add(m)
        return v[:, :2], v[:, 2:], m[:, :2], m[:, 2:]


def balance(h, w, xys, conics, pixel_topk, mask=None):
    """(loss, counts [N], importance [N], totals [2], the Gates)."""
    g = Gates(h, w, xys, conics, pixel_topk, mask)
    counts = np.zeros(g.n, np.int64)
    np.add.at(counts, g.ids[g.filled], 1)
    importance = g.add(g.gate)
    a, t = int(counts.sum()), int(g.filled.any(1).sum())
    loss = g.n / (a * t) * float((counts * importance).sum()) if a else 0.0
    return loss, counts, importance, (a, t), g


def balance_grad(g, counts, totals, v_loss=0.0, v_importance=None):
    """(v_xy, v_conic, their magnitude sums) of v_loss * loss + v_importance . importance, the counts constant."""
    alpha = v_loss * g.n / (totals[0] * totals[1]) * counts if totals[0] else np.zeros(g.n)
    if v_importance is not None:
        alpha = alpha + np.asarray(v_importance, np.float64)
    alpha = alpha[g.ids] if g.n else np.zeros(g.ids.shape)
    mean = (g.gate * alpha).sum(1, keepdims=True)
    return g.geometry(g.gate * (mean - alpha), g.gate * ((g.gate * abs(alpha)).sum(1, keepdims=True) + abs(alpha)))


def dropout(h, w, xys, conics, colors, pixel_topk, kept):
    """(image [C, H, W], sum of the terms' magnitudes [C, H, W], the Gates); kept [P, 10] from keep_mask."""
    g = Gates(h, w, xys, conics, pixel_topk, None, kept)
    colors = np.asarray(colors, np.float64)
    f = np.where(g.live[..., None], colors[g.ids], 0) if g.n else np.zeros(g.ids.shape + (colors.shape[1],))
    image, size = (np.moveaxis((g.gate[..., None] * x).sum(1), 1, 0).reshape(-1, h, w) for x in (f, abs(f)))
    return image, size, g


def dropout_grad(g, colors, v_output):
    """(v_xy, v_conic, v_colors, their magnitude sums)."""
    colors = np.asarray(colors, np.float64)
    v = np.moveaxis(np.asarray(v_output, np.float64).reshape(colors.shape[1], -1), 0, 1)
    f = np.where(g.live[..., None], colors[g.ids], 0)
    score, size = (f * v[:, None, :]).sum(-1), abs(f * v[:, None, :]).sum(-1)
    mean, mean_size = (g.gate * score).sum(1, keepdims=True), (g.gate * size).sum(1, keepdims=True)
    v_xy, v_conic, m_xy, m_conic = g.geometry(g.gate * (mean - score), g.gate * (mean_size + size))
    terms = g.gate[..., None] * v[:, None, :]
    return v_xy, v_conic, g.add(terms), m_xy, m_conic, g.add(abs(terms))
