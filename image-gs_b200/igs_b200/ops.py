"""
Tensor-level operators over the igs_b200 C ABI, with the names, argument order, return values and input checks of the reference's
pybind functions (gsplat/gsplat/cuda/csrc/ext.cpp:4-32, bindings.h). Outputs are allocated with PyTorch's caching allocator on the input's
device and every launch goes to the current CUDA stream, so the operators can be captured in CUDA graphs (the *_capacity paths never read
device memory back to the host).
"""
import functools
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check, ptr, raw_stream_of, stream_of

TILE = 16
TOP_K = 10
MAX_CHANNELS = 12
EPS = 1e-4


def _check_input(t: torch.Tensor, name: str, dtype=None):
    # CHECK_INPUT of the reference (bindings.h:9-14): CUDA and contiguous
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")


def _lib_call(name, *args):
    check(getattr(_lib.load(), name)(*args), name)


def tile_grid(img_height: int, img_width: int) -> Tuple[int, int, int]:
    return ((img_width + TILE - 1) // TILE, (img_height + TILE - 1) // TILE, 1)


# ---- projection ----------------------------------------------------------------------------------------------------------------------

def project_gaussians_2d_scale_rot_forward(num_points, means2d, scales2d, rotation, img_height, img_width, tile_bounds):
    """-> xys [N,2], radii [N] int32, conics [N,3], num_tiles_hit [N] int32 (bindings.cu:791-837)."""
    for t, n in ((means2d, "means2d"), (scales2d, "scales2d"), (rotation, "rotation")):
        _check_input(t, n, torch.float32)
    dev = means2d.device
    xys = torch.empty(num_points, 2, device=dev, dtype=torch.float32)
    radii = torch.empty(num_points, device=dev, dtype=torch.int32)
    conics = torch.empty(num_points, 3, device=dev, dtype=torch.float32)
    num_tiles_hit = torch.empty(num_points, device=dev, dtype=torch.int32)
    with torch.cuda.device(dev):
        _lib_call("igs_project_fwd", int(num_points), ptr(means2d), ptr(scales2d), ptr(rotation), int(img_height), int(img_width),
                  int(tile_bounds[0]), int(tile_bounds[1]), ptr(xys), ptr(radii), ptr(conics), ptr(num_tiles_hit), stream_of(dev))
    return xys, radii, conics, num_tiles_hit


def project_gaussians_2d_scale_rot_backward(num_points, means2d, scales2d, rotation, img_height, img_width, radii, conics, v_xy,
                                            v_conic):
    """-> v_cov2d [N,3], v_mean2d [N,2], v_scale [N,2], v_rot [N,1] (bindings.cu:845-891)."""
    scales2d, rotation, radii, conics = scales2d.contiguous(), rotation.contiguous(), radii.contiguous(), conics.contiguous()
    v_xy, v_conic = v_xy.contiguous(), v_conic.contiguous()
    for t, n in ((scales2d, "scales2d"), (rotation, "rotation"), (conics, "conics"), (v_xy, "v_xy"), (v_conic, "v_conic")):
        _check_input(t, n, torch.float32)
    _check_input(radii, "radii", torch.int32)
    dev = scales2d.device
    v_cov2d = torch.empty(num_points, 3, device=dev, dtype=torch.float32)
    v_mean2d = torch.empty(num_points, 2, device=dev, dtype=torch.float32)
    v_scale = torch.empty(num_points, 2, device=dev, dtype=torch.float32)
    v_rot = torch.empty(num_points, 1, device=dev, dtype=torch.float32)
    with torch.cuda.device(dev):
        _lib_call("igs_project_bwd", int(num_points), ptr(scales2d), ptr(rotation), int(img_height), int(img_width), ptr(radii),
                  ptr(conics), ptr(v_xy), ptr(v_conic), ptr(v_cov2d), ptr(v_mean2d), ptr(v_scale), ptr(v_rot), stream_of(dev))
    return v_cov2d, v_mean2d, v_scale, v_rot


# ---- binning -------------------------------------------------------------------------------------------------------------------------

def cumulative_intersects(num_tiles_hit: torch.Tensor):
    """Inclusive int32 prefix sum and its last element as a 1-element device tensor (no host synchronization)."""
    _check_input(num_tiles_hit, "num_tiles_hit", torch.int32)
    n = num_tiles_hit.numel()
    dev = num_tiles_hit.device
    cum = torch.empty(n, device=dev, dtype=torch.int32)
    total = torch.empty(1, device=dev, dtype=torch.int32)
    ws_bytes = _lib.load().igs_cumsum_workspace(n)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    with torch.cuda.device(dev):
        _lib_call("igs_cumsum", int(n), ptr(num_tiles_hit), ptr(cum), ptr(total), ptr(ws), ws_bytes, stream_of(dev))
    return cum, total


def sort_intersects_by_tile(num_points, capacity, xys, radii, cum_tiles_hit, tile_bounds):
    """-> gaussian_ids_sorted [capacity] int32, tile_bins [T,2] int32 (bindings.cu:106-167)."""
    _check_input(xys, "xys", torch.float32)
    _check_input(radii, "radii", torch.int32)
    _check_input(cum_tiles_hit, "cum_tiles_hit", torch.int32)
    dev = xys.device
    tiles_x, tiles_y = int(tile_bounds[0]), int(tile_bounds[1])
    num_tiles = tiles_x * tiles_y
    capacity = int(capacity)
    if capacity <= 0:
        return (torch.zeros(0, device=dev, dtype=torch.int32), torch.zeros(num_tiles, 2, device=dev, dtype=torch.int32))
    ids = torch.empty(capacity, device=dev, dtype=torch.int32)
    tile_bins = torch.empty(num_tiles, 2, device=dev, dtype=torch.int32)
    ws_bytes = _lib.load().igs_sort_workspace(capacity, tiles_x, tiles_y)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    with torch.cuda.device(dev):
        _lib_call("igs_sort_intersects", int(num_points), capacity, ptr(xys), ptr(radii), ptr(cum_tiles_hit), tiles_x, tiles_y, ptr(ids),
                  ptr(tile_bins), ptr(ws), ws_bytes, stream_of(dev))
    return ids, tile_bins


# ---- rasterization -------------------------------------------------------------------------------------------------------------------

def _check_raster_geometry(tile_bounds, block, img_size):
    if tuple(block)[:2] != (TILE, TILE):
        raise ValueError(f"block must be ({TILE}, {TILE}, 1) (the tile size is fixed at compile time), got {tuple(block)}")
    w, h = int(img_size[0]), int(img_size[1])
    if (int(tile_bounds[0]), int(tile_bounds[1])) != tile_grid(h, w)[:2]:
        raise ValueError(f"tile_bounds {tuple(tile_bounds)} do not cover a {w}x{h} image with {TILE}x{TILE} tiles")
    return h, w


def nd_rasterize_forward_topk_norm(tile_bounds, block, img_size, gaussian_ids_sorted, tile_bins, xys, conics, colors):
    """-> out_img [C,H,W], pixel_topk [H,W,10] int32 (bindings.cu:380-437)."""
    h, w = _check_raster_geometry(tile_bounds, block, img_size)
    _check_input(gaussian_ids_sorted, "gaussian_ids_sorted", torch.int32)
    _check_input(tile_bins, "tile_bins", torch.int32)
    for t, n in ((xys, "xys"), (conics, "conics"), (colors, "colors")):
        _check_input(t, n, torch.float32)
    channels = colors.size(1)
    if channels > MAX_CHANNELS:
        raise RuntimeError("at most MAX_CHANNELS channels")
    dev = xys.device
    out_img = torch.empty(channels, h, w, device=dev, dtype=torch.float32)
    pixel_topk = torch.empty(h, w, TOP_K, device=dev, dtype=torch.int32)
    with torch.cuda.device(dev):
        _lib_call("igs_raster_fwd_topk", int(tile_bounds[0]), int(tile_bounds[1]), h, w, channels, ptr(gaussian_ids_sorted),
                  ptr(tile_bins), ptr(xys), ptr(conics), ptr(colors), ptr(out_img), ptr(pixel_topk), stream_of(dev))
    return out_img, pixel_topk


def nd_rasterize_forward_topk_norm_tiles(tile_bounds, img_size, max_list_len, gaussian_ids_sorted, tile_bins, xys, conics, colors):
    """The training-step forward: out_img [C,H,W] and the top-K lists as 16-bit tile-list positions [T,10,256] uint16."""
    h, w = _check_raster_geometry(tile_bounds, (TILE, TILE, 1), img_size)
    channels = colors.size(1)
    dev = xys.device
    num_tiles = int(tile_bounds[0]) * int(tile_bounds[1])
    out_img = torch.empty(channels, h, w, device=dev, dtype=torch.float32)
    tile_topk = torch.empty(num_tiles, TOP_K, TILE * TILE, device=dev, dtype=torch.int16)  # uint16 bit patterns
    with torch.cuda.device(dev):
        _lib_call("igs_raster_fwd_topk_tiles", int(tile_bounds[0]), int(tile_bounds[1]), h, w, channels, int(max_list_len),
                  ptr(gaussian_ids_sorted), ptr(tile_bins), ptr(xys), ptr(conics), ptr(colors), ptr(out_img), ptr(tile_topk),
                  stream_of(dev))
    return out_img, tile_topk


def nd_rasterize_forward_topk_norm_tiles_l1(tile_bounds, img_size, max_list_len, gaussian_ids_sorted, tile_bins, xys, conics, colors,
                                            target, ratio=1.0):
    """The training-step forward with the L1 loss fused: (out_img [C,H,W], tile_topk, loss = ratio * mean|out_img - target|,
    v_output = its gradient with respect to out_img); target [C,H,W] float32."""
    h, w = _check_raster_geometry(tile_bounds, (TILE, TILE, 1), img_size)
    channels = colors.size(1)
    _check_input(target, "target", torch.float32)
    if tuple(target.shape) != (channels, h, w):
        raise RuntimeError(f"target must be [{channels}, {h}, {w}]")
    dev = xys.device
    num_tiles = int(tile_bounds[0]) * int(tile_bounds[1])
    lib = _lib.load()
    out_img = torch.empty(channels, h, w, device=dev, dtype=torch.float32)
    v_output = torch.empty_like(out_img)
    loss = torch.empty((), device=dev, dtype=torch.float32)
    tile_topk = torch.empty(num_tiles, TOP_K, TILE * TILE, device=dev, dtype=torch.int16)
    ws_bytes = lib.igs_raster_l1_workspace(num_tiles)
    ws = torch.zeros(ws_bytes, device=dev, dtype=torch.uint8)
    with torch.cuda.device(dev):
        _lib_call("igs_raster_fwd_topk_tiles_l1", int(tile_bounds[0]), int(tile_bounds[1]), h, w, channels, int(max_list_len),
                  ptr(gaussian_ids_sorted), ptr(tile_bins), ptr(xys), ptr(conics), ptr(colors), ptr(target), float(ratio), ptr(out_img),
                  ptr(tile_topk), ptr(loss), ptr(v_output), ptr(ws), ws_bytes, stream_of(dev))
    return out_img, tile_topk, loss, v_output


def raster_step_l1(tile_bounds, img_size, gaussian_ids_sorted, tile_bins, xys, conics, colors, target, ratio=1.0, with_v_output=False):
    """The training step's rasterization with the L1 loss in one kernel (igs_raster_step_l1): out_img [C,H,W], loss = ratio *
    mean|out_img - target|, and the gradients of the loss v_xy [N,2], v_conic [N,3], v_colors [N,C] (plus v_output, the loss's gradient
    with respect to out_img, when with_v_output), as nd_rasterize_forward_topk_norm_tiles_l1 followed by
    nd_rasterize_backward_topk_norm_tiles would give them."""
    h, w = _check_raster_geometry(tile_bounds, (TILE, TILE, 1), img_size)
    _check_input(gaussian_ids_sorted, "gaussian_ids_sorted", torch.int32)
    _check_input(tile_bins, "tile_bins", torch.int32)
    for t, name in ((xys, "xys"), (conics, "conics"), (colors, "colors"), (target, "target")):
        _check_input(t, name, torch.float32)
    channels = colors.size(1)
    if channels > MAX_CHANNELS:
        raise RuntimeError(f"at most {MAX_CHANNELS} channels")
    if tuple(target.shape) != (channels, h, w):
        raise RuntimeError(f"target must be [{channels}, {h}, {w}]")
    n = xys.size(0)
    dev = xys.device
    num_tiles = int(tile_bounds[0]) * int(tile_bounds[1])
    lib = _lib.load()
    out_img = torch.empty(channels, h, w, device=dev, dtype=torch.float32)
    v_output = torch.empty_like(out_img) if with_v_output else None
    loss = torch.empty((), device=dev, dtype=torch.float32)
    grads = torch.empty(n * (5 + channels), device=dev, dtype=torch.float32)
    v_xy, v_conic, v_colors = grads[:2 * n].view(n, 2), grads[2 * n:5 * n].view(n, 3), grads[5 * n:].view(n, channels)
    ws_bytes = lib.igs_raster_l1_workspace(num_tiles)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    with torch.cuda.device(dev):
        _lib_call("igs_raster_step_l1", int(tile_bounds[0]), int(tile_bounds[1]), h, w, channels, n, ptr(gaussian_ids_sorted),
                  ptr(tile_bins), ptr(xys), ptr(conics), ptr(colors), ptr(target), float(ratio), ptr(out_img), ptr(loss), ptr(v_output),
                  ptr(v_xy), ptr(v_conic), ptr(v_colors), ptr(ws), ws_bytes, stream_of(dev))
    out = (out_img, loss, v_xy, v_conic, v_colors)
    return out + (v_output,) if with_v_output else out


def nd_rasterize_backward_topk_norm(img_height, img_width, BLOCK_H, BLOCK_W, xys, conics, colors, v_output, pixel_topk):
    """-> v_xy [N,2], v_conic [N,3], v_colors [N,C] (bindings.cu:444-502); v_output channel-planar [C,H,W]."""
    for t, n in ((xys, "xys"), (conics, "conics"), (colors, "colors"), (v_output, "v_output")):
        _check_input(t, n, torch.float32)
    _check_input(pixel_topk, "pixel_topk", torch.int32)
    if xys.ndim != 2 or xys.size(1) != 2:
        raise RuntimeError("xys must have dimensions (num_points, 2)")
    if colors.ndim != 2:
        raise RuntimeError("colors must have 2 dimensions")
    if BLOCK_W % 8 != 0 or BLOCK_H % 4 != 0 or (BLOCK_H, BLOCK_W) != (TILE, TILE):
        raise RuntimeError(f"the block must be {TILE}x{TILE} (warps cover 8x4 pixels)")
    channels = colors.size(1)
    if channels > MAX_CHANNELS:
        raise RuntimeError("at most MAX_CHANNELS channels")
    n = xys.size(0)
    dev = xys.device
    grads = torch.empty(n * (5 + channels), device=dev, dtype=torch.float32)
    v_xy, v_conic, v_colors = grads[:2 * n].view(n, 2), grads[2 * n:5 * n].view(n, 3), grads[5 * n:].view(n, channels)
    with torch.cuda.device(dev):
        _lib_call("igs_raster_bwd_topk", int(img_height), int(img_width), channels, n, ptr(xys), ptr(conics), ptr(colors), ptr(v_output),
                  ptr(pixel_topk), ptr(v_xy), ptr(v_conic), ptr(v_colors), stream_of(dev))
    return v_xy, v_conic, v_colors


def nd_rasterize_backward_topk_norm_tiles(img_height, img_width, gaussian_ids_sorted, tile_bins, xys, conics, colors, v_output, tile_topk):
    """Backward pass from the tile-list form of the top-K lists."""
    channels = colors.size(1)
    n = xys.size(0)
    dev = xys.device
    grads = torch.empty(n * (5 + channels), device=dev, dtype=torch.float32)
    v_xy, v_conic, v_colors = grads[:2 * n].view(n, 2), grads[2 * n:5 * n].view(n, 3), grads[5 * n:].view(n, channels)
    with torch.cuda.device(dev):
        _lib_call("igs_raster_bwd_topk_tiles", int(img_height), int(img_width), channels, n, ptr(gaussian_ids_sorted), ptr(tile_bins),
                  ptr(xys), ptr(conics), ptr(colors), ptr(v_output), ptr(tile_topk), ptr(v_xy), ptr(v_conic), ptr(v_colors),
                  stream_of(dev))
    return v_xy, v_conic, v_colors


def topk_norm_loo_loss_increase(img_height, img_width, xys, conics, colors, pixel_topk, targets, squared, eps):
    """-> loss_increase [N] (bindings.cu:895-936)."""
    for t, n in ((xys, "xys"), (conics, "conics"), (colors, "colors"), (targets, "targets")):
        _check_input(t, n, torch.float32)
    _check_input(pixel_topk, "pixel_topk", torch.int32)
    channels = colors.size(1)
    if channels > MAX_CHANNELS:
        raise RuntimeError("at most MAX_CHANNELS channels")
    if targets.numel() != channels * img_height * img_width:
        raise RuntimeError("targets must be [C, H, W]")
    if pixel_topk.numel() != img_height * img_width * TOP_K:
        raise RuntimeError("pixel_topk must be [H, W, TOP_K]")
    dev = xys.device
    out = torch.empty(xys.size(0), device=dev, dtype=torch.float32)
    with torch.cuda.device(dev):
        _lib_call("igs_loo_loss_increase", int(img_height), int(img_width), channels, xys.size(0), ptr(xys), ptr(conics), ptr(colors),
                  ptr(pixel_topk), ptr(targets), int(bool(squared)), float(eps), ptr(out), stream_of(dev))
    return out


def topk_feature_weights_fixed(img_height, img_width, xys, conics, pixel_topk, eps=EPS):
    """Per-Gaussian sum over pixels of the squared normalized top-K weight as int64 fixed point with 40 fractional bits: the integer sums
    of compress.quantization.feature_weights (quantization.py:218-230) over model._iter_topk_weights (model.py:1404-1421)."""
    for t, n in ((xys, "xys"), (conics, "conics")):
        _check_input(t, n, torch.float32)
    _check_input(pixel_topk, "pixel_topk", torch.int32)
    if pixel_topk.numel() != img_height * img_width * TOP_K:
        raise RuntimeError("pixel_topk must be [H, W, TOP_K]")
    dev = xys.device
    out = torch.empty(xys.size(0), device=dev, dtype=torch.int64)
    with torch.cuda.device(dev):
        _lib_call("igs_feature_weights", int(img_height), int(img_width), xys.size(0), ptr(xys), ptr(conics), ptr(pixel_topk), float(eps),
                  ptr(out), stream_of(dev))
    return out


def topk_feature_weights(img_height, img_width, xys, conics, pixel_topk, eps=EPS):
    """compress.quantization.feature_weights(model._iter_topk_weights(...)) -> [N] float64."""
    return topk_feature_weights_fixed(img_height, img_width, xys, conics, pixel_topk, eps).to(torch.float64) / 2.0**40


# ---- routing lists: balance and gate dropout ------------------------------------------------------------------------------------------

def _run(dev, name, *args):
    """One entry point on dev's current stream, the arguments (pointers as integers) before the stream. These operators are used on small
    images too, where the host's time is the time: the device is only changed where it is not the current one."""
    call = getattr(_lib.load(), name)
    if torch.cuda.current_device() == dev.index:
        status = call(*args, raw_stream_of(dev.index))
    else:
        with torch.cuda.device(dev):
            status = call(*args, raw_stream_of(dev.index))
    if status:
        check(status, name)


def _address(t):
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=256)
def _workspace_bytes(name, *sizes):
    return getattr(_lib.load(), name)(*sizes)


def _check_lists(img_height, img_width, xys, conics, pixel_topk, *others):
    """The inputs shared by the operators over pixel_topk: shapes, types, one device (others: further tensors, or None). Returns
    (H, W, N, device)."""
    h, w = int(img_height), int(img_width)
    if h < 0 or w < 0:
        raise ValueError(f"negative image size {w}x{h}")
    _check_input(xys, "xys", torch.float32)
    _check_input(conics, "conics", torch.float32)
    _check_input(pixel_topk, "pixel_topk", torch.int32)
    n = xys.size(0) if xys.ndim == 2 else -1
    if n < 0 or xys.size(1) != 2:
        raise RuntimeError("xys must have dimensions (num_points, 2)")
    if conics.ndim != 2 or conics.size(0) != n or conics.size(1) != 3:
        raise RuntimeError("conics must have dimensions (num_points, 3)")
    if pixel_topk.numel() != h * w * TOP_K:
        raise RuntimeError("pixel_topk must be [H, W, TOP_K]")
    if max(h, w, n) > 2**31 - 1:  # the entry points refuse what is past their limits, but would see the low 32 bits of these
        raise RuntimeError("at most 2^31 / 10 pixels, 65535 tiles a side and 2^26 Gaussians")
    dev = xys.device
    for t in (conics, pixel_topk) + others:
        if t is not None and t.device != dev:
            raise RuntimeError(f"every tensor must be on {dev}, as xys; got one on {t.device}")
    return h, w, n, dev


def _check_mask(pixel_mask, h, w):
    if pixel_mask is None:
        return
    _check_input(pixel_mask, "pixel_mask")
    if pixel_mask.dtype not in (torch.bool, torch.uint8):
        raise RuntimeError(f"pixel_mask must be torch.bool or torch.uint8, got {pixel_mask.dtype}")
    if pixel_mask.numel() != h * w:
        raise RuntimeError("pixel_mask must be [H, W]")


def topk_balance_forward(img_height, img_width, xys, conics, pixel_topk, pixel_mask=None):
    """How the pixels spread over the Gaussians: (loss (0-dim), counts [N] int32, importance [N], totals [2] int64). counts are the slots of
    pixel_topk that hold each Gaussian, importance the sum of their gates exp(-sigma) / (sum + 1e-4), totals the filled slots A and the
    pixels T with one, loss = N / (A T) * sum(counts * importance): 1 for an even spread, 0 without slots. pixel_mask [H, W] (bool or uint8)
    leaves pixels out. The results do not depend on the order of the atomics."""
    h, w, n, dev = _check_lists(img_height, img_width, xys, conics, pixel_topk, pixel_mask)
    _check_mask(pixel_mask, h, w)
    loss = torch.empty((), device=dev, dtype=torch.float32)
    counts = torch.empty(n, device=dev, dtype=torch.int32)
    importance = torch.empty(n, device=dev, dtype=torch.float32)
    totals = torch.empty(2, device=dev, dtype=torch.int64)
    ws_bytes = _workspace_bytes("igs_topk_balance_workspace", n)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    _run(dev, "igs_topk_balance_fwd", h, w, n, xys.data_ptr(), conics.data_ptr(), pixel_topk.data_ptr(), _address(pixel_mask),
         loss.data_ptr(), counts.data_ptr(), importance.data_ptr(), totals.data_ptr(), ws.data_ptr(), ws_bytes)
    return loss, counts, importance, totals


def topk_balance_backward(img_height, img_width, xys, conics, pixel_topk, counts, totals, grad_loss=None, grad_importance=None,
                          pixel_mask=None):
    """v_xy [N, 2], v_conic [N, 3] of grad_loss * loss + sum(grad_importance * importance), the counts held constant; counts, totals and
    pixel_mask as topk_balance_forward returned and took them, grad_loss a device scalar, grad_importance [N]."""
    h, w, n, dev = _check_lists(img_height, img_width, xys, conics, pixel_topk, counts, totals, grad_loss, grad_importance, pixel_mask)
    _check_mask(pixel_mask, h, w)
    _check_input(counts, "counts", torch.int32)
    _check_input(totals, "totals", torch.int64)
    if counts.numel() != n or totals.numel() != 2:
        raise RuntimeError("counts must be [N] and totals [2]")
    if grad_loss is not None:
        _check_input(grad_loss, "grad_loss", torch.float32)
        if grad_loss.numel() != 1:
            raise RuntimeError("grad_loss must hold one value")
    if grad_importance is not None:
        _check_input(grad_importance, "grad_importance", torch.float32)
        if grad_importance.numel() != n:
            raise RuntimeError("grad_importance must be [N]")
    v_xy, v_conic = torch.empty_like(xys), torch.empty_like(conics)
    ws_bytes = _workspace_bytes("igs_topk_balance_workspace", n)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    _run(dev, "igs_topk_balance_bwd", h, w, n, xys.data_ptr(), conics.data_ptr(), pixel_topk.data_ptr(), _address(pixel_mask),
         counts.data_ptr(), totals.data_ptr(), _address(grad_loss), _address(grad_importance), 0, v_xy.data_ptr(), v_conic.data_ptr(),
         ws.data_ptr(), ws_bytes)
    return v_xy, v_conic


def _check_dropout(h, w, n, colors, p, rng_state):
    _check_input(colors, "colors", torch.float32)
    if colors.ndim != 2 or colors.size(0) != n:
        raise RuntimeError("colors must have dimensions (num_points, channels)")
    channels = colors.size(1)
    if not 1 <= channels <= MAX_CHANNELS:
        raise RuntimeError(f"1 to {MAX_CHANNELS} channels, got {channels}")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must lie in [0, 1], got {p}")
    _check_input(rng_state, "rng_state", torch.int64)
    if rng_state.numel() != 2:
        raise RuntimeError("rng_state must hold a seed and an offset")
    return channels, p


def topk_dropout_forward(img_height, img_width, xys, conics, colors, pixel_topk, p, rng_state):
    """The render out_img [C, H, W] from the lists pixel_topk with every slot dropped with probability p before the weights are normalized
    (a pixel with nothing left is 0), and rng_used [2], the seed and offset that the pass saw in rng_state (int64 [2] on the device): the
    backward pass takes rng_used, and draws the same mask from it. Move the offset on between passes (rng_state[1] += 1, in a captured graph
    too) for a new mask."""
    h, w, n, dev = _check_lists(img_height, img_width, xys, conics, pixel_topk, colors, rng_state)
    channels, p = _check_dropout(h, w, n, colors, p, rng_state)
    out_img = torch.empty(channels, h, w, device=dev, dtype=torch.float32)
    rng_used = torch.empty(2, device=dev, dtype=torch.int64)
    _run(dev, "igs_topk_dropout_fwd", h, w, channels, n, xys.data_ptr(), conics.data_ptr(), colors.data_ptr(), pixel_topk.data_ptr(), p,
         rng_state.data_ptr(), out_img.data_ptr(), rng_used.data_ptr())
    return out_img, rng_used


def topk_dropout_backward(img_height, img_width, xys, conics, colors, v_output, pixel_topk, p, rng_used):
    """v_xy [N, 2], v_conic [N, 3], v_colors [N, C] of topk_dropout_forward, for v_output [C, H, W] and the rng_used it returned."""
    h, w, n, dev = _check_lists(img_height, img_width, xys, conics, pixel_topk, colors, v_output, rng_used)
    channels, p = _check_dropout(h, w, n, colors, p, rng_used)
    _check_input(v_output, "v_output", torch.float32)
    if v_output.numel() != channels * h * w:
        raise RuntimeError("v_output must be [C, H, W]")
    v_xy, v_conic, v_colors = torch.empty_like(xys), torch.empty_like(conics), torch.empty_like(colors)
    ws_bytes = _workspace_bytes("igs_topk_dropout_workspace", n, channels)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    _run(dev, "igs_topk_dropout_bwd", h, w, channels, n, xys.data_ptr(), conics.data_ptr(), colors.data_ptr(), v_output.data_ptr(),
         pixel_topk.data_ptr(), p, rng_used.data_ptr(), v_xy.data_ptr(), v_conic.data_ptr(), v_colors.data_ptr(), ws.data_ptr(),
         ws_bytes)
    return v_xy, v_conic, v_colors


# ---- losses, quantization, rate term -------------------------------------------------------------------------------------------------

def l1_loss_and_grad(image: torch.Tensor, target: torch.Tensor, ratio: float = 1.0, workspace: Optional[torch.Tensor] = None):
    """(ratio * mean|image - target| as a 0-dim tensor, its gradient with respect to image), in one pass."""
    _check_input(image, "image", torch.float32)
    _check_input(target, "target", torch.float32)
    if image.shape != target.shape:
        raise ValueError(f"image {tuple(image.shape)} and target {tuple(target.shape)} differ")
    dev = image.device
    numel = image.numel()
    loss = torch.empty((), device=dev, dtype=torch.float32)
    grad = torch.empty_like(image)
    ws_bytes = _lib.load().igs_l1_workspace(numel)
    if workspace is None:
        workspace = torch.zeros(ws_bytes, device=dev, dtype=torch.uint8)
    with torch.cuda.device(dev):
        _lib_call("igs_l1_loss", numel, ptr(image), ptr(target), float(ratio), ptr(loss), ptr(grad), ptr(workspace), ws_bytes,
                  stream_of(dev))
    return loss, grad


def l1_loss_signs(image: torch.Tensor, target: torch.Tensor, ratio: float = 1.0, workspace: Optional[torch.Tensor] = None):
    """(ratio * mean|image - target| as a 0-dim tensor, sign(image - target) as int8), in one pass; see igs_l1_loss_signs."""
    _check_input(image, "image", torch.float32)
    _check_input(target, "target", torch.float32)
    if image.shape != target.shape:
        raise ValueError(f"image {tuple(image.shape)} and target {tuple(target.shape)} differ")
    dev = image.device
    loss = torch.empty((), device=dev, dtype=torch.float32)
    signs = torch.empty(image.shape, device=dev, dtype=torch.int8)
    ws_bytes = _lib.load().igs_l1_workspace(image.numel())
    if workspace is None:
        workspace = torch.zeros(ws_bytes, device=dev, dtype=torch.uint8)
    with torch.cuda.device(dev):
        _lib_call("igs_l1_loss_signs", image.numel(), ptr(image), ptr(target), float(ratio), ptr(loss), ptr(signs), ptr(workspace),
                  ws_bytes, stream_of(dev))
    return loss, signs


def l1_grad_from_signs(signs: torch.Tensor, grad_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """sign * (g / numel) as float32 (g = grad_scale, a device scalar, or 1): the gradient of mean|image - target|, as ATen forms it."""
    _check_input(signs, "signs", torch.int8)
    dev = signs.device
    grad = torch.empty(signs.shape, device=dev, dtype=torch.float32)
    scale = None
    if grad_scale is not None:
        scale = grad_scale.detach().to(device=dev, dtype=torch.float32).contiguous()
        if scale.numel() != 1:
            raise ValueError("grad_scale must hold one value")
    with torch.cuda.device(dev):
        _lib_call("igs_l1_grad_from_signs", signs.numel(), ptr(signs), ptr(scale) if scale is not None else None, ptr(grad),
                  stream_of(dev))
    return grad


def quantize_ste_forward(xy, scale, rot, feat, pos_steps, scale_step, rot_step, feat_steps, feat_transform=None, with_symbols=False):
    """Straight-through step quantization values (and optionally symbols and loss-space features); see igs_quantize_ste."""
    for t, n in ((xy, "xy"), (scale, "scale"), (rot, "rot"), (feat, "feat"), (pos_steps, "pos_steps"), (feat_steps, "feat_steps")):
        _check_input(t, n, torch.float32)
    n, channels = feat.shape
    dev = xy.device
    out = [torch.empty_like(xy), torch.empty_like(scale), torch.empty_like(rot), torch.empty_like(feat)]
    out_t = torch.empty_like(feat) if feat_transform is not None else None
    sym = [torch.empty_like(xy), torch.empty_like(scale), torch.empty_like(rot), torch.empty_like(feat)] if with_symbols else [None] * 4
    if feat_transform is not None:
        _check_input(feat_transform, "feat_transform", torch.float32)
    with torch.cuda.device(dev):
        _lib_call("igs_quantize_ste", n, channels, ptr(xy), ptr(scale), ptr(rot), ptr(feat), ptr(pos_steps), float(scale_step),
                  float(rot_step), ptr(feat_steps), ptr(feat_transform), *[ptr(t) for t in out], ptr(out_t), *[ptr(t) for t in sym],
                  stream_of(dev))
    return out, out_t, (sym if with_symbols else None)


def rate_loss_forward(feat, rot, l1_loss, neighbors, weights, slope, color_refs, pred_refs, inv_steps, feat_coeffs, rot_coeffs,
                      inv_rot_step, l1_ratio, factor):
    """-> loss (0-dim), loss_weight [1], own_grad [N,C], rot_grad [N] (rate.cu:201-279)."""
    for t, n in ((feat, "feat"), (rot, "rot"), (l1_loss, "l1_loss"), (weights, "weights"), (slope, "slope"), (inv_steps, "inv_steps"),
                 (feat_coeffs, "feat_coeffs"), (rot_coeffs, "rot_coeffs")):
        _check_input(t, n, torch.float32)
    _check_input(neighbors, "neighbors", torch.int32)
    num, channels = feat.shape
    if channels > MAX_CHANNELS:
        raise RuntimeError("at most MAX_CHANNELS feature channels")
    if len(color_refs) != channels or len(pred_refs) != channels:
        raise RuntimeError("one reference per channel")
    if rot.numel() != num or rot_coeffs.numel() != num:
        raise RuntimeError("one rotation per Gaussian")
    if neighbors.size(0) != num or weights.shape != neighbors.shape:
        raise RuntimeError("neighbors and weights must be [P, K]")
    dev = feat.device
    loss = torch.empty((), device=dev, dtype=torch.float32)
    loss_weight = torch.empty(1, device=dev, dtype=torch.float32)
    own_grad = torch.empty_like(feat)
    rot_grad = torch.empty(num, device=dev, dtype=torch.float32)
    ws_bytes = _lib.load().igs_rate_workspace(num)
    ws = torch.zeros(ws_bytes, device=dev, dtype=torch.uint8)
    import ctypes
    crefs = (ctypes.c_int32 * channels)(*[int(c) for c in color_refs])
    prefs = (ctypes.c_int32 * channels)(*[int(c) for c in pred_refs])
    with torch.cuda.device(dev):
        _lib_call("igs_rate_fwd", num, channels, neighbors.size(1), ptr(feat), ptr(rot), ptr(l1_loss), ptr(neighbors), ptr(weights),
                  ptr(slope), ctypes.cast(crefs, ctypes.c_void_p), ctypes.cast(prefs, ctypes.c_void_p), ptr(inv_steps), ptr(feat_coeffs),
                  ptr(rot_coeffs), float(inv_rot_step), float(l1_ratio), float(factor), ptr(loss), ptr(loss_weight), ptr(own_grad),
                  ptr(rot_grad), ptr(ws), ws_bytes, stream_of(dev))
    return loss, loss_weight, own_grad, rot_grad


def rate_loss_backward(grad_loss, loss_weight, own_grad, rot_grad, offsets, sources, source_weights):
    """-> grad_feat [N,C], grad_rot [N] (rate.cu:281-321)."""
    for t, n in ((grad_loss, "grad_loss"), (loss_weight, "loss_weight"), (own_grad, "own_grad"), (rot_grad, "rot_grad"),
                 (source_weights, "source_weights")):
        _check_input(t, n, torch.float32)
    _check_input(offsets, "offsets", torch.int32)
    _check_input(sources, "sources", torch.int32)
    num, channels = own_grad.shape
    if offsets.numel() != num + 1:
        raise RuntimeError("offsets must be [P + 1]")
    dev = own_grad.device
    grad_feat = torch.empty_like(own_grad)
    grad_rot = torch.empty_like(rot_grad)
    with torch.cuda.device(dev):
        _lib_call("igs_rate_bwd", num, channels, ptr(grad_loss), ptr(loss_weight), ptr(own_grad), ptr(rot_grad), ptr(offsets),
                  ptr(sources), ptr(source_weights), ptr(grad_feat), ptr(grad_rot), stream_of(dev))
    return grad_feat, grad_rot
