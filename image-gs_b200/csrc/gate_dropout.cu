// The render from given top-K lists with gates dropped before the normalization, and its backward pass. A dropped slot leaves its pixel's
// sums as if its Gaussian were not there, which is what the leave-one-out pruning score evaluates (loo.cu):
//   out_c = sum_kept w_k f_kc / (sum_kept w_k + eps)          (0 where no slot is kept)
// and with gates n_k = w_k / (sum_kept w_j + eps), s_k = f_k . v_out:
//   v_f += n_k v_out,  dL/dsigma_k = -n_k (s_k - sum_j n_j s_j),  and the geometry's gradients from dL/dsigma (topk_sums.cuh).
// The mask is drawn from the pixel's index and two 64-bit values on the device, seed and offset (KeptSlots in topk_lists.cuh), in the
// forward pass and again in the backward pass, so it is never stored, and a captured graph draws a new one whenever the offset has moved.
//
// The render takes 56 us at 1920x1080 with 20,000 Gaussians and three channels, 213 us at 3840x2160 with 80,000 (the lists and the image at
// the memory's rate: 17 and 66 us), bound as topk_lists.cuh says, here with a quarter of the instructions in the generator; one thread per
// pixel that gathers its ten Gaussians took 89 and 355 us.
#include "topk_sums.cuh"

namespace {

using igs::kMaxChannels;
using igs::kPix;
using igs::kTile;
using igs::kTopK;

struct DropoutArgs {
    int img_h, img_w, channels, n;
    const float *xys, *conics, *colors;
    const int *pixel_topk;
    uint32_t threshold;
    const long long *rng;
    float *out_img;
    long long *rng_used;
};

// One pixel's slots one by one, from global memory
__device__ __forceinline__ void blend_pixel_slots(const DropoutArgs &a, const int p) {
    const igs::KeptSlots kept({(uint64_t)a.rng[0], (uint64_t)a.rng[1], a.threshold}, (uint32_t)p, true);
    unsigned keep = 0;
#pragma unroll
    for (int k = 0; k < kTopK; ++k) keep |= kept.any() && kept(k) ? 1u << k : 0u;
    const float px = (float)(p % a.img_w), py = (float)(p / a.img_w);
    const int *list = a.pixel_topk + (size_t)p * kTopK;
    float *out = a.out_img + p;
    const size_t plane = (size_t)a.img_h * a.img_w;
    for (int c = 0; c < a.channels; ++c) {
        float total = (float)igs::kNormEps, pix = 0.f;
        for (int k = 0; k < kTopK; ++k) {
            const int id = list[k];
            if ((unsigned)id >= (unsigned)a.n || !(keep >> k & 1)) continue;
            const float w = igs::slot_weight(igs::row_geometry(a.xys, a.conics, id), px, py);
            if (w == 0.f) continue;
            total += w;
            pix = fmaf(w, __ldg(&a.colors[(size_t)id * a.channels + c]), pix);
        }
        out[c * plane] = pix / total;
    }
}

__device__ __noinline__ void blend_slots(const DropoutArgs &a) {
    const igs::Patch patch(a.img_h, a.img_w);  // (made again: passed from the caller, it would live in the caller's local memory)
#pragma unroll
    for (int b = 0; b < kPix; ++b)
        if (patch.inside[b]) blend_pixel_slots(a, patch.p[b]);
}

template <int C>
struct DropoutSmem {
    int keys[igs::kKeyWords];
    float4 pairs[igs::Rows<C>::kGroupQuads];
};

__device__ __forceinline__ igs::PatchRows dropout_rows(const DropoutArgs &a, const igs::Patch &patch, const int g, int *keys) {
    return igs::find_rows(
        a.pixel_topk, patch, a.n,
        [&](const int p, const bool inside) {
            return igs::KeptSlots({(uint64_t)a.rng[0], (uint64_t)a.rng[1], a.threshold}, (uint32_t)p, inside);
        },
        g, keys);
}

template <int C>
__device__ __forceinline__ bool dropout_gather(const DropoutArgs &a, const igs::PatchRows &rows, float4 *pairs) {
    return igs::Rows<C>::gather(
        rows, a.xys, a.conics, [&](const int id, const int c) { return __ldg(&a.colors[(size_t)id * C + c]); }, pairs);
}

// A lane is its pixels: their weights' and weighted colours' sums over the rows
template <int C>
struct Blend {
    float2 total[kPix], pix[kPix][C];
    __device__ __forceinline__ Blend() {
#pragma unroll
        for (int b = 0; b < kPix; ++b) {
            total[b] = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < C; ++c) pix[b][c] = make_float2(0.f, 0.f);
        }
    }
    __device__ __forceinline__ void add(const igs::Patch &patch, const igs::PatchRows &rows, const float4 *pairs) {
        const float2 minus_x = make_float2(-(float)patch.j, -(float)patch.j);
        float2 minus_y[kPix];
        unsigned held[kPix];
#pragma unroll
        for (int b = 0; b < kPix; ++b) minus_y[b] = make_float2(-(float)patch.i[b], -(float)patch.i[b]), held[b] = rows.bits[b];
#pragma unroll 1
        for (int pair = 0; 2 * pair < rows.n; ++pair, pairs += igs::Rows<C>::kPairQuads) {
            float2 w[kPix];
            igs::Rows<C>::weights(pairs, held, minus_x, minus_y, w);
#pragma unroll
            for (int b = 0; b < kPix; ++b) {
                held[b] >>= 2;
                total[b] = igs::add2(total[b], w[b]);
#pragma unroll
                for (int c = 0; c < C; ++c) pix[b][c] = igs::fma2(w[b], igs::Rows<C>::value(pairs, c), pix[b][c]);
            }
        }
    }
    __device__ __forceinline__ void store(const DropoutArgs &a, const igs::Patch &patch) const {
        const size_t plane = (size_t)a.img_h * a.img_w;
#pragma unroll
        for (int b = 0; b < kPix; ++b) {
            if (!patch.inside[b]) continue;
            const float inv = igs::reciprocal(total[b].x + total[b].y + (float)igs::kNormEps);
#pragma unroll
            for (int c = 0; c < C; ++c) a.out_img[c * plane + patch.p[b]] = (pix[b][c].x + pix[b][c].y) * inv;
        }
    }
};

// A patch of more rows than a group's
template <int C>
__device__ __noinline__ bool blend_groups(const DropoutArgs &a, DropoutSmem<C> &sm) {
    const igs::Patch patch(a.img_h, a.img_w);
    Blend<C> blend;
    bool more = true;
    for (int g = 0; more; ++g) {
        const igs::PatchRows rows = dropout_rows(a, patch, g, sm.keys);
        more = rows.more;
        if (!dropout_gather<C>(a, rows, sm.pairs)) return false;
        __syncwarp();
        blend.add(patch, rows, sm.pairs);
    }
    blend.store(a, patch);
    return true;
}

// A warp is a patch
template <int C>
// (at 3840x2160: 213 us with 8 CTAs on an SM, 218 with 7, 220 with 9)
__global__ void __launch_bounds__(igs::kPatchThreads, C <= 3 ? 8 : C <= 7 ? 7 : 6) dropout_kernel(const __grid_constant__ DropoutArgs a) {
    __shared__ DropoutSmem<C> smem[igs::kPatches];
    DropoutSmem<C> &sm = smem[threadIdx.x >> 5];
    igs::wait_for_predecessor();
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 2) a.rng_used[threadIdx.x] = a.rng[threadIdx.x];
    const igs::Patch patch(a.img_h, a.img_w);
    if (patch.x0 >= a.img_w || patch.y0 >= a.img_h) return;
    const igs::PatchRows rows = dropout_rows(a, patch, 0, sm.keys);
    bool regular;
    if (rows.more) {
        regular = blend_groups<C>(a, sm);
    } else {
        regular = dropout_gather<C>(a, rows, sm.pairs);
        __syncwarp();
        if (regular) {
            Blend<C> blend;
            blend.add(patch, rows, sm.pairs);
            blend.store(a, patch);
        }
    }
    if (!regular) blend_slots(a);  // among others, zero times a colour that is not finite would reach pixels that do not name it
}

__global__ void rng_used_kernel(const long long *rng, long long *rng_used) {
    igs::wait_for_predecessor();
    rng_used[0] = rng[0], rng_used[1] = rng[1];
}

// One kernel for each number of channels
template <int C = kMaxChannels, typename F>
void with_channels(const int channels, F f) {
    if constexpr (C > 1) {
        if (channels < C) return with_channels<C - 1>(channels, f);
    }
    f(std::integral_constant<int, C>());
}

size_t workspace_bytes_of(int num_points, int channels) {
    size_t bytes = 0;
    with_channels(channels, [&](auto count) { bytes = igs::sum_bytes<decltype(count)::value, true>(num_points); });
    return bytes;
}

}  // namespace

extern "C" {

size_t igs_topk_dropout_workspace(int num_points, int channels) {
    return num_points < 0 || channels < 0 ? 0 : workspace_bytes_of(num_points, channels);
}

int igs_topk_dropout_fwd(int img_height, int img_width, int channels, int num_points, const float *xys, const float *conics,
                         const float *colors, const int32_t *pixel_topk, double p, const int64_t *rng_state, float *out_img,
                         int64_t *rng_used, void *stream) {
    IGS_REQUIRE(img_height >= 0 && img_width >= 0 && num_points >= 0, "igs_topk_dropout_fwd: negative size");
    IGS_REQUIRE(channels >= 1 && channels <= kMaxChannels, "igs_topk_dropout_fwd: 1 to %d channels", kMaxChannels);
    IGS_REQUIRE(igs::lists_addressable(img_height, img_width, num_points), "igs_topk_dropout_fwd: %s", igs::kListsLimit);
    IGS_REQUIRE(p >= 0.0 && p <= 1.0, "igs_topk_dropout_fwd: p must lie in [0, 1]");
    IGS_REQUIRE(rng_state && rng_used, "igs_topk_dropout_fwd: null rng state");
    const int pixels = img_height * img_width;
    IGS_REQUIRE(pixels == 0 || (pixel_topk && out_img && (num_points == 0 || (xys && conics && colors))),
                "igs_topk_dropout_fwd: null pointer");
    IGS_REQUIRE(igs::aligned(pixel_topk, 8), "igs_topk_dropout_fwd: pixel_topk must be 8-byte aligned");
    cudaStream_t s = igs::as_stream(stream);
    const long long *rng = reinterpret_cast<const long long *>(rng_state);
    long long *used = reinterpret_cast<long long *>(rng_used);
    if (pixels == 0) {
        igs::launch(rng_used_kernel, dim3(1), dim3(1), 0, s, rng, used);
    } else {
        const DropoutArgs a = {img_height, img_width, channels, num_points, xys, conics, colors, pixel_topk,
                               (uint32_t)rint(p * 16777216.0), rng, out_img, used};
        with_channels(channels, [&](auto count) {
            igs::launch(dropout_kernel<decltype(count)::value>, igs::tile_grid(img_height, img_width), dim3(igs::kPatchThreads), 0, s, a);
        });
    }
    return igs::check_launch("igs_topk_dropout_fwd");
}

int igs_topk_dropout_bwd(int img_height, int img_width, int channels, int num_points, const float *xys, const float *conics,
                         const float *colors, const float *v_output, const int32_t *pixel_topk, double p, const int64_t *rng_used,
                         float *v_xy, float *v_conic, float *v_colors, void *workspace, size_t workspace_bytes, void *stream) {
    IGS_REQUIRE(img_height >= 0 && img_width >= 0 && num_points >= 0, "igs_topk_dropout_bwd: negative size");
    IGS_REQUIRE(channels >= 1 && channels <= kMaxChannels, "igs_topk_dropout_bwd: 1 to %d channels", kMaxChannels);
    IGS_REQUIRE(igs::lists_addressable(img_height, img_width, num_points), "igs_topk_dropout_bwd: %s", igs::kListsLimit);
    IGS_REQUIRE(p >= 0.0 && p <= 1.0, "igs_topk_dropout_bwd: p must lie in [0, 1]");
    if (num_points == 0) return IGS_OK;
    IGS_REQUIRE(workspace && workspace_bytes >= workspace_bytes_of(num_points, channels), "igs_topk_dropout_bwd: workspace too small");
    IGS_REQUIRE(igs::aligned(workspace, 16), "igs_topk_dropout_bwd: workspace must be 16-byte aligned");
    IGS_REQUIRE(v_xy && v_conic && v_colors, "igs_topk_dropout_bwd: null output");
    const int pixels = img_height * img_width;
    IGS_REQUIRE(xys && conics && colors && (pixels == 0 || (v_output && pixel_topk && rng_used)), "igs_topk_dropout_bwd: null pointer");
    IGS_REQUIRE(igs::aligned(pixel_topk, 8), "igs_topk_dropout_bwd: pixel_topk must be 8-byte aligned");
    cudaStream_t s = igs::as_stream(stream);
    igs::SumArgs a = {};
    a.img_h = img_height, a.img_w = img_width, a.channels = channels, a.n = num_points;
    a.xys = xys, a.conics = conics, a.colors = colors, a.v_output = v_output, a.pixel_topk = pixel_topk;
    a.rng = reinterpret_cast<const long long *>(rng_used), a.threshold = (uint32_t)rint(p * 16777216.0);
    a.v_xy = v_xy, a.v_conic = v_conic, a.v_colors = v_colors;
    with_channels(channels, [&](auto count) {
        igs::launch_sums<decltype(count)::value, true>(a, workspace, s);
    });
    return igs::check_launch("igs_topk_dropout_bwd");
}

}  // extern "C"
