// The render from given top-K lists with gates dropped before the normalization, and its backward pass. A dropped slot leaves its pixel's
// sums as if its Gaussian were not there, which is what the leave-one-out pruning score evaluates (loo.cu):
//   out_c = sum_kept w_k f_kc / (sum_kept w_k + eps)          (0 where no slot is kept)
// and with gates n_k = w_k / (sum_kept w_j + eps), s_k = f_k . v_out:
//   v_f += n_k v_out,  dL/dsigma_k = -n_k (s_k - sum_j n_j s_j),  and the geometry's gradients from dL/dsigma as in balance.cu.
// The mask is drawn from the pixel's index and two 64-bit values on the device, seed and offset (keep_bits in topk_lists.cuh), in the
// forward pass and again in the backward pass, so it is never stored, and a captured graph draws a new one whenever the offset has moved.
#include "topk_lists.cuh"

namespace {

using igs::kMaxChannels;
using igs::kTopK;

constexpr int kThreads = 256;

size_t workspace_bytes_of(int num_points, int channels) { return 16; }

struct Slots {
    int id[kTopK];  // -1: empty or dropped
    float dx[kTopK], dy[kTopK], gate[kTopK];
};

__device__ __forceinline__ void read_slots(Slots &s, const int p, const int img_w, const int n, const float2 *xys, const float *conics,
                                           const int *pixel_topk, const unsigned keep) {
    const float px = (float)(p % img_w), py = (float)(p / img_w);
    const int2 *row = reinterpret_cast<const int2 *>(pixel_topk + (size_t)p * kTopK);
    float sum = (float)igs::kNormEps;
#pragma unroll
    for (int k = 0; k < kTopK; k += 2) {
        const int2 v = __ldg(&row[k / 2]);
        s.id[k] = (unsigned)v.x < (unsigned)n && (keep >> k & 1) ? v.x : -1;
        s.id[k + 1] = (unsigned)v.y < (unsigned)n && (keep >> (k + 1) & 1) ? v.y : -1;
    }
#pragma unroll
    for (int k = 0; k < kTopK; ++k) {
        s.gate[k] = 0.f;
        if (s.id[k] < 0) continue;
        const float2 xy = __ldg(&xys[s.id[k]]);
        const float *c = conics + 3 * (size_t)s.id[k];
        s.dx[k] = xy.x - px, s.dy[k] = xy.y - py;
        s.gate[k] = igs::slot_weight(igs::gaussian_sigma(xy.x, xy.y, __ldg(&c[0]), __ldg(&c[1]), __ldg(&c[2]), px, py));
        sum += s.gate[k];
    }
    const float inv = 1.f / sum;
#pragma unroll
    for (int k = 0; k < kTopK; ++k) s.gate[k] *= inv;
}

__global__ void __launch_bounds__(kThreads) dropout_fwd_kernel(const int pixels, const int img_w, const int channels, const int n,
                                                               const float2 *__restrict__ xys, const float *__restrict__ conics,
                                                               const float *__restrict__ colors, const int *__restrict__ pixel_topk,
                                                               const uint32_t threshold, const long long *__restrict__ rng,
                                                               float *__restrict__ out_img, long long *__restrict__ rng_used) {
    const int p = blockIdx.x * kThreads + threadIdx.x;
    const long long seed = rng[0], offset = rng[1];
    if (p == 0) rng_used[0] = seed, rng_used[1] = offset;
    if (p >= pixels) return;
    Slots s;
    read_slots(s, p, img_w, n, xys, conics, pixel_topk, igs::keep_bits(p, seed, offset, threshold));
    float pix[kMaxChannels];
#pragma unroll
    for (int c = 0; c < kMaxChannels; ++c) pix[c] = 0.f;
#pragma unroll
    for (int k = 0; k < kTopK; ++k) {
        if (s.id[k] < 0) continue;
#pragma unroll
        for (int c = 0; c < kMaxChannels; ++c)
            if (c < channels) pix[c] += s.gate[k] * __ldg(&colors[(size_t)s.id[k] * channels + c]);
    }
#pragma unroll
    for (int c = 0; c < kMaxChannels; ++c)
        if (c < channels) out_img[(size_t)c * pixels + p] = pix[c];
}

__global__ void __launch_bounds__(kThreads) dropout_bwd_kernel(const int pixels, const int img_w, const int channels, const int n,
                                                               const float2 *__restrict__ xys, const float *__restrict__ conics,
                                                               const float *__restrict__ colors, const float *__restrict__ v_output,
                                                               const int *__restrict__ pixel_topk, const uint32_t threshold,
                                                               const long long *__restrict__ rng, float *__restrict__ v_xy,
                                                               float *__restrict__ v_conic, float *__restrict__ v_colors) {
    const int p = blockIdx.x * kThreads + threadIdx.x;
    if (p >= pixels) return;
    Slots s;
    read_slots(s, p, img_w, n, xys, conics, pixel_topk, igs::keep_bits(p, rng[0], rng[1], threshold));
    float score[kTopK], mean = 0.f;
#pragma unroll
    for (int k = 0; k < kTopK; ++k) {
        score[k] = 0.f;
        if (s.id[k] < 0) continue;
        for (int c = 0; c < channels; ++c) {
            const float v = __ldg(&v_output[(size_t)c * pixels + p]);
            score[k] += __ldg(&colors[(size_t)s.id[k] * channels + c]) * v;
            atomicAdd(&v_colors[(size_t)s.id[k] * channels + c], s.gate[k] * v);
        }
        mean += s.gate[k] * score[k];
    }
#pragma unroll
    for (int k = 0; k < kTopK; ++k) {
        const int g = s.id[k];
        if (s.gate[k] == 0.f) continue;  // empty, or a Gaussian whose parameters may not even be finite
        const float t = s.gate[k] * (mean - score[k]);
        const float *c = conics + 3 * (size_t)g;
        atomicAdd(&v_xy[2 * (size_t)g], t * (c[0] * s.dx[k] + c[1] * s.dy[k]));
        atomicAdd(&v_xy[2 * (size_t)g + 1], t * (c[1] * s.dx[k] + c[2] * s.dy[k]));
        atomicAdd(&v_conic[3 * (size_t)g], 0.5f * t * s.dx[k] * s.dx[k]);
        atomicAdd(&v_conic[3 * (size_t)g + 1], t * s.dx[k] * s.dy[k]);
        atomicAdd(&v_conic[3 * (size_t)g + 2], 0.5f * t * s.dy[k] * s.dy[k]);
    }
}

}  // namespace

extern "C" {

size_t igs_topk_dropout_workspace(int num_points, int channels) { return num_points < 0 || channels < 0 ? 0 : workspace_bytes_of(num_points, channels); }

int igs_topk_dropout_fwd(int img_height, int img_width, int channels, int num_points, const float *xys, const float *conics,
                         const float *colors, const int32_t *pixel_topk, double p, const int64_t *rng_state, float *out_img,
                         int64_t *rng_used, void *workspace, size_t workspace_bytes, void *stream) {
    IGS_REQUIRE(img_height >= 0 && img_width >= 0 && num_points >= 0, "igs_topk_dropout_fwd: negative size");
    IGS_REQUIRE(channels >= 1 && channels <= kMaxChannels, "igs_topk_dropout_fwd: 1 to %d channels", kMaxChannels);
    IGS_REQUIRE(igs::lists_addressable(img_height, img_width), "igs_topk_dropout_fwd: at most 2^31 / 10 pixels and 2^24 a side");
    IGS_REQUIRE(p >= 0.0 && p <= 1.0, "igs_topk_dropout_fwd: p must lie in [0, 1]");
    IGS_REQUIRE(workspace && workspace_bytes >= workspace_bytes_of(num_points, channels), "igs_topk_dropout_fwd: workspace too small");
    IGS_REQUIRE(igs::aligned(workspace, 16), "igs_topk_dropout_fwd: workspace must be 16-byte aligned");
    IGS_REQUIRE(rng_state && rng_used, "igs_topk_dropout_fwd: null rng state");
    const int pixels = img_height * img_width;
    IGS_REQUIRE(pixels == 0 || (pixel_topk && out_img && (num_points == 0 || (xys && conics && colors))),
                "igs_topk_dropout_fwd: null pointer");
    IGS_REQUIRE(igs::aligned(xys, 8) && igs::aligned(pixel_topk, 8), "igs_topk_dropout_fwd: xys and pixel_topk must be 8-byte aligned");
    const int blocks = pixels > 0 ? igs::ceil_div(pixels, kThreads) : 1;
    dropout_fwd_kernel<<<blocks, kThreads, 0, igs::as_stream(stream)>>>(
        pixels, img_width, channels, num_points, reinterpret_cast<const float2 *>(xys), conics, colors, pixel_topk,
        (uint32_t)rint(p * 16777216.0), reinterpret_cast<const long long *>(rng_state), out_img, reinterpret_cast<long long *>(rng_used));
    return igs::check_launch("igs_topk_dropout_fwd");
}

int igs_topk_dropout_bwd(int img_height, int img_width, int channels, int num_points, const float *xys, const float *conics,
                         const float *colors, const float *v_output, const int32_t *pixel_topk, double p, const int64_t *rng_used,
                         float *v_xy, float *v_conic, float *v_colors, void *workspace, size_t workspace_bytes, void *stream) {
    IGS_REQUIRE(img_height >= 0 && img_width >= 0 && num_points >= 0, "igs_topk_dropout_bwd: negative size");
    IGS_REQUIRE(channels >= 1 && channels <= kMaxChannels, "igs_topk_dropout_bwd: 1 to %d channels", kMaxChannels);
    IGS_REQUIRE(igs::lists_addressable(img_height, img_width), "igs_topk_dropout_bwd: at most 2^31 / 10 pixels and 2^24 a side");
    IGS_REQUIRE(p >= 0.0 && p <= 1.0, "igs_topk_dropout_bwd: p must lie in [0, 1]");
    if (num_points == 0) return IGS_OK;
    IGS_REQUIRE(workspace && workspace_bytes >= workspace_bytes_of(num_points, channels), "igs_topk_dropout_bwd: workspace too small");
    IGS_REQUIRE(igs::aligned(workspace, 16), "igs_topk_dropout_bwd: workspace must be 16-byte aligned");
    IGS_REQUIRE(v_xy && v_conic && v_colors, "igs_topk_dropout_bwd: null output");
    const int pixels = img_height * img_width;
    IGS_REQUIRE(pixels == 0 || (xys && conics && colors && v_output && pixel_topk && rng_used), "igs_topk_dropout_bwd: null pointer");
    IGS_REQUIRE(igs::aligned(xys, 8) && igs::aligned(pixel_topk, 8), "igs_topk_dropout_bwd: xys and pixel_topk must be 8-byte aligned");
    cudaStream_t s = igs::as_stream(stream);
    cudaMemsetAsync(v_xy, 0, sizeof(float) * 2 * (size_t)num_points, s);
    cudaMemsetAsync(v_conic, 0, sizeof(float) * 3 * (size_t)num_points, s);
    cudaMemsetAsync(v_colors, 0, sizeof(float) * channels * (size_t)num_points, s);
    if (pixels > 0)
        dropout_bwd_kernel<<<igs::ceil_div(pixels, kThreads), kThreads, 0, s>>>(
            pixels, img_width, channels, num_points, reinterpret_cast<const float2 *>(xys), conics, colors, v_output, pixel_topk,
            (uint32_t)rint(p * 16777216.0), reinterpret_cast<const long long *>(rng_used), v_xy, v_conic, v_colors);
    return igs::check_launch("igs_topk_dropout_bwd");
}

}  // extern "C"
