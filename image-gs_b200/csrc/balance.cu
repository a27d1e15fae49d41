// How the pixels spread over the Gaussians: the load of a top-K router whose tokens are the pixels and whose experts are the Gaussians.
// With n_pk the gates of the filled slots (topk_lists.cuh):
//   counts_g = filled slots that hold g,  importance_g = sum of their gates,  A = sum_g counts_g,  T = pixels with a filled slot
//   loss = N / (A T) sum_g counts_g importance_g     (0 when A = 0; 1 when every Gaussian has the same share and the gates sum to one)
// and, the counts held constant, with alpha_g = v_loss N counts_g / (A T) + v_importance_g:
//   dL/dsigma_k = -n_k (alpha_k - sum_j n_j alpha_j),
//   v_xy += dL/dsigma (a dx + b dy, b dx + c dy),  v_conic += dL/dsigma (dx^2 / 2, dx dy, dy^2 / 2).
//
// The importance is summed as 64-bit fixed point with as many fractional bits as the image leaves room for (a Gaussian's importance is at
// most the pixel count), so the sums, and the loss, do not depend on the order of the atomics.
#include "topk_lists.cuh"

namespace {

using igs::kTopK;

constexpr int kThreads = 256;

struct BalanceWorkspace {
    unsigned long long filled;  // A
    unsigned long long routed;  // T
    unsigned int ticket;
    unsigned int pad[11];
    // then uint64 fixed [n] and double partials [blocks of the finish kernel]
};

int finish_blocks(int n) { return n > 0 ? igs::ceil_div(n, kThreads) : 1; }

size_t fixed_offset() { return sizeof(BalanceWorkspace); }
size_t partials_offset(int n) { return fixed_offset() + sizeof(unsigned long long) * (size_t)n; }
size_t workspace_bytes_of(int n) { return partials_offset(n) + sizeof(double) * (size_t)finish_blocks(n) + sizeof(float) * (size_t)n; }

// Fractional bits of the importance sums: pixels * 2^bits stays below 2^63
int fraction_bits(int64_t pixels) {
    int log2 = 0;
    while (((int64_t)1 << log2) < pixels) ++log2;
    return 62 - log2;
}

struct Slots {
    int id[kTopK];  // -1: empty
    float dx[kTopK], dy[kTopK], gate[kTopK];
};

__device__ __forceinline__ void read_slots(Slots &s, const int p, const int img_w, const int n, const float2 *xys, const float *conics,
                                           const int *pixel_topk) {
    const float px = (float)(p % img_w), py = (float)(p / img_w);
    const int2 *row = reinterpret_cast<const int2 *>(pixel_topk + (size_t)p * kTopK);
    float sum = (float)igs::kNormEps;
#pragma unroll
    for (int k = 0; k < kTopK; k += 2) {
        const int2 v = __ldg(&row[k / 2]);
        s.id[k] = (unsigned)v.x < (unsigned)n ? v.x : -1, s.id[k + 1] = (unsigned)v.y < (unsigned)n ? v.y : -1;
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

__global__ void __launch_bounds__(kThreads) balance_kernel(const int pixels, const int img_w, const int n, const float2 *__restrict__ xys,
                                                           const float *__restrict__ conics, const int *__restrict__ pixel_topk,
                                                           const uint8_t *__restrict__ mask, const float scale, int *__restrict__ counts,
                                                           unsigned long long *__restrict__ fixed, BalanceWorkspace *__restrict__ ws) {
    const int p = blockIdx.x * kThreads + threadIdx.x;
    bool routed = false;
    if (p < pixels && (mask == nullptr || mask[p] != 0)) {
        Slots s;
        read_slots(s, p, img_w, n, xys, conics, pixel_topk);
#pragma unroll
        for (int k = 0; k < kTopK; ++k) {
            if (s.id[k] < 0) continue;
            routed = true;
            atomicAdd(&counts[s.id[k]], 1);
            atomicAdd(&fixed[s.id[k]], (unsigned long long)__float2ll_rn(s.gate[k] * scale));
        }
    }
    const int in_block = __syncthreads_count(routed);
    if (threadIdx.x == 0 && in_block) atomicAdd(&ws->routed, (unsigned long long)in_block);
}

// importance from the fixed-point sums, and the loss: each block's sums of counts and of counts * importance (in double, in thread order),
// the last block to finish adds them in block order
__global__ void __launch_bounds__(kThreads) balance_finish_kernel(const int n, const int *__restrict__ counts,
                                                                  const unsigned long long *__restrict__ fixed, const double inv_scale,
                                                                  float *__restrict__ importance, double *__restrict__ partials,
                                                                  BalanceWorkspace *__restrict__ ws, float *__restrict__ loss,
                                                                  long long *__restrict__ totals) {
    __shared__ double s_sum[kThreads / 32];
    __shared__ bool last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = blockIdx.x * kThreads + threadIdx.x;
    double v = 0.0;
    int c = 0;
    if (g < n) {
        const double imp = (double)(long long)fixed[g] * inv_scale;
        importance[g] = (float)imp;
        c = counts[g];
        v = imp * c;
    }
    auto block_sum = [&](double x) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        __syncthreads();
        if (lane == 0) s_sum[warp] = x;
        __syncthreads();
        double total = 0.0;
        for (int w = 0; w < kThreads / 32; ++w) total += s_sum[w];
        return total;
    };
    const double block = block_sum(v), filled = block_sum((double)c);
    if (threadIdx.x == 0) {
        partials[blockIdx.x] = block;
        atomicAdd(&ws->filled, (unsigned long long)filled);
        __threadfence();
        last = atomicAdd(&ws->ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double sum = 0.0;
    for (int b = threadIdx.x; b < (int)gridDim.x; b += kThreads) sum += __ldcg(&partials[b]);
    const double all = block_sum(sum);
    if (threadIdx.x == 0) {
        const unsigned long long a = __ldcg(&ws->filled), t = __ldcg(&ws->routed);
        *loss = a ? (float)((double)n / ((double)a * (double)t) * all) : 0.f;
        totals[0] = (long long)a, totals[1] = (long long)t;
    }
}

// alpha [n], and the gradients zeroed unless they are added to
__global__ void __launch_bounds__(kThreads) balance_alpha_kernel(const int n, const int *__restrict__ counts,
                                                                 const long long *__restrict__ totals, const float *__restrict__ v_loss,
                                                                 const float *__restrict__ v_importance, const bool zero,
                                                                 float *__restrict__ alpha, float *__restrict__ v_xy,
                                                                 float *__restrict__ v_conic) {
    const int g = blockIdx.x * kThreads + threadIdx.x;
    if (g >= n) return;
    const double a = (double)totals[0], t = (double)totals[1];
    const float scale = v_loss != nullptr && totals[0] > 0 ? (float)((double)n / (a * t)) * *v_loss : 0.f;
    alpha[g] = scale * (float)counts[g] + (v_importance != nullptr ? v_importance[g] : 0.f);
    if (zero) {
        v_xy[2 * (size_t)g] = 0.f, v_xy[2 * (size_t)g + 1] = 0.f;
#pragma unroll
        for (int j = 0; j < 3; ++j) v_conic[3 * (size_t)g + j] = 0.f;
    }
}

__global__ void __launch_bounds__(kThreads) balance_bwd_kernel(const int pixels, const int img_w, const int n, const float2 *__restrict__ xys,
                                                               const float *__restrict__ conics, const int *__restrict__ pixel_topk,
                                                               const uint8_t *__restrict__ mask, const float *__restrict__ alpha,
                                                               float *__restrict__ v_xy, float *__restrict__ v_conic) {
    const int p = blockIdx.x * kThreads + threadIdx.x;
    if (p >= pixels || (mask != nullptr && mask[p] == 0)) return;
    Slots s;
    read_slots(s, p, img_w, n, xys, conics, pixel_topk);
    float mean = 0.f;
#pragma unroll
    for (int k = 0; k < kTopK; ++k)
        if (s.id[k] >= 0) mean += s.gate[k] * __ldg(&alpha[s.id[k]]);
#pragma unroll
    for (int k = 0; k < kTopK; ++k) {
        const int g = s.id[k];
        if (s.gate[k] == 0.f) continue;  // empty, or a Gaussian whose parameters may not even be finite
        const float t = s.gate[k] * (mean - __ldg(&alpha[g]));
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

size_t igs_topk_balance_workspace(int num_points) { return num_points < 0 ? 0 : workspace_bytes_of(num_points); }

int igs_topk_balance_fwd(int img_height, int img_width, int num_points, const float *xys, const float *conics, const int32_t *pixel_topk,
                         const uint8_t *pixel_mask, float *loss, int32_t *counts, float *importance, int64_t *totals, void *workspace,
                         size_t workspace_bytes, void *stream) {
    IGS_REQUIRE(img_height >= 0 && img_width >= 0 && num_points >= 0, "igs_topk_balance_fwd: negative size");
    IGS_REQUIRE(igs::lists_addressable(img_height, img_width), "igs_topk_balance_fwd: at most 2^31 / 10 pixels and 2^24 a side");
    IGS_REQUIRE(loss && totals && (num_points == 0 || (counts && importance)), "igs_topk_balance_fwd: null output");
    IGS_REQUIRE(workspace && workspace_bytes >= workspace_bytes_of(num_points), "igs_topk_balance_fwd: workspace too small");
    IGS_REQUIRE(igs::aligned(workspace, 16), "igs_topk_balance_fwd: workspace must be 16-byte aligned");
    const int pixels = img_height * img_width;
    IGS_REQUIRE(pixels == 0 || num_points == 0 || (xys && conics && pixel_topk), "igs_topk_balance_fwd: null pointer");
    IGS_REQUIRE(igs::aligned(xys, 8) && igs::aligned(pixel_topk, 8), "igs_topk_balance_fwd: xys and pixel_topk must be 8-byte aligned");
    cudaStream_t s = igs::as_stream(stream);
    char *base = static_cast<char *>(workspace);
    BalanceWorkspace *ws = reinterpret_cast<BalanceWorkspace *>(base);
    unsigned long long *fixed = reinterpret_cast<unsigned long long *>(base + fixed_offset());
    double *partials = reinterpret_cast<double *>(base + partials_offset(num_points));
    cudaMemsetAsync(workspace, 0, partials_offset(num_points), s);
    if (num_points > 0) cudaMemsetAsync(counts, 0, sizeof(int32_t) * (size_t)num_points, s);
    const int bits = fraction_bits(pixels);
    if (pixels > 0 && num_points > 0)
        balance_kernel<<<igs::ceil_div(pixels, kThreads), kThreads, 0, s>>>(pixels, img_width, num_points,
                                                                            reinterpret_cast<const float2 *>(xys), conics, pixel_topk,
                                                                            pixel_mask, (float)((int64_t)1 << bits), counts, fixed, ws);
    balance_finish_kernel<<<finish_blocks(num_points), kThreads, 0, s>>>(
        num_points, counts, fixed, 1.0 / (double)((int64_t)1 << bits), importance, partials, ws, loss, reinterpret_cast<long long *>(totals));
    return igs::check_launch("igs_topk_balance_fwd");
}

int igs_topk_balance_bwd(int img_height, int img_width, int num_points, const float *xys, const float *conics, const int32_t *pixel_topk,
                         const uint8_t *pixel_mask, const int32_t *counts, const int64_t *totals, const float *v_loss,
                         const float *v_importance, int accumulate, float *v_xy, float *v_conic, void *workspace, size_t workspace_bytes,
                         void *stream) {
    IGS_REQUIRE(img_height >= 0 && img_width >= 0 && num_points >= 0, "igs_topk_balance_bwd: negative size");
    IGS_REQUIRE(igs::lists_addressable(img_height, img_width), "igs_topk_balance_bwd: at most 2^31 / 10 pixels and 2^24 a side");
    if (num_points == 0) return IGS_OK;
    IGS_REQUIRE(xys && conics && counts && totals && v_xy && v_conic, "igs_topk_balance_bwd: null pointer");
    IGS_REQUIRE(workspace && workspace_bytes >= workspace_bytes_of(num_points), "igs_topk_balance_bwd: workspace too small");
    IGS_REQUIRE(igs::aligned(workspace, 16), "igs_topk_balance_bwd: workspace must be 16-byte aligned");
    const int pixels = img_height * img_width;
    IGS_REQUIRE(pixels == 0 || pixel_topk, "igs_topk_balance_bwd: null pointer");
    IGS_REQUIRE(igs::aligned(xys, 8) && igs::aligned(pixel_topk, 8), "igs_topk_balance_bwd: xys and pixel_topk must be 8-byte aligned");
    cudaStream_t s = igs::as_stream(stream);
    float *alpha = reinterpret_cast<float *>(static_cast<char *>(workspace) + partials_offset(num_points) +
                                             sizeof(double) * (size_t)finish_blocks(num_points));
    balance_alpha_kernel<<<igs::ceil_div(num_points, kThreads), kThreads, 0, s>>>(
        num_points, counts, reinterpret_cast<const long long *>(totals), v_loss, v_importance, accumulate == 0, alpha, v_xy, v_conic);
    if (pixels > 0)
        balance_bwd_kernel<<<igs::ceil_div(pixels, kThreads), kThreads, 0, s>>>(pixels, img_width, num_points,
                                                                                reinterpret_cast<const float2 *>(xys), conics, pixel_topk,
                                                                                pixel_mask, alpha, v_xy, v_conic);
    return igs::check_launch("igs_topk_balance_bwd");
}

}  // extern "C"
