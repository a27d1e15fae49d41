// How the pixels spread over the Gaussians: the load of a top-K router whose tokens are the pixels and whose experts are the Gaussians.
// With n_pk the gates of the filled slots (topk_lists.cuh):
//   counts_g = filled slots that hold g,  importance_g = sum of their gates,  A = sum_g counts_g,  T = pixels with a filled slot
//   loss = N / (A T) sum_g counts_g importance_g     (0 when A = 0; 1 when every Gaussian has the same share and the gates sum to one)
// and, the counts held constant, with alpha_g = v_loss N counts_g / (A T) + v_importance_g:
//   dL/dsigma_k = -n_k (alpha_k - sum_j n_j alpha_j),
//   v_xy += dL/dsigma (a dx + b dy, b dx + c dy),  v_conic += dL/dsigma (dx^2 / 2, dx dy, dy^2 / 2)      (topk_sums.cuh).
//
// The importance is summed over a patch in float, in one order, and from there as 64-bit fixed point with as many fractional bits as the
// image leaves room for (a Gaussian's importance is at most the pixel count), so no result depends on the order of the atomics. The float sums
// of at most 64 gates round by 2^-24 of themselves (the results are within 1e-7 of the definition's in 64 bits, where sums in 64 bits
// throughout are within 0.5e-7); the fixed point rounds a patch's share to 2^-(62 - ceil(log2 pixels)), 2^-39 at 3840x2160, and half of that
// to 0.
//
// At 1920x1080 with 20,000 Gaussians the counts, importance and loss take 54 us and the gradient 59 us (the lists at the memory's rate 13 us
// each); what bounds them stands in topk_lists.cuh.
#include <algorithm>

#include "topk_sums.cuh"

namespace {

using igs::kPatchPixels;
using igs::kPix;
using igs::kWeightPitch;
using Rows = igs::Rows<0>;

constexpr int kThreads = 256;
constexpr int kRoutedSlots = 32;

struct BalanceWorkspace {
    unsigned int ticket;
    unsigned int pad[3];
    unsigned long long routed[kRoutedSlots];  // T, over this many words, so that no one word takes every patch's atomic
    // then uint64 fixed [n], double2 partials [blocks of the finish kernel]
};

int finish_blocks(int n) { return n > 0 ? igs::ceil_div(n, kThreads) : 1; }
size_t forward_bytes(int n) {
    return sizeof(BalanceWorkspace) + sizeof(unsigned long long) * (size_t)(n + 1) + sizeof(double2) * (size_t)finish_blocks(n);
}
size_t workspace_bytes_of(int n) { return std::max(forward_bytes(n), igs::sum_bytes<1, false>(n)); }

// Fractional bits of the importance sums: pixels * 2^bits stays below 2^63
int fraction_bits(int64_t pixels) {
    int log2 = 0;
    while (((int64_t)1 << log2) < pixels) ++log2;
    return 62 - log2;
}

struct BalanceArgs {
    int img_h, img_w, n;
    const float *xys, *conics;
    const int *pixel_topk;
    const uint8_t *mask;
    float scale;  // 2^fraction bits
    int *counts;
    unsigned long long *fixed;
    BalanceWorkspace *ws;
    double inv_scale;
    float *importance;
    double2 *partials;  // A and the loss's sum, of each block of the finish kernel
    float *loss;
    long long *totals;
};

__global__ void __launch_bounds__(kThreads) balance_zero_kernel(const __grid_constant__ BalanceArgs a) {
    igs::wait_for_predecessor();
    const int id = blockIdx.x * kThreads + threadIdx.x;
    if (id == 0) a.ws->ticket = 0;
    if (id < kRoutedSlots) a.ws->routed[id] = 0;
    if (id < a.n) a.counts[id] = 0, a.fixed[id] = 0;
}

// One pixel's slots one by one, from global memory (topk_sums.cuh says when)
__device__ __forceinline__ void count_pixel_slots(const BalanceArgs &a, const int p) {
    if (a.mask != nullptr && a.mask[p] == 0) return;
    const float px = (float)(p % a.img_w), py = (float)(p / a.img_w);
    const int *list = a.pixel_topk + (size_t)p * igs::kTopK;
    float total = (float)igs::kNormEps;
    for (int pass = 0; pass < 2; ++pass) {
        const float inv = igs::reciprocal(total);
        for (int k = 0; k < igs::kTopK; ++k) {
            const int id = list[k];
            if ((unsigned)id >= (unsigned)a.n) continue;
            const float w = igs::slot_weight(igs::row_geometry(a.xys, a.conics, id), px, py);
            if (pass == 0) {
                total += w;
            } else {
                atomicAdd(&a.counts[id], 1);
                atomicAdd(&a.fixed[id], (unsigned long long)__float2ll_rn(w * inv * a.scale));
            }
        }
    }
}

__device__ __noinline__ void count_slots(const BalanceArgs &a) {
    const igs::Patch patch(a.img_h, a.img_w);  // (made again: passed from the caller, it would live in the caller's local memory)
#pragma unroll
    for (int b = 0; b < kPix; ++b)
        if (patch.inside[b]) count_pixel_slots(a, patch.p[b]);
}

struct BalanceSmem {
    union {
        int keys[igs::kKeyWords];
        alignas(16) float weight[igs::kRows * kWeightPitch];
    };
    float4 pairs[Rows::kGroupQuads];
    alignas(16) float inv[kPatchPixels];
};

__device__ __forceinline__ igs::PatchRows balance_rows(const BalanceArgs &a, const igs::Patch &patch, const int g, int *keys) {
    return igs::find_rows(
        a.pixel_topk, patch, a.n,
        [&](const int p, const bool inside) { return igs::AllSlots{inside && (a.mask == nullptr || a.mask[p] != 0)}; }, g, keys);
}

// A lane is its pixels: the group's weights into shared memory, and into the pixels' sums
__device__ __forceinline__ void weigh_rows(const igs::PatchRows &rows, const igs::Patch &patch, BalanceSmem &sm, float2 (&total)[kPix]) {
    const float2 minus_x = make_float2(-(float)patch.j, -(float)patch.j);
    float2 minus_y[kPix];
    unsigned held[kPix];
#pragma unroll
    for (int b = 0; b < kPix; ++b) minus_y[b] = make_float2(-(float)patch.i[b], -(float)patch.i[b]), held[b] = rows.bits[b];
    const float4 *pairs = sm.pairs;
    float *weight = sm.weight + (threadIdx.x & 31);
#pragma unroll 2
    for (int pair = 0; 2 * pair < rows.n; ++pair, pairs += Rows::kPairQuads, weight += 2 * kWeightPitch) {
        float2 w[kPix];
        Rows::weights(pairs, held, minus_x, minus_y, w);
#pragma unroll
        for (int b = 0; b < kPix; ++b) {
            held[b] >>= 2;
            weight[32 * b] = w[b].x, weight[kWeightPitch + 32 * b] = w[b].y;
            total[b] = igs::add2(total[b], w[b]);
        }
    }
}

__device__ __forceinline__ void invert_totals(BalanceSmem &sm, const float2 (&total)[kPix]) {
#pragma unroll
    for (int b = 0; b < kPix; ++b)
        sm.inv[32 * b + (threadIdx.x & 31)] = igs::reciprocal(total[b].x + total[b].y + (float)igs::kNormEps);
}

// A lane is a row or, up to 16 rows, half of one (as in topk_sums.cuh): its gates' sum and its holders
__device__ __forceinline__ void count_rows(const BalanceArgs &a, const igs::PatchRows &rows, const BalanceSmem &sm) {
    const int lane = threadIdx.x & 31;
    const bool halves = rows.n <= 16;
    const int r = halves ? lane & 15 : min(lane, igs::kRows - 1), half = halves ? lane >> 4 : 0;
    const float *w_at = sm.weight + r * kWeightPitch + half * (kPatchPixels / 2), *inv_at = sm.inv + half * (kPatchPixels / 2);
    float sum = 0.f;
#pragma unroll 4
    for (int q = 0; q < (halves ? kPatchPixels / 8 : kPatchPixels / 4); ++q, w_at += 4, inv_at += 4) {
        const float4 w = *reinterpret_cast<const float4 *>(w_at);
        const float4 inv = *reinterpret_cast<const float4 *>(inv_at);
        sum = fmaf(w.x, inv.x, fmaf(w.y, inv.y, fmaf(w.z, inv.z, fmaf(w.w, inv.w, sum))));
    }
    const int id = __shfl_sync(0xffffffffu, rows.id, r);
    if (halves) sum += __shfl_xor_sync(0xffffffffu, sum, 16);
    if (half == 0 && (halves ? r : lane) < rows.n) atomicAdd(&a.fixed[id], (unsigned long long)__float2ll_rn(sum * a.scale));
    if (lane < rows.n) atomicAdd(&a.counts[rows.id], rows.holders);
}

// A patch of more rows than a group: all groups for the pixels' sums, then all again for the rows'
__device__ __noinline__ bool count_groups(const BalanceArgs &a, BalanceSmem &sm) {
    const igs::Patch patch(a.img_h, a.img_w);
    float2 total[kPix] = {};
    for (int pass = 0; pass < 2; ++pass) {
        bool more = true;
        for (int g = 0; more; ++g) {
            const igs::PatchRows rows = balance_rows(a, patch, g, sm.keys);
            more = rows.more;
            if (!Rows::gather(rows, a.xys, a.conics, [](int, int) { return 0.f; }, sm.pairs)) return false;
            __syncwarp();
            weigh_rows(rows, patch, sm, total);
            __syncwarp();
            if (pass == 1) count_rows(a, rows, sm);
        }
        if (pass == 0) invert_totals(sm, total);
        __syncwarp();
    }
    return true;
}

// A warp is a patch
__device__ __forceinline__ void count_patch(const BalanceArgs &a, BalanceSmem &sm) {
    const igs::Patch patch(a.img_h, a.img_w);
    if (patch.x0 >= a.img_w || patch.y0 >= a.img_h) return;
    const igs::PatchRows rows = balance_rows(a, patch, 0, sm.keys);
    const unsigned routed = __reduce_add_sync(0xffffffffu, (unsigned)rows.filled);
    if ((threadIdx.x & 31) == 0 && routed > 0)
        atomicAdd(&a.ws->routed[(blockIdx.x + blockIdx.y) % kRoutedSlots], (unsigned long long)routed);
    bool regular;
    if (rows.more) {
        regular = count_groups(a, sm);
    } else {
        regular = Rows::gather(rows, a.xys, a.conics, [](int, int) { return 0.f; }, sm.pairs);
        __syncwarp();
        float2 total[kPix] = {};
        weigh_rows(rows, patch, sm, total);
        invert_totals(sm, total);
        __syncwarp();
        if (regular) count_rows(a, rows, sm);
    }
    if (!regular) count_slots(a);
}

// The sums over the CTA, in one order, on all threads; s_sum: a double2 per warp
template <int kCta>
__device__ __forceinline__ double2 cta_sum(double2 v, double2 *s_sum) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v.x += __shfl_xor_sync(0xffffffffu, v.x, o), v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    v = make_double2(0.0, 0.0);
#pragma unroll
    for (int w = 0; w < kCta / 32; ++w) v.x += s_sum[w].x, v.y += s_sum[w].y;
    return v;
}

// A Gaussian's importance, from its fixed-point sum; its counts and its term of the loss are added to v
__device__ __forceinline__ void finish_gaussian(const BalanceArgs &a, const int g, double2 &v) {
    const double importance = (double)(long long)__ldcg(&a.fixed[g]) * a.inv_scale;
    a.importance[g] = (float)importance;
    const int count = __ldcg(&a.counts[g]);
    v.x += count, v.y += importance * count;
}

// By one warp
__device__ __forceinline__ void finish_loss(const BalanceArgs &a, const double2 v) {
    static_assert(kRoutedSlots == 32, "a word per lane");
    const int lane = threadIdx.x & 31;
    unsigned long long routed = __ldcg(&a.ws->routed[lane]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) routed += __shfl_xor_sync(0xffffffffu, routed, o);
    if (lane != 0) return;
    *a.loss = v.x > 0.0 ? (float)((double)a.n / (v.x * (double)routed) * v.y) : 0.f;
    a.totals[0] = (long long)v.x, a.totals[1] = (long long)routed;
}

// kFinish: the last CTA finishes
template <bool kFinish>
__global__ void __launch_bounds__(igs::kPatchThreads, 6) balance_kernel(const __grid_constant__ BalanceArgs a) {
    __shared__ BalanceSmem smem[igs::kPatches];
    igs::wait_for_predecessor();
    count_patch(a, smem[threadIdx.x >> 5]);
    if constexpr (kFinish) {
        if (!igs::last_cta(&a.ws->ticket)) return;
        double2 v = make_double2(0.0, 0.0);
        for (int g = threadIdx.x; g < a.n; g += igs::kPatchThreads) finish_gaussian(a, g, v);
        v = cta_sum<igs::kPatchThreads>(v, reinterpret_cast<double2 *>(smem));
        if (threadIdx.x < 32) finish_loss(a, v);
    }
}

// Each block's sums, added in block order by the last block to finish
__global__ void __launch_bounds__(kThreads) balance_finish_kernel(const __grid_constant__ BalanceArgs a) {
    igs::wait_for_predecessor();
    __shared__ double2 s_sum[kThreads / 32];
    const int g = blockIdx.x * kThreads + threadIdx.x;
    double2 v = make_double2(0.0, 0.0);
    if (g < a.n) finish_gaussian(a, g, v);
    v = cta_sum<kThreads>(v, s_sum);
    if (threadIdx.x == 0) a.partials[blockIdx.x] = v;
    if (!igs::last_cta(&a.ws->ticket)) return;
    v = make_double2(0.0, 0.0);
    for (int b = threadIdx.x; b < (int)gridDim.x; b += kThreads) {
        const double2 q = __ldcg(&a.partials[b]);
        v.x += q.x, v.y += q.y;
    }
    v = cta_sum<kThreads>(v, s_sum);
    if (threadIdx.x < 32) finish_loss(a, v);
}

}  // namespace

extern "C" {

size_t igs_topk_balance_workspace(int num_points) { return num_points < 0 ? 0 : workspace_bytes_of(num_points); }

int igs_topk_balance_fwd(int img_height, int img_width, int num_points, const float *xys, const float *conics, const int32_t *pixel_topk,
                         const uint8_t *pixel_mask, float *loss, int32_t *counts, float *importance, int64_t *totals, void *workspace,
                         size_t workspace_bytes, void *stream) {
    IGS_REQUIRE(img_height >= 0 && img_width >= 0 && num_points >= 0, "igs_topk_balance_fwd: negative size");
    IGS_REQUIRE(igs::lists_addressable(img_height, img_width, num_points), "igs_topk_balance_fwd: %s", igs::kListsLimit);
    IGS_REQUIRE(loss && totals && (num_points == 0 || (counts && importance)), "igs_topk_balance_fwd: null output");
    IGS_REQUIRE(workspace && workspace_bytes >= workspace_bytes_of(num_points), "igs_topk_balance_fwd: workspace too small");
    IGS_REQUIRE(igs::aligned(workspace, 16), "igs_topk_balance_fwd: workspace must be 16-byte aligned");
    const int pixels = img_height * img_width;
    IGS_REQUIRE(num_points == 0 || (xys && conics && (pixels == 0 || pixel_topk)), "igs_topk_balance_fwd: null pointer");
    IGS_REQUIRE(igs::aligned(pixel_topk, 8), "igs_topk_balance_fwd: pixel_topk must be 8-byte aligned");
    cudaStream_t s = igs::as_stream(stream);
    char *base = static_cast<char *>(workspace);
    BalanceWorkspace *ws = reinterpret_cast<BalanceWorkspace *>(base);
    unsigned long long *fixed = reinterpret_cast<unsigned long long *>(base + sizeof(BalanceWorkspace));
    double2 *partials = reinterpret_cast<double2 *>(fixed + (num_points + 1) / 2 * 2);  // 16-byte aligned
    const int bits = fraction_bits(pixels);
    const int blocks = finish_blocks(num_points);
    const bool patches = pixels > 0 && num_points > 0, in_last = patches && num_points <= igs::kFinishInLast;
    const BalanceArgs a = {img_height, img_width, num_points, xys, conics, pixel_topk, pixel_mask, (float)((int64_t)1 << bits), counts,
                           fixed, ws, 1.0 / (double)((int64_t)1 << bits), importance, partials, loss,
                           reinterpret_cast<long long *>(totals)};
    igs::launch(balance_zero_kernel, dim3(blocks), dim3(kThreads), 0, s, a);
    if (patches)
        igs::launch(in_last ? balance_kernel<true> : balance_kernel<false>, igs::tile_grid(img_height, img_width), dim3(igs::kPatchThreads),
                    0, s, a);
    if (!in_last) igs::launch(balance_finish_kernel, dim3(blocks), dim3(kThreads), 0, s, a);
    return igs::check_launch("igs_topk_balance_fwd");
}

int igs_topk_balance_bwd(int img_height, int img_width, int num_points, const float *xys, const float *conics, const int32_t *pixel_topk,
                         const uint8_t *pixel_mask, const int32_t *counts, const int64_t *totals, const float *v_loss,
                         const float *v_importance, int accumulate, float *v_xy, float *v_conic, void *workspace, size_t workspace_bytes,
                         void *stream) {
    IGS_REQUIRE(img_height >= 0 && img_width >= 0 && num_points >= 0, "igs_topk_balance_bwd: negative size");
    IGS_REQUIRE(igs::lists_addressable(img_height, img_width, num_points), "igs_topk_balance_bwd: %s", igs::kListsLimit);
    if (num_points == 0) return IGS_OK;
    IGS_REQUIRE(xys && conics && counts && totals && v_xy && v_conic, "igs_topk_balance_bwd: null pointer");
    IGS_REQUIRE(workspace && workspace_bytes >= workspace_bytes_of(num_points), "igs_topk_balance_bwd: workspace too small");
    IGS_REQUIRE(igs::aligned(workspace, 16), "igs_topk_balance_bwd: workspace must be 16-byte aligned");
    const int pixels = img_height * img_width;
    IGS_REQUIRE(pixels == 0 || pixel_topk, "igs_topk_balance_bwd: null pointer");
    IGS_REQUIRE(igs::aligned(pixel_topk, 8), "igs_topk_balance_bwd: pixel_topk must be 8-byte aligned");
    cudaStream_t s = igs::as_stream(stream);
    igs::SumArgs a = {};
    a.img_h = img_height, a.img_w = img_width, a.n = num_points;
    a.xys = xys, a.conics = conics, a.pixel_topk = pixel_topk, a.mask = pixel_mask;
    a.counts = counts, a.totals = reinterpret_cast<const long long *>(totals), a.v_loss = v_loss, a.v_importance = v_importance;
    a.accumulate = accumulate != 0, a.v_xy = v_xy, a.v_conic = v_conic;
    igs::launch_sums<1, false>(a, workspace, s);
    return igs::check_launch("igs_topk_balance_bwd");
}

}  // extern "C"
