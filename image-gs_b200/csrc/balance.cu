// How the pixels spread over the Gaussians: the load of a top-K router whose tokens are the pixels and whose experts are the Gaussians.
// With n_pk the gates of the filled slots (topk_lists.cuh):
//   counts_g = filled slots that hold g,  importance_g = sum of their gates,  A = sum_g counts_g,  T = pixels with a filled slot
//   loss = N / (A T) sum_g counts_g importance_g     (0 when A = 0; 1 when every Gaussian has the same share and the gates sum to one)
// and, the counts held constant, with alpha_g = v_loss N counts_g / (A T) + v_importance_g:
//   dL/dsigma_k = -n_k (alpha_k - sum_j n_j alpha_j),
//   v_xy += dL/dsigma (a dx + b dy, b dx + c dy),  v_conic += dL/dsigma (dx^2 / 2, dx dy, dy^2 / 2)      (topk_sums.cuh).
//
// The importance is summed over a patch in float, in one order, and from there as 64-bit fixed point with as many fractional bits as the
// image leaves room for (a Gaussian's importance is at most the pixel count), so no result depends on the order of the atomics.
#include "topk_sums.cuh"

namespace {

using igs::kGroup;
using igs::kTile;
using igs::kTilePixels;
using igs::kTopK;
using igs::kWeightPitch;

constexpr int kThreads = 256;
using SumsOf = igs::SumLayout<1, false>;

struct BalanceWorkspace {
    unsigned long long filled;  // A
    unsigned long long routed;  // T
    unsigned int ticket;
    float scale;                // backward: v_loss N / (A T)
    unsigned int pad[10];
    // forward: then uint64 fixed [n] and double partials [blocks of the finish kernel]; backward: then float sums [n, SumsOf::kValues]
};

int finish_blocks(int n) { return n > 0 ? igs::ceil_div(n, kThreads) : 1; }
size_t forward_bytes(int n) { return sizeof(BalanceWorkspace) + sizeof(unsigned long long) * (size_t)n + sizeof(double) * (size_t)finish_blocks(n); }
size_t backward_bytes(int n) { return sizeof(BalanceWorkspace) + sizeof(float) * SumsOf::kValues * (size_t)n; }
size_t workspace_bytes_of(int n) { return forward_bytes(n) > backward_bytes(n) ? forward_bytes(n) : backward_bytes(n); }

// Fractional bits of the importance sums: pixels * 2^bits stays below 2^63
int fraction_bits(int64_t pixels) {
    int log2 = 0;
    while (((int64_t)1 << log2) < pixels) ++log2;
    return 62 - log2;
}

__global__ void __launch_bounds__(kThreads) balance_zero_kernel(const int n, int *__restrict__ counts, unsigned long long *__restrict__ fixed,
                                                                BalanceWorkspace *__restrict__ ws) {
    igs::wait_for_predecessor();
    const int g = blockIdx.x * kThreads + threadIdx.x;
    if (g == 0) ws->filled = 0, ws->routed = 0, ws->ticket = 0;
    if (g < n) counts[g] = 0, fixed[g] = 0;
}

struct BalanceSmem {
    igs::TileTable table;
    union {
        alignas(16) int lists[igs::kListWords];
        struct {
            alignas(16) float weight[igs::kWarps][kGroup * kWeightPitch];
            alignas(16) float inv[igs::kWarps][32];
        };
    };
    float4 rows[igs::kMaxRows * igs::Rows<0>::kRowQuads];
    float4 group[igs::kWarps][igs::Rows<0>::kGroupQuads];
};

struct BalanceArgs {
    int tiles_x, img_h, img_w, n;
    const float *xys, *conics;
    const int *pixel_topk;
    const uint8_t *mask;
    float scale;  // 2^fraction bits
    int *counts;
    unsigned long long *fixed;
    BalanceWorkspace *ws;
};

// One pixel's slots one by one, from global memory (topk_sums.cuh says when)
__device__ __noinline__ void count_slots(const BalanceArgs &a, const int p) {
    const float px = (float)(p % a.img_w), py = (float)(p / a.img_w);
    const int *list = a.pixel_topk + (size_t)p * kTopK;
    float total = (float)igs::kNormEps;
    for (int pass = 0; pass < 2; ++pass) {
        const float inv = 1.f / total;
        for (int k = 0; k < kTopK; ++k) {
            const int id = list[k];
            if ((unsigned)id >= (unsigned)a.n) continue;
            const float w = igs::slot_weight(igs::stage_geometry(a.xys, a.conics, id), px, py);
            if (pass == 0) {
                total += w;
            } else {
                atomicAdd(&a.counts[id], 1);
                atomicAdd(&a.fixed[id], (unsigned long long)__float2ll_rn(w * inv * a.scale));
            }
        }
    }
}

__global__ void __launch_bounds__(kTilePixels, 5) balance_kernel(const __grid_constant__ BalanceArgs a) {
    using Rows = igs::Rows<0>;
    __shared__ __align__(16) BalanceSmem sm;
    igs::wait_for_predecessor();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int i0 = (blockIdx.x / a.tiles_x) * kTile, j0 = (blockIdx.x % a.tiles_x) * kTile;
    const int i = i0 + igs::patch_y(), j = j0 + igs::patch_x();
    const bool inside = i < a.img_h && j < a.img_w;
    const int p = inside ? i * a.img_w + j : 0;
    igs::load_lists(sm.lists, sm.table, a.pixel_topk, i0, j0, a.img_h, a.img_w);
    const unsigned keep = inside && (a.mask == nullptr || a.mask[p] != 0) ? ~0u : 0u;
    igs::seed_table(sm.table, sm.lists, i0, j0, a.img_h, a.img_w, a.n);
    igs::PixelSlots s;
    igs::place_slots(s, sm.table, sm.lists, a.n, keep);
    const int routed = __syncthreads_count(s.filled > 0);
    if (threadIdx.x == 0 && routed > 0) atomicAdd(&a.ws->routed, (unsigned long long)routed);
    const int count = sm.table.count;
    if (count > igs::kMaxRows) {
        if (keep) count_slots(a, p);
        return;
    }
    igs::rank_rows(sm.table, count, [&](const int row, const int id) {
        const igs::RowGeometry g = igs::stage_geometry(a.xys, a.conics, id);
        sm.rows[2 * row] = make_float4(g.x, g.y, g.a, g.b), sm.rows[2 * row + 1] = make_float4(g.c, 0.f, 0.f, 0.f);
    });
    __syncthreads();
    if (!__all_sync(0xffffffffu, igs::find_rows(s, sm.table, count))) {
        if (keep) count_slots(a, p);
        return;
    }
    // a lane is a pixel: the first group's weights and the sum over all (topk_sums.cuh). The sign of a weight says whether the slot is
    // there: -0 for an absent one (which adds nothing either), so that counts come from the same words as the sums.
    float *const weight = sm.weight[warp];
    float4 *const group = sm.group[warp];
    const float2 minus_x = make_float2(-(float)j, -(float)j), minus_y = make_float2(-(float)i, -(float)i);
    const int half = lane >> 4, r = lane & (kGroup - 1);
    float2 total = make_float2(0.f, 0.f);
    int my_row = 0, my_rows = 0;
    auto weigh = [&](const int first, const unsigned bits, const int begin, const int n, const bool keep_weights) {
        const int row = Rows::gather(sm.rows, sm.table.order[warp], begin, n, first, group).row;
        if (keep_weights) my_row = row, my_rows = min(n - begin, kGroup);
        __syncwarp();
        for (int pair = 0; 2 * pair < min(n - begin, kGroup); ++pair) {
            const float4 *q = group + pair * Rows::kPairQuads;
            const float2 w = Rows::weights(q, bits, minus_x, minus_y);
            total = igs::add2(total, w);
            if (keep_weights) {
                weight[2 * pair * kWeightPitch + lane] = (bits & __float_as_uint(q[2].z)) != 0 ? w.x : -0.f;
                weight[(2 * pair + 1) * kWeightPitch + lane] = (bits & __float_as_uint(q[2].w)) != 0 ? w.y : -0.f;
            }
        }
        __syncwarp();
    };
    // a lane is half a row: its gates' sum and its holders
    auto sum_rows = [&]() {
        float sum = 0.f;
        int absent = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 w = *reinterpret_cast<const float4 *>(&weight[r * kWeightPitch + half * 16 + q * 4]);
            const float4 inv = *reinterpret_cast<const float4 *>(&sm.inv[warp][half * 16 + q * 4]);
            sum = fmaf(w.x, inv.x, fmaf(w.y, inv.y, fmaf(w.z, inv.z, fmaf(w.w, inv.w, sum))));
            absent += (int)((__float_as_uint(w.x) >> 31) + (__float_as_uint(w.y) >> 31) + (__float_as_uint(w.z) >> 31) +
                            (__float_as_uint(w.w) >> 31));
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        absent += __shfl_xor_sync(0xffffffffu, absent, 16);
        if (r < my_rows) {
            const int id = sm.table.sorted[my_row];
            if (half == 0) atomicAdd(&a.counts[id], 32 - absent);
            else atomicAdd(&a.fixed[id], (unsigned long long)__float2ll_rn(sum * a.scale));
        }
        __syncwarp();
    };
    const int groups = igs::visit_groups(
        s, sm.table, count,
        [&](const int at, const int first, const unsigned bits, const int begin, const int n) { weigh(first, bits, begin, n, at == 0); });
    sm.inv[warp][lane] = 1.f / (total.x + total.y + (float)igs::kNormEps);
    __syncwarp();
    if (groups > 0) sum_rows();
    if (groups > 1)
        igs::visit_groups(s, sm.table, count, [&](const int at, const int first, const unsigned bits, const int begin, const int n) {
            if (at == 0) return;
            weigh(first, bits, begin, n, true);
            sum_rows();
        });
}

// importance from the fixed-point sums, and the loss: each block's sums of counts and of counts * importance (in double, in thread order),
// the last block to finish adds them in block order
__global__ void __launch_bounds__(kThreads) balance_finish_kernel(const int n, const int *__restrict__ counts,
                                                                  const unsigned long long *__restrict__ fixed, const double inv_scale,
                                                                  float *__restrict__ importance, double *__restrict__ partials,
                                                                  BalanceWorkspace *__restrict__ ws, float *__restrict__ loss,
                                                                  long long *__restrict__ totals) {
    igs::wait_for_predecessor();
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

// The backward pass's sums zeroed, and the loss's share of alpha: v_loss N / (A T)
__global__ void __launch_bounds__(kThreads) balance_scale_kernel(const int n, const long long *__restrict__ totals,
                                                                 const float *__restrict__ v_loss, float4 *__restrict__ sums,
                                                                 BalanceWorkspace *__restrict__ ws) {
    igs::wait_for_predecessor();
    const int e = blockIdx.x * kThreads + threadIdx.x;
    if (e == 0)
        ws->scale = v_loss != nullptr && totals[0] > 0 ? (float)((double)n / ((double)totals[0] * (double)totals[1])) * *v_loss : 0.f;
    if (e < n * (SumsOf::kValues / 4)) sums[e] = make_float4(0.f, 0.f, 0.f, 0.f);
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
    IGS_REQUIRE(pixels == 0 || num_points == 0 || (xys && conics && pixel_topk), "igs_topk_balance_fwd: null pointer");
    IGS_REQUIRE(igs::aligned(pixel_topk, 8), "igs_topk_balance_fwd: pixel_topk must be 8-byte aligned");
    cudaStream_t s = igs::as_stream(stream);
    char *base = static_cast<char *>(workspace);
    BalanceWorkspace *ws = reinterpret_cast<BalanceWorkspace *>(base);
    unsigned long long *fixed = reinterpret_cast<unsigned long long *>(base + sizeof(BalanceWorkspace));
    double *partials = reinterpret_cast<double *>(fixed + num_points);
    const int bits = fraction_bits(pixels);
    const int blocks = finish_blocks(num_points);
    igs::launch(balance_zero_kernel, dim3(blocks), dim3(kThreads), 0, s, num_points, counts, fixed, ws);
    if (pixels > 0 && num_points > 0) {
        const int tiles_x = igs::ceil_div(img_width, kTile), tiles_y = igs::ceil_div(img_height, kTile);
        const BalanceArgs a = {tiles_x, img_height, img_width, num_points, xys, conics, pixel_topk, pixel_mask,
                               (float)((int64_t)1 << bits), counts, fixed, ws};
        igs::launch(balance_kernel, dim3(tiles_x * tiles_y), dim3(kTilePixels), 0, s, a);
    }
    igs::launch(balance_finish_kernel, dim3(blocks), dim3(kThreads), 0, s, num_points, (const int *)counts,
                (const unsigned long long *)fixed, 1.0 / (double)((int64_t)1 << bits), importance, partials, ws, loss,
                reinterpret_cast<long long *>(totals));
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
    BalanceWorkspace *ws = reinterpret_cast<BalanceWorkspace *>(workspace);
    float *sums = reinterpret_cast<float *>(ws + 1);
    igs::launch(balance_scale_kernel, dim3(igs::ceil_div(num_points * (SumsOf::kValues / 4), kThreads)), dim3(kThreads), 0, s, num_points,
                reinterpret_cast<const long long *>(totals), v_loss, reinterpret_cast<float4 *>(sums), ws);
    if (pixels > 0) {
        igs::SumArgs a = {};
        a.tiles_x = igs::ceil_div(img_width, kTile), a.img_h = img_height, a.img_w = img_width, a.n = num_points;
        a.xys = xys, a.conics = conics, a.pixel_topk = pixel_topk, a.mask = pixel_mask;
        a.counts = counts, a.scale = &ws->scale, a.v_importance = v_importance, a.sums = sums;
        igs::launch_sums<1, false>(a, s);
    }
    igs::launch(igs::finish_sums_kernel<SumsOf::kValues>, dim3(igs::ceil_div(num_points, 256)), dim3(256), 0, s, num_points, 0, conics,
                (const float *)sums, accumulate != 0, v_xy, v_conic, (float *)nullptr);
    return igs::check_launch("igs_topk_balance_bwd");
}

}  // extern "C"
