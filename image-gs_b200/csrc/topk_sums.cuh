// The backward pass shared by the balance loss and the gate dropout: sums over pixels, per Gaussian, of products of its weight with values
// of the pixel. Both losses reach the gates n_k = w_k / D, D = eps + sum_j w_j, through a score that is linear in the row's values f_c and
// the pixel's values v_c, s_k = sum_c f_c v_c (dropout: the colour and v_out; balance: one value, alpha, and v = 1). With
//   v'_c = v_c / D,  m' = sum_j w_j s_j / D^2,  t = dL/dsigma = w (m' - sum_c f_c v'_c)
// a Gaussian's sums are sum t dx, t dy, t dx^2, t dx dy, t dy^2 and (dropout) w v'_c, from which finish_kernel forms
//   v_xy = (a Sx + b Sy, b Sx + c Sy),  v_conic = (Sxx / 2, Sxy, Syy / 2),  v_f = S_c.
//
// A warp (an 8x4 patch, topk_lists.cuh) goes over its rows twice. First a lane is a pixel: weights into shared memory (16 rows of 32), D
// and the scores' sum in registers. Then a lane is half a row: lane l sums row l % 16 over 16 pixels (two patch rows of 8), reading the
// weights four at a time and the pixels' v' and m' as broadcasts, two pixels per packed instruction; dy is one value per patch row, so t
// and t dx are summed along it first. One shuffle joins the halves, and the sums go to global memory with one 16-byte vector atomic per
// four values. A patch of more than 16 rows computes the later groups' weights again. A tile with an ID twice in a list, too many IDs or
// values that are not finite takes the per-slot path instead: zero times a value that is not finite would reach Gaussians that the pixel
// does not name.
#pragma once

#include "topk_lists.cuh"

namespace igs {

constexpr int kWeightPitch = 36;  // words: the reads of four pixels by eight lanes (rows) fall on distinct banks

struct SumArgs {
    int tiles_x, img_h, img_w, channels, n;
    const float *xys, *conics;
    const int *pixel_topk;
    const uint8_t *mask;         // balance: pixels that count (NULL: all)
    const int *counts;           // balance: alpha = *scale * counts + v_importance
    const float *scale, *v_importance;
    const float *colors, *v_output;  // dropout
    const long long *rng;
    uint32_t threshold;
    float *sums;                 // [N, SumLayout::kValues], zero before
};

// C: the values per row and pixel (1 for balance; 3, 7, 11 or 12 channels, the unused ones zero)
template <int C, bool kDropout>
struct SumLayout {
    static constexpr int kValues = ((5 + (kDropout ? C : 0)) + 3) / 4 * 4;  // Sx, Sy, Sxx, Sxy, Syy, S_c
};

template <int C, bool kDropout>
struct SumSmem {
    TileTable table;
    union {
        alignas(16) int lists[kListWords];
        struct {
            alignas(16) float weight[kWarps][kGroup * kWeightPitch];
            alignas(16) float pixel[kWarps][C + 1][32];  // v'_c, m'
        };
    };
    float4 rows[kMaxRows * Rows<C>::kRowQuads];
    float4 group[kWarps][Rows<C>::kGroupQuads];
};

// Value c of a Gaussian's score
template <bool kDropout>
__device__ __forceinline__ float row_value(const SumArgs &a, const int id, const int c) {
    if constexpr (kDropout) return c < a.channels ? __ldg(&a.colors[(size_t)id * a.channels + c]) : 0.f;
    return *a.scale * (float)__ldg(&a.counts[id]) + (a.v_importance != nullptr ? __ldg(&a.v_importance[id]) : 0.f);
}
template <bool kDropout>
__device__ __forceinline__ float pixel_value(const SumArgs &a, const int p, const int c) {
    if constexpr (kDropout) return c < a.channels ? __ldg(&a.v_output[(size_t)c * (a.img_h * a.img_w) + p]) : 0.f;
    return 1.f;
}

// One pixel's slots one by one, from global memory: a slot of weight 0 adds nothing
template <int C, bool kDropout>
__device__ __noinline__ void add_slots(const SumArgs &a, const int p, const unsigned keep) {
    constexpr int kValues = SumLayout<C, kDropout>::kValues;
    const float px = (float)(p % a.img_w), py = (float)(p / a.img_w);
    const int *list = a.pixel_topk + (size_t)p * kTopK;
    float total = (float)kNormEps, scores = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
        const float inv = 1.f / total, m = scores * inv * inv;
        for (int k = 0; k < kTopK; ++k) {
            const int id = list[k];
            if ((unsigned)id >= (unsigned)a.n || !(keep >> k & 1)) continue;
            const RowGeometry g = stage_geometry(a.xys, a.conics, id);
            const float w = slot_weight(g, px, py);
            if (w == 0.f) continue;
            float score = 0.f;
            for (int c = 0; c < (kDropout ? a.channels : 1); ++c) score += row_value<kDropout>(a, id, c) * pixel_value<kDropout>(a, p, c);
            if (pass == 0) {
                total += w, scores += w * score;
                continue;
            }
            float *s = a.sums + (size_t)id * kValues;
            const float dx = g.x - px, dy = g.y - py, t = w * (m - score * inv);
            atomicAdd(&s[0], t * dx), atomicAdd(&s[1], t * dy);
            atomicAdd(&s[2], t * dx * dx), atomicAdd(&s[3], t * dx * dy), atomicAdd(&s[4], t * dy * dy);
            if constexpr (kDropout)
                for (int c = 0; c < a.channels; ++c) atomicAdd(&s[5 + c], w * inv * pixel_value<kDropout>(a, p, c));
        }
    }
}

template <int C, bool kDropout>
__global__ void __launch_bounds__(kTilePixels, C <= 3 ? 4 : 3) sums_kernel(const __grid_constant__ SumArgs a) {
    constexpr int kValues = SumLayout<C, kDropout>::kValues;
    constexpr int kRowQuads = Rows<C>::kRowQuads, kPairQuads = Rows<C>::kPairQuads;
    extern __shared__ __align__(16) char smem_bytes[];
    SumSmem<C, kDropout> &sm = *reinterpret_cast<SumSmem<C, kDropout> *>(smem_bytes);
    wait_for_predecessor();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int i0 = (blockIdx.x / a.tiles_x) * kTile, j0 = (blockIdx.x % a.tiles_x) * kTile;
    const int i = i0 + patch_y(), j = j0 + patch_x();
    const bool inside = i < a.img_h && j < a.img_w;
    const int p = inside ? i * a.img_w + j : 0;
    load_lists(sm.lists, sm.table, a.pixel_topk, i0, j0, a.img_h, a.img_w);
    unsigned keep = 0;
    if (inside) {
        if constexpr (kDropout) keep = keep_bits((uint32_t)p, (uint64_t)a.rng[0], (uint64_t)a.rng[1], a.threshold);
        else keep = a.mask == nullptr || a.mask[p] != 0 ? ~0u : 0u;
    }
    float v[C];
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] = inside ? pixel_value<kDropout>(a, p, c) : 0.f;
    seed_table(sm.table, sm.lists, i0, j0, a.img_h, a.img_w, a.n);
    PixelSlots s;
    place_slots(s, sm.table, sm.lists, a.n, keep);
    __syncthreads();
    const int count = sm.table.count;
    if (count > kMaxRows) {
        add_slots<C, kDropout>(a, p, keep);
        return;
    }
    rank_rows(sm.table, count, [&](const int row, const int id) {
        const RowGeometry g = stage_geometry(a.xys, a.conics, id);
        float q[4 * kRowQuads];
        q[0] = g.x, q[1] = g.y, q[2] = g.a, q[3] = g.b, q[4] = g.c;
        bool finite = true;
#pragma unroll
        for (int c = 0; c < 4 * kRowQuads - 5; ++c) {
            q[5 + c] = c < C ? row_value<kDropout>(a, id, c) : 0.f;
            finite = finite && isfinite(q[5 + c]);
        }
        if (!finite) sm.table.per_slot = 1;
#pragma unroll
        for (int e = 0; e < kRowQuads; ++e) sm.rows[row * kRowQuads + e] = make_float4(q[4 * e], q[4 * e + 1], q[4 * e + 2], q[4 * e + 3]);
    });
    __syncthreads();
    bool regular = find_rows(s, sm.table, count) && sm.table.per_slot == 0;
    float *const weight = sm.weight[warp];
    float4 *const group = sm.group[warp];
    const float2 minus_x = make_float2(-(float)j, -(float)j), minus_y = make_float2(-(float)i, -(float)i);
    // a lane is a pixel: the first group's weights, the sums over all groups
    typename Rows<C>::Mine mine;
    float2 total2 = make_float2(0.f, 0.f), scores2 = make_float2(0.f, 0.f);
    int first_rows = 0;
    const int groups = visit_groups(s, sm.table, count, [&](const int at, const int first, const unsigned bits, const int begin, const int n) {
        const typename Rows<C>::Mine got = Rows<C>::gather(sm.rows, sm.table.order[warp], begin, n, first, group);
        if (at == 0) mine = got, first_rows = min(n - begin, kGroup);
        __syncwarp();
        for (int pair = 0; 2 * pair < min(n - begin, kGroup); ++pair) {
            const float4 *q = group + pair * kPairQuads;
            const float2 w = Rows<C>::weights(q, bits, minus_x, minus_y);
            float2 score = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < C; c += 2) {
                const float4 f = q[3 + c / 2];
                score = fma2(make_float2(f.x, f.y), make_float2(v[c], v[c]), score);
                if (c + 1 < C) score = fma2(make_float2(f.z, f.w), make_float2(v[c + 1 < C ? c + 1 : c], v[c + 1 < C ? c + 1 : c]), score);
            }
            total2 = add2(total2, w);
            scores2 = fma2(w, score, scores2);
            if (at == 0) weight[2 * pair * kWeightPitch + lane] = w.x, weight[(2 * pair + 1) * kWeightPitch + lane] = w.y;
        }
        __syncwarp();
    });
    const float total = total2.x + total2.y, scores = scores2.x + scores2.y;
    const bool some = total > 0.f;  // a pixel without a weight adds nothing, whatever its values
    const float inv = 1.f / (total + (float)kNormEps), m = some ? scores * inv * inv : 0.f;
    float size = fabsf(m);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        v[c] = some ? v[c] * inv : 0.f;
        size += fabsf(v[c]);
        sm.pixel[warp][c][lane] = v[c];
    }
    sm.pixel[warp][C][lane] = m;
    regular = regular && isfinite(size);
    if (!__all_sync(0xffffffffu, regular)) {
        if (inside) add_slots<C, kDropout>(a, p, keep);
        return;
    }
    // a lane is half a row
    const int half = lane >> 4, r = lane & (kGroup - 1);
    const float x0 = (float)(j0 + (warp & 1) * 8), y0 = (float)(i0 + (warp >> 1) * 4 + half * 2);
    auto sum_rows = [&](const int rows) {
        float2 dx[4], f[C], color[C];
#pragma unroll
        for (int e = 0; e < 4; ++e) dx[e] = make_float2(mine.x - (x0 + (float)(2 * e)), mine.x - (x0 + (float)(2 * e + 1)));
#pragma unroll
        for (int c = 0; c < C; ++c) f[c] = make_float2(-mine.f[c], -mine.f[c]), color[c] = make_float2(0.f, 0.f);
        float2 xx = make_float2(0.f, 0.f);
        float sx = 0.f, sy = 0.f, sxy = 0.f, syy = 0.f;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            float2 ts = make_float2(0.f, 0.f), us = make_float2(0.f, 0.f);
#pragma unroll
            for (int quad = 0; quad < 2; ++quad) {
                const int at = half * 16 + y * 8 + quad * 4;
                const float4 w4 = *reinterpret_cast<const float4 *>(&weight[r * kWeightPitch + at]);
                const float4 m4 = *reinterpret_cast<const float4 *>(&sm.pixel[warp][C][at]);
                float2 d0 = make_float2(m4.x, m4.y), d1 = make_float2(m4.z, m4.w);
                const float2 w0 = make_float2(w4.x, w4.y), w1 = make_float2(w4.z, w4.w);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const float4 v4 = *reinterpret_cast<const float4 *>(&sm.pixel[warp][c][at]);
                    const float2 v0 = make_float2(v4.x, v4.y), v1 = make_float2(v4.z, v4.w);
                    d0 = fma2(f[c], v0, d0), d1 = fma2(f[c], v1, d1);
                    if constexpr (kDropout) color[c] = fma2(w1, v1, fma2(w0, v0, color[c]));
                }
                const float2 t0 = mul2(w0, d0), t1 = mul2(w1, d1);
                const float2 u0 = mul2(t0, dx[2 * quad]), u1 = mul2(t1, dx[2 * quad + 1]);
                ts = add2(ts, add2(t0, t1)), us = add2(us, add2(u0, u1));
                xx = fma2(u1, dx[2 * quad + 1], fma2(u0, dx[2 * quad], xx));
            }
            const float dy = mine.y - (y0 + (float)y);
            const float tr = ts.x + ts.y, ur = us.x + us.y, ty = tr * dy;
            sx += ur, sy += ty;
            sxy = fmaf(ur, dy, sxy), syy = fmaf(ty, dy, syy);
        }
        float sum[kValues];
#pragma unroll
        for (int e = 0; e < kValues; ++e) sum[e] = 0.f;
        sum[0] = sx, sum[1] = sy, sum[2] = xx.x + xx.y, sum[3] = sxy, sum[4] = syy;
        if constexpr (kDropout) {
#pragma unroll
            for (int c = 0; c < C; ++c) sum[5 + c] = color[c].x + color[c].y;
        }
#pragma unroll
        for (int e = 0; e < 5 + (kDropout ? C : 0); ++e) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 16);
        if (r < rows) {
            float4 *out = reinterpret_cast<float4 *>(a.sums + (size_t)sm.table.sorted[mine.row] * kValues);
#pragma unroll
            for (int e = 0; e < kValues / 4; ++e)
                if ((e & 1) == half) atomicAdd(&out[e], make_float4(sum[4 * e], sum[4 * e + 1], sum[4 * e + 2], sum[4 * e + 3]));
        }
    };
    __syncwarp();
    if (groups > 0) sum_rows(first_rows);
    if (groups > 1)
        visit_groups(s, sm.table, count, [&](const int at, const int first, const unsigned bits, const int begin, const int n) {
            if (at == 0) return;
            mine = Rows<C>::gather(sm.rows, sm.table.order[warp], begin, n, first, group);
            __syncwarp();
            for (int pair = 0; 2 * pair < min(n - begin, kGroup); ++pair) {
                const float2 w = Rows<C>::weights(group + pair * kPairQuads, bits, minus_x, minus_y);
                weight[2 * pair * kWeightPitch + lane] = w.x, weight[(2 * pair + 1) * kWeightPitch + lane] = w.y;
            }
            __syncwarp();
            sum_rows(min(n - begin, kGroup));
            __syncwarp();
        });
}

template <int C, bool kDropout>
void launch_sums(const SumArgs &a, cudaStream_t s) {
    constexpr int kBytes = (int)sizeof(SumSmem<C, kDropout>);
    // past 48 KB (11 and 12 channels) the kernel has to be told; the setting is the device's, so every call makes it
    if (kBytes > 48 * 1024) cudaFuncSetAttribute(sums_kernel<C, kDropout>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    launch(sums_kernel<C, kDropout>, dim3(a.tiles_x * ceil_div(a.img_h, kTile)), dim3(kTilePixels), kBytes, s, a);
}

// Zero times a conic that is not finite is nothing here: a Gaussian without a weight has no gradient
__device__ __forceinline__ float times(const float conic, const float sum) { return sum != 0.f ? conic * sum : 0.f; }

template <int kValues>
__global__ void __launch_bounds__(256) finish_sums_kernel(const int n, const int channels, const float *__restrict__ conics,
                                                          const float *__restrict__ sums, const bool accumulate, float *__restrict__ v_xy,
                                                          float *__restrict__ v_conic, float *__restrict__ v_colors) {
    wait_for_predecessor();
    const int g = blockIdx.x * 256 + threadIdx.x;
    if (g >= n) return;
    float s[kValues];
#pragma unroll
    for (int e = 0; e < kValues / 4; ++e) {
        const float4 q = reinterpret_cast<const float4 *>(sums)[(size_t)g * (kValues / 4) + e];
        s[4 * e] = q.x, s[4 * e + 1] = q.y, s[4 * e + 2] = q.z, s[4 * e + 3] = q.w;
    }
    const float a = conics[3 * (size_t)g], b = conics[3 * (size_t)g + 1], c = conics[3 * (size_t)g + 2];
    const float out[5] = {times(a, s[0]) + times(b, s[1]), times(b, s[0]) + times(c, s[1]), 0.5f * s[2], s[3], 0.5f * s[4]};
#pragma unroll
    for (int e = 0; e < 5; ++e) {
        float *dst = e < 2 ? &v_xy[2 * (size_t)g + e] : &v_conic[3 * (size_t)g + e - 2];
        *dst = accumulate ? *dst + out[e] : out[e];
    }
#pragma unroll
    for (int e = 5; e < kValues; ++e)
        if (e - 5 < channels) v_colors[(size_t)g * channels + e - 5] = s[e];
}

}  // namespace igs
