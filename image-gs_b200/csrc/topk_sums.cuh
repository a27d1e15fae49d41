// The backward pass shared by the balance loss and the gate dropout: sums over pixels, per Gaussian, of products of its weight with values
// of the pixel. Both losses reach the gates n_k = w_k / D, D = eps + sum_j w_j, through a score that is linear in the row's values f_c and
// the pixel's values v_c, s_k = sum_c f_c v_c (dropout: the colour and v_out; balance: one value, alpha, and v = 1). With
//   v'_c = v_c / D,  m' = sum_j w_j s_j / D^2,  t = dL/dsigma = w (m' - sum_c f_c v'_c)
// a Gaussian's sums are sum t dx, t dy, t dx^2, t dx dy, t dy^2 and (dropout) w v'_c, from which the end forms
//   v_xy = (a Sx + b Sy, b Sx + c Sy),  v_conic = (Sxx / 2, Sxy, Syy / 2),  v_f = S_c.
//
// A warp (an 8x8 patch, topk_lists.cuh) goes over its rows twice. First a lane is two pixels: weights into shared memory (a row of 64 for
// each Gaussian), D and the scores' sum in registers. Then a lane is a row or, up to 16 rows, half of one, summing over the pixels: the
// weights are read four at a time and the pixels' v' and m' as broadcasts, two pixels per packed instruction; dy is one value per line of
// the patch, so t and t dx are summed along it first. The sums go to global memory with one 16-byte vector atomic per four values, in a
// buffer of their own that the last kernel (or CTA) turns into the gradients. A patch of more rows than a group goes over its groups once
// for D and the scores and once more for the sums. Where a value is not finite, or so large that a product could overflow (kValueLimit), the
// patch takes the per-slot path instead: zero times it would reach Gaussians that the pixel does not name.
//
// At 1920x1080 with 20,000 Gaussians the pass takes 59 us for the balance loss and 87 us for the dropout with three channels (the lists
// alone, read at the memory's rate, 13 us); one thread per pixel and five or eight atomics per slot took 900 and 1090 us. With nine
// channels (2048x2048, 50,000 Gaussians: 275 us) the shared-memory pipe is 79 % busy with the pixels' values. What bounds it
// stands in topk_lists.cuh. The sums are float and their atomics come in any order: the last bits of the gradients differ from run to run,
// as the render's do.
#pragma once

#include "topk_lists.cuh"

namespace igs {

struct SumArgs {
    int img_h, img_w, channels, n;
    const float *xys, *conics;
    const int *pixel_topk;
    const uint8_t *mask;         // balance: pixels that count (NULL: all)
    const int *counts;           // balance: alpha = *scale counts + v_importance, *scale = v_loss N / (A T)
    const long long *totals;
    const float *v_loss, *v_importance;
    float *scale;
    const float *colors, *v_output;  // dropout
    const long long *rng;
    uint32_t threshold;
    float *sums;                 // [N, SumLayout::kValues]
    unsigned *ticket;
    bool accumulate;
    float *v_xy, *v_conic, *v_colors;
};

// C: the values per row and pixel (balance: 1; dropout: the channels)
template <int C, bool kDropout>
struct SumLayout {
    static constexpr int kValues = ((5 + (kDropout ? C : 0)) + 3) / 4 * 4;  // Sx, Sy, Sxx, Sxy, Syy, S_c
};

template <int C, bool kDropout>
struct SumSmem {
    struct Warp {
        union {
            int keys[kKeyWords];
            alignas(16) float weight[kRows * kWeightPitch];
        };
        float4 pairs[Rows<C>::kGroupQuads];
        alignas(16) float pixel[C + 1][kPatchPixels];  // v'_c, m'
    } warp[kPatches];
};

// Value c of a Gaussian's score
template <bool kDropout>
__device__ __forceinline__ float row_value(const SumArgs &a, const int id, const int c) {
    if constexpr (kDropout) return __ldg(&a.colors[(size_t)id * a.channels + c]);
    const float scale = *a.scale;
    return scale * (float)a.counts[id] + (a.v_importance != nullptr ? a.v_importance[id] : 0.f);
}
template <bool kDropout>
__device__ __forceinline__ float pixel_value(const SumArgs &a, const int p, const int c) {
    if constexpr (kDropout) return __ldg(&a.v_output[(size_t)c * (a.img_h * a.img_w) + p]);
    return 1.f;
}

template <bool kDropout>
__device__ __forceinline__ auto sum_slots(const SumArgs &a, const int p, const bool inside) {
    if constexpr (kDropout) return KeptSlots({(uint64_t)a.rng[0], (uint64_t)a.rng[1], a.threshold}, (uint32_t)p, inside);
    else return AllSlots{inside && (a.mask == nullptr || a.mask[p] != 0)};
}

// One pixel's slots one by one, from global memory: a slot of weight 0 adds nothing
template <int C, bool kDropout>
__device__ __forceinline__ void add_pixel_slots(const SumArgs &a, const int p, const bool inside) {
    const auto may = sum_slots<kDropout>(a, p, inside);
    if (!may.any()) return;
    unsigned keep = 0;
#pragma unroll
    for (int k = 0; k < kTopK; ++k) keep |= may(k) ? 1u << k : 0u;
    constexpr int kValues = SumLayout<C, kDropout>::kValues;
    const float px = (float)(p % a.img_w), py = (float)(p / a.img_w);
    const int *list = a.pixel_topk + (size_t)p * kTopK;
    float total = (float)kNormEps, scores = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
        const float inv = 1.f / total, m = scores * inv * inv;
        for (int k = 0; k < kTopK; ++k) {
            const int id = list[k];
            if ((unsigned)id >= (unsigned)a.n || !(keep >> k & 1)) continue;
            const RowGeometry g = row_geometry(a.xys, a.conics, id);
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

// The sums zeroed, and balance's scale and the ticket
template <int kValues, bool kDropout>
__global__ void __launch_bounds__(256) zero_sums_kernel(const __grid_constant__ SumArgs a) {
    wait_for_predecessor();
    const int e = blockIdx.x * 256 + threadIdx.x;
    if (e == 0) *a.ticket = 0;
    if (!kDropout && e == 0) {
        const double slots = (double)a.totals[0], pixels = (double)a.totals[1];
        *a.scale = a.v_loss != nullptr && slots > 0.0 ? (float)((double)a.n / (slots * pixels)) * *a.v_loss : 0.f;
    }
    if (e < a.n * (kValues / 4)) reinterpret_cast<float4 *>(a.sums)[e] = make_float4(0.f, 0.f, 0.f, 0.f);
}

// Zero times a conic that is not finite is nothing here: a Gaussian without a weight has no gradient
__device__ __forceinline__ float times(const float conic, const float sum) { return sum != 0.f ? conic * sum : 0.f; }

// A Gaussian's gradients from its sums
template <int C, bool kDropout>
__device__ __forceinline__ void finish_gaussian(const SumArgs &a, const int g) {
    constexpr int kValues = SumLayout<C, kDropout>::kValues;
    float s[kValues];
#pragma unroll
    for (int e = 0; e < kValues / 4; ++e) {
        const float4 q = __ldcg(&reinterpret_cast<const float4 *>(a.sums)[(size_t)g * (kValues / 4) + e]);
        s[4 * e] = q.x, s[4 * e + 1] = q.y, s[4 * e + 2] = q.z, s[4 * e + 3] = q.w;
    }
    const float ca = a.conics[3 * (size_t)g], cb = a.conics[3 * (size_t)g + 1], cc = a.conics[3 * (size_t)g + 2];
    const float out[5] = {times(ca, s[0]) + times(cb, s[1]), times(cb, s[0]) + times(cc, s[1]), 0.5f * s[2], s[3], 0.5f * s[4]};
#pragma unroll
    for (int e = 0; e < 5; ++e) {
        float *dst = e < 2 ? &a.v_xy[2 * (size_t)g + e] : &a.v_conic[3 * (size_t)g + e - 2];
        *dst = a.accumulate ? *dst + out[e] : out[e];
    }
    if constexpr (kDropout) {
#pragma unroll
        for (int c = 0; c < C; ++c) a.v_colors[(size_t)g * C + c] = s[5 + c];
    }
}

template <int C, bool kDropout>
__global__ void __launch_bounds__(256) finish_sums_kernel(const __grid_constant__ SumArgs a) {
    wait_for_predecessor();
    const int g = blockIdx.x * 256 + threadIdx.x;
    if (g < a.n) finish_gaussian<C, kDropout>(a, g);
}

template <int C, bool kDropout>
__device__ __noinline__ void add_slots(const SumArgs &a) {
    const Patch patch(a.img_h, a.img_w);  // (made again: passed from the caller, it would live in the caller's local memory)
#pragma unroll
    for (int b = 0; b < kPix; ++b) add_pixel_slots<C, kDropout>(a, patch.p[b], patch.inside[b]);
}

template <int C, bool kDropout>
__device__ __forceinline__ PatchRows sum_rows(const SumArgs &a, const Patch &patch, const int g, int *keys) {
    return find_rows(a.pixel_topk, patch, a.n, [&](const int p, const bool inside) { return sum_slots<kDropout>(a, p, inside); }, g, keys);
}

// A lane is kPix pixels: the sums over the rows of its pixels' weights and of the weights times the scores
template <int C>
struct PixelSums {
    float v[kPix][C];
    float2 minus_x, minus_y[kPix], total[kPix], scores[kPix];

    template <bool kDropout>
    __device__ __forceinline__ void start(const SumArgs &a, const Patch &patch) {
        minus_x = make_float2(-(float)patch.j, -(float)patch.j);
#pragma unroll
        for (int b = 0; b < kPix; ++b) {
            minus_y[b] = make_float2(-(float)patch.i[b], -(float)patch.i[b]);
            total[b] = make_float2(0.f, 0.f), scores[b] = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < C; ++c) v[b][c] = patch.inside[b] ? pixel_value<kDropout>(a, patch.p[b], c) : 0.f;
        }
    }

    // The group's weights into shared memory, and into the sums
    __device__ __forceinline__ void add(const PatchRows &rows, const float4 *pairs, float *weight) {
        weight += threadIdx.x & 31;
        unsigned held[kPix];
#pragma unroll
        for (int b = 0; b < kPix; ++b) held[b] = rows.bits[b];
#pragma unroll 2
        for (int pair = 0; 2 * pair < rows.n; ++pair, pairs += Rows<C>::kPairQuads, weight += 2 * kWeightPitch) {
            float2 w[kPix];
            Rows<C>::weights(pairs, held, minus_x, minus_y, w);
#pragma unroll
            for (int b = 0; b < kPix; ++b) {
                held[b] >>= 2;
                weight[32 * b] = w[b].x, weight[kWeightPitch + 32 * b] = w[b].y;
                float2 score = make_float2(0.f, 0.f);
#pragma unroll
                for (int c = 0; c < C; ++c) score = fma2(Rows<C>::value(pairs, c), make_float2(v[b][c], v[b][c]), score);
                total[b] = add2(total[b], w[b]);
                scores[b] = fma2(w[b], score, scores[b]);
            }
        }
    }

    // v' and m' into shared memory; false, on all lanes, where they are not below kValueLimit
    __device__ __forceinline__ bool finish(float (&pixel)[C + 1][kPatchPixels]) {
        bool good = true;
#pragma unroll
        for (int b = 0; b < kPix; ++b) {
            const float t = total[b].x + total[b].y;
            const bool some = t > 0.f;  // a pixel without a weight adds nothing, whatever its values
            const float inv = reciprocal(t + (float)kNormEps), m = some ? (scores[b].x + scores[b].y) * inv * inv : 0.f;
            float size = fabsf(m);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float vc = some ? v[b][c] * inv : 0.f;
                size += fabsf(vc);
                pixel[c][32 * b + (threadIdx.x & 31)] = vc;
            }
            pixel[C][32 * b + (threadIdx.x & 31)] = m;
            good = good && size < kValueLimit;  // (not where it is NaN)
        }
        return __all_sync(0xffffffffu, good);
    }
};

// A lane is a row or, up to 16 rows, half of one: the group's sums into global memory
template <int C, bool kDropout>
__device__ __forceinline__ void add_rows(const SumArgs &a, const Patch &patch, const PatchRows &rows,
                                         const typename SumSmem<C, kDropout>::Warp &sm) {
    constexpr int kValues = SumLayout<C, kDropout>::kValues;
    const int lane = threadIdx.x & 31;
    const bool halves = rows.n <= 16;
    const int r = halves ? lane & 15 : min(lane, kRows - 1), half = halves ? lane >> 4 : 0;
    const int lines = halves ? kLines / 2 : kLines;
    const float *mine = reinterpret_cast<const float *>(sm.pairs + (r >> 1) * Rows<C>::kPairQuads) + (r & 1);
    auto field = [&](const int e) { return mine[2 * e]; };
    const float x = field(0) - (float)patch.x0;
    float dy = field(1) - (float)(patch.y0 + half * lines);
    float2 dx[4], f[C], color[C];
#pragma unroll
    for (int e = 0; e < 4; ++e) dx[e] = make_float2(x - (float)(2 * e), x - (float)(2 * e + 1));
#pragma unroll
    for (int c = 0; c < C; ++c) f[c].x = -field(5 + c), f[c].y = f[c].x, color[c] = make_float2(0.f, 0.f);
    float2 xx = make_float2(0.f, 0.f);
    float sx = 0.f, sy = 0.f, sxy = 0.f, syy = 0.f;
    const float *w_at = sm.weight + r * kWeightPitch + half * (kPatchPixels / 2), *v_at = &sm.pixel[0][half * (kPatchPixels / 2)];
#pragma unroll 4
    for (int line = 0; line < lines; ++line, dy -= 1.f, w_at += 8, v_at += 8) {
        float2 ts = make_float2(0.f, 0.f), us = make_float2(0.f, 0.f);
#pragma unroll
        for (int quad = 0; quad < 2; ++quad) {
            const float4 w4 = *reinterpret_cast<const float4 *>(w_at + quad * 4);
            const float4 m4 = *reinterpret_cast<const float4 *>(v_at + C * kPatchPixels + quad * 4);
            float2 d0 = make_float2(m4.x, m4.y), d1 = make_float2(m4.z, m4.w);
            const float2 w0 = make_float2(w4.x, w4.y), w1 = make_float2(w4.z, w4.w);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float4 v4 = *reinterpret_cast<const float4 *>(v_at + c * kPatchPixels + quad * 4);
                const float2 v0 = make_float2(v4.x, v4.y), v1 = make_float2(v4.z, v4.w);
                d0 = fma2(f[c], v0, d0), d1 = fma2(f[c], v1, d1);
                if constexpr (kDropout) color[c] = fma2(w1, v1, fma2(w0, v0, color[c]));
            }
            const float2 t0 = mul2(w0, d0), t1 = mul2(w1, d1);
            const float2 u0 = mul2(t0, dx[2 * quad]), u1 = mul2(t1, dx[2 * quad + 1]);
            ts = add2(ts, add2(t0, t1)), us = add2(us, add2(u0, u1));
            xx = fma2(u1, dx[2 * quad + 1], fma2(u0, dx[2 * quad], xx));
        }
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
    const int id = __shfl_sync(0xffffffffu, rows.id, r);
    if (halves) {
#pragma unroll
        for (int e = 0; e < 5 + (kDropout ? C : 0); ++e) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 16);
    }
    if ((halves ? r : lane) < rows.n) {
        float4 *out = reinterpret_cast<float4 *>(a.sums + (size_t)id * kValues);
#pragma unroll
        for (int e = 0; e < kValues / 4; ++e)
            if (!halves || (e & 1) == half) atomicAdd(&out[e], make_float4(sum[4 * e], sum[4 * e + 1], sum[4 * e + 2], sum[4 * e + 3]));
    }
}

// A patch of more rows than a group: all groups for the pixels' sums, then all again for the rows'
template <int C, bool kDropout>
__device__ __noinline__ bool sum_groups(const SumArgs &a, typename SumSmem<C, kDropout>::Warp &sm) {
    const Patch patch(a.img_h, a.img_w);
    PixelSums<C> pixels;
    pixels.template start<kDropout>(a, patch);
    for (int pass = 0; pass < 2; ++pass) {
        bool more = true;
        for (int g = 0; more; ++g) {
            const PatchRows rows = sum_rows<C, kDropout>(a, patch, g, sm.keys);
            more = rows.more;
            if (!Rows<C>::gather(rows, a.xys, a.conics, [&](const int id, const int c) { return row_value<kDropout>(a, id, c); }, sm.pairs))
                return false;
            __syncwarp();
            pixels.add(rows, sm.pairs, sm.weight);
            __syncwarp();
            if (pass == 1) add_rows<C, kDropout>(a, patch, rows, sm);
        }
        if (pass == 0 && !pixels.finish(sm.pixel)) return false;
        __syncwarp();
    }
    return true;
}

template <int C, bool kDropout>
__device__ __forceinline__ void sum_patch(const SumArgs &a) {
    extern __shared__ __align__(16) char smem_bytes[];
    typename SumSmem<C, kDropout>::Warp &sm = reinterpret_cast<SumSmem<C, kDropout> *>(smem_bytes)->warp[threadIdx.x >> 5];
    const Patch patch(a.img_h, a.img_w);
    if (patch.x0 >= a.img_w || patch.y0 >= a.img_h) return;
    const PatchRows rows = sum_rows<C, kDropout>(a, patch, 0, sm.keys);
    bool regular;
    if (rows.more) {
        regular = sum_groups<C, kDropout>(a, sm);
    } else {
        PixelSums<C> pixels;
        pixels.template start<kDropout>(a, patch);
        regular = Rows<C>::gather(rows, a.xys, a.conics, [&](const int id, const int c) { return row_value<kDropout>(a, id, c); }, sm.pairs);
        __syncwarp();
        pixels.add(rows, sm.pairs, sm.weight);
        regular = pixels.finish(sm.pixel) && regular;
        __syncwarp();
        if (regular) add_rows<C, kDropout>(a, patch, rows, sm);
    }
    if (!regular) add_slots<C, kDropout>(a);
}

// kFinish: the last CTA finishes the gradients. (A kernel of its own: with the barrier behind it, even never reached, the patch's code took
// 18 % more instructions.)
template <int C, bool kDropout, bool kFinish>
__global__ void __launch_bounds__(kPatchThreads, C <= 1 ? 6 : C <= 3 ? 5 : 4) sums_kernel(const __grid_constant__ SumArgs a) {
    wait_for_predecessor();
    sum_patch<C, kDropout>(a);
    if constexpr (kFinish) {
        if (!last_cta(a.ticket)) return;
        for (int g = threadIdx.x; g < a.n; g += kPatchThreads) finish_gaussian<C, kDropout>(a, g);
    }
}

// The backward pass; its workspace holds balance's scale and the ticket (16 bytes) and the sums
template <int C, bool kDropout>
constexpr size_t sum_bytes(const int n) {
    return 16 + sizeof(float) * SumLayout<C, kDropout>::kValues * (size_t)n;
}

template <int C, bool kDropout>
void launch_sums(SumArgs a, void *workspace, cudaStream_t s) {
    constexpr int kValues = SumLayout<C, kDropout>::kValues;
    constexpr int kBytes = (int)sizeof(SumSmem<C, kDropout>);
    const bool pixels = a.img_h > 0 && a.img_w > 0, in_last = pixels && a.n <= kFinishInLast;
    a.scale = static_cast<float *>(workspace);
    a.ticket = reinterpret_cast<unsigned *>(a.scale + 1);
    a.sums = a.scale + 4;
    launch(zero_sums_kernel<kValues, kDropout>, dim3(ceil_div(a.n * (kValues / 4), 256)), dim3(256), 0, s, a);
    if (pixels) {
        const auto kernel = in_last ? sums_kernel<C, kDropout, true> : sums_kernel<C, kDropout, false>;
        // past 48 KB the kernel has to be told; the setting belongs to the device, so every call makes it
        if (kBytes > 48 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
        launch(kernel, tile_grid(a.img_h, a.img_w), dim3(kPatchThreads), kBytes, s, a);
    }
    if (!in_last) launch(finish_sums_kernel<C, kDropout>, dim3(ceil_div(a.n, 256)), dim3(256), 0, s, a);
}

}  // namespace igs
