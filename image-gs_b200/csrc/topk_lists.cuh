// What the operators over the top-K lists (balance.cu, gate_dropout.cu) share: one pixel's slots read from pixel_topk [H, W, 10], the
// weight of a slot, and the counter-based generator of the gate dropout.
//
// A slot is filled when its ID lies in [0, N) (and the pixel's mask is set, where there is one). Its weight is w = exp(-sigma) where sigma
// is finite and not negative, and 0 otherwise (the rasterizer's selection skips such a Gaussian, so its lists hold none; lists kept while
// the parameters move on may). The gate is n = w / (sum_j w_j + eps), eps = 1e-4 as in the render.
#pragma once

#include "igs_common.cuh"

namespace igs {

// Philox4x32-10: J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011 (table 2 and section 3.3:
// the multipliers, the Weyl constants of the key and the round). A counter of four words and a key of two give four random words.
__device__ __forceinline__ uint4 philox4x32(uint4 c, uint2 key) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)0xD2511F53u * c.x, b = (uint64_t)0xCD9E8D57u * c.z;
        c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ key.x, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ key.y, (uint32_t)a);
        key.x += 0x9E3779B9u, key.y += 0xBB67AE85u;
    }
    return c;
}

// Which slots of a pixel may be filled: all of them (counts says whether the pixel does at all), or those that a dropout draw keeps
struct AllSlots {
    bool counts;
    __device__ __forceinline__ bool any() const { return counts; }
    __device__ __forceinline__ bool operator()(int) const { return true; }
};

struct Dropout {
    uint64_t seed, offset;
    uint32_t threshold;  // rint(p 2^24)
};

// The ten 24-bit draws of a pixel, kept where they are not below the threshold. Two calls give eight words: slot k < 8 takes the upper 24
// bits of word k, slots 8 and 9 the low bytes of words 0, 1, 2 and 3, 4, 5 (the first most significant), which no other slot uses; a third
// call for two slots would cost half as much again.
struct KeptSlots {
    uint32_t words[8];
    uint32_t threshold;
    bool counts;
    __device__ __forceinline__ KeptSlots(const Dropout &d, const uint32_t pixel, const bool inside)
        : words{}, threshold(d.threshold), counts(inside && d.threshold < 1u << 24) {
        if (threshold == 0) return;  // p = 0: every word is high enough
        const uint2 key = make_uint2((uint32_t)d.seed, (uint32_t)(d.seed >> 32));
        const uint32_t o0 = (uint32_t)d.offset, o1 = (uint32_t)(d.offset >> 32);
        const uint4 a = philox4x32(make_uint4(pixel, 0u, o0, o1), key), b = philox4x32(make_uint4(pixel, 1u, o0, o1), key);
        words[0] = a.x, words[1] = a.y, words[2] = a.z, words[3] = a.w, words[4] = b.x, words[5] = b.y, words[6] = b.z, words[7] = b.w;
    }
    __device__ __forceinline__ bool any() const { return counts; }
    __device__ __forceinline__ bool operator()(const int k) const {  // where any()
        if (k < 8) return words[k] >= threshold << 8;                // word >> 8 >= threshold
        const int w = k == 8 ? 0 : 3;
        return ((words[w] & 255u) << 16 | (words[w + 1] & 255u) << 8 | (words[w + 2] & 255u)) >= threshold;
    }
};

// ---- a patch's Gaussians as rows -------------------------------------------------------------------------------------------------------
//
// A warp takes an 8x8 patch of pixels, a lane two of them. Neighbouring pixels name nearly the same Gaussians (at a trained image's 100
// pixels per Gaussian the 640 slots of a patch name 14 to 16, those of an 8x4 patch 13 to 14), so the patch's distinct IDs become rows, in
// the order of their IDs: every lane sorts its pixels' ten slots (a 29-comparator network) into shared memory, and the warp takes the
// smallest unconsumed ID of all its pixels again and again. An ID twice in one list becomes two rows. What a row means to a pixel is a bit
// of the lane's mask; the rows' parameters are read once, by a lane each, and laid side by side in pairs, so that the warp reads them as
// broadcasts, two rows per packed (f32x2) instruction, with no gather per slot, and sums per Gaussian become sums along a row. Patches need
// no other warp, so nothing waits at a barrier.
//
// The kernels are bound by instruction issue and the shared-memory pipe together (65 and 75 % busy; DRAM 20 %): of the 1120 instructions
// of a patch's counts and importance some 140 load the lists, 120 sort, 400 walk to the rows, 330 weigh and 100 sum along the rows.
// Measured on the way, counts and importance of 1920x1080 pixels and 20,000 Gaussians: one thread per pixel and an atomic per slot 330 us;
// the tile's IDs collected by its warps in one hash table in shared memory 88 us (twice the instructions, and time at barriers); patches of
// 8x4 pixels 63 us; 8x8 54 us. Copying a patch's lists through shared memory in whole lines (58 us where direct loads took 57) and
// prefetching those of a later patch (115.6 us for both passes, 113.4 without) gained nothing.
//
// kRows is the shared memory of a patch's weights against the patches that do not fit it: 32 rows leave 5 CTAs on an SM, 28 leave 6 (125
// and 118 us for both passes of the balance loss at 100 pixels per Gaussian, 142 and 137 at 40, 153 and 171 at 25), 24 leave 7 (116, 157
// and 262 us).
constexpr int kRows = 28;  // rows of a group: a patch with more goes over them group by group
constexpr unsigned kRowsEnd = 1u << kRows;
static_assert(kRows % 2 == 0 && kRows < 32, "whole pairs, and a bit for each row with one to spare");

// The patch of a warp: 8 pixels by kLines, kPix of a lane, one above the other, four lines apart
constexpr int kPix = 2;
constexpr int kLines = 4 * kPix;
constexpr int kPatchPixels = 32 * kPix;
constexpr int kPatches = kTilePixels / kPatchPixels;  // of a CTA: a 16x16 tile
constexpr int kPatchThreads = kPatches * 32;
constexpr int kKeyWords = kPix * (kTopK + 1) * 32;    // shared memory of a warp for find_rows
constexpr int kWeightPitch = kPatchPixels + 4;        // of a row of weights: four pixels by eight rows are read from distinct banks

struct Patch {
    int x0, y0, j, i[kPix], p[kPix];
    bool inside[kPix];
    __device__ __forceinline__ Patch(const int img_h, const int img_w) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        x0 = blockIdx.x * kTile + (warp & 1) * 8, y0 = blockIdx.y * kTile + (warp >> 1) * kLines;
        j = x0 + (lane & 7);
#pragma unroll
        for (int b = 0; b < kPix; ++b) {
            i[b] = y0 + (lane >> 3) + 4 * b;
            inside[b] = i[b] < img_h && j < img_w;
            p[b] = inside[b] ? i[b] * img_w + j : 0;
        }
    }
};

// A sorting network for ten keys: A. Waksman's of 29 comparators (1969; D. Knuth, The Art of Computer Programming, volume 3, section 5.3.4),
// nine steps deep
__device__ __forceinline__ void sort_slots(int (&key)[kTopK]) {
    constexpr int kPairs[29][2] = {{4, 9}, {3, 8}, {2, 7}, {1, 6}, {0, 5}, {1, 4}, {6, 9}, {0, 3}, {5, 8}, {0, 2}, {3, 6}, {7, 9},
                                   {0, 1}, {2, 4}, {5, 7}, {8, 9}, {1, 2}, {4, 6}, {7, 8}, {3, 5}, {2, 5}, {6, 8}, {1, 3}, {4, 7},
                                   {2, 3}, {6, 7}, {3, 4}, {5, 6}, {4, 5}};
#pragma unroll
    for (int c = 0; c < 29; ++c) {
        const int i = kPairs[c][0], j = kPairs[c][1];
        const int lo = min(key[i], key[j]), hi = max(key[i], key[j]);
        key[i] = lo, key[j] = hi;
    }
}

// Rows [kRows g, kRows (g + 1)) of the patch
struct PatchRows {
    int n;                // how many there are, at most kRows
    bool more;            // whether others follow
    unsigned bits[kPix];  // the rows that this lane's pixels hold
    int id;               // lane l < n: the ID of row l,
    int holders;          // and how many pixels hold it
    int filled;           // how many of this lane's pixels have a slot at all
};

// slots(pixel, inside) says which of a pixel's slots may be filled; keys: kKeyWords of shared memory. All lanes together.
template <typename Slots>
__device__ __forceinline__ PatchRows find_rows(const int *pixel_topk, const Patch &patch, const int n_points, const Slots slots, const int g,
                                               int *keys) {
    const int lane = threadIdx.x & 31;
    const int none = n_points;  // the key of an empty slot: behind every ID
    int key[kPix][kTopK];
    bool counts[kPix];
#pragma unroll
    for (int b = 0; b < kPix; ++b) {
        const int2 *list = reinterpret_cast<const int2 *>(pixel_topk + (size_t)patch.p[b] * kTopK);  // (some pixel's, if it is outside)
#pragma unroll
        for (int k = 0; k < kTopK; k += 2) {
            const int2 v = __ldg(&list[k / 2]);
            key[b][k] = v.x, key[b][k + 1] = v.y;
        }
    }
#pragma unroll
    for (int b = 0; b < kPix; ++b) {
        const auto may = slots(patch.p[b], patch.inside[b]);
#pragma unroll
        for (int k = 0; k < kTopK; ++k) key[b][k] = may(k) ? (int)min((unsigned)key[b][k], (unsigned)none) : none;
        counts[b] = may.any();
    }
    PatchRows rows = {};
    int head[kPix], next[kPix];
#pragma unroll
    for (int b = 0; b < kPix; ++b) {
        sort_slots(key[b]);
        head[b] = counts[b] ? key[b][0] : none;  // a list is read on only where its head was taken
        rows.filled += head[b] != none;
        next[b] = (b * (kTopK + 1) + 1) * 32 + lane;
    }
    __syncwarp();
#pragma unroll
    for (int b = 0; b < kPix; ++b) {
        int *const column = keys + b * (kTopK + 1) * 32 + lane;
#pragma unroll
        for (int k = 1; k < kTopK; ++k) column[k * 32] = key[b][k];
        column[kTopK * 32] = none;
    }
    auto smallest = [&]() { return __reduce_min_sync(0xffffffffu, min(head[0], head[kPix - 1])); };
    for (int skip = kRows * g; skip > 0; --skip) {
        const int id = smallest();
#pragma unroll
        for (int b = 0; b < kPix; ++b)
            if (head[b] == id && id != none) head[b] = keys[next[b]], next[b] += 32;
    }
    const unsigned mine = 1u << lane;
    unsigned bit = 1, holders[kPix] = {};
    do {
        const int id = smallest();
        if (id == none) break;
#pragma unroll
        for (int b = 0; b < kPix; ++b) {
            const bool held = head[b] == id;
            const unsigned all = __ballot_sync(0xffffffffu, held);
            if (held) head[b] = keys[next[b]], next[b] += 32, rows.bits[b] |= bit;
            if (bit == mine) holders[b] = all;
        }
        if (bit == mine) rows.id = id;
        bit <<= 1;
    } while (bit != kRowsEnd);
    rows.n = bit != kRowsEnd ? __ffs(bit) - 1 : kRows;
    rows.more = bit == kRowsEnd && smallest() != none;
#pragma unroll
    for (int b = 0; b < kPix; ++b) rows.holders += __popc(holders[b]);
    __syncwarp();
    return rows;
}

// exp2(x) (ex2.approx: 2 ulp, 2^-22 of the weight; results below 2^-126 are 0, far below what eps leaves of a gate)
__device__ __forceinline__ float exp2_approx(const float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// A Gaussian's geometry as the kernels use it: centre, and the conic times -log2(e) (its outer terms halved too), so that the weight is
// exp2 of
//   (a' dx) dx + (c' dy + b' dx) dy
// which is not positive for a positive definite conic. Folding the factor in costs two of the at most 8 roundings of 2^-24 of the terms'
// magnitudes that the exponent has. Where the conic's determinant is at least 2^-16 of a c, none of them makes it positive either: the terms'
// magnitudes are then at most 2^18 times sigma and round by 2^-21 of themselves, and the weight needs no test. Other conics (axes more than
// about 500 to 1 among them), and parameters that are not finite or so large that the terms could overflow, are not regular: the patches that
// meet one take the per-slot path, which tests.
struct RowGeometry {
    float x, y, a, b, c;
    bool regular;
};

__device__ __forceinline__ RowGeometry row_geometry(const float *xys, const float *conics, const int id) {
    constexpr float kLog2e = 1.4426950408889634f;
    const float x = __ldg(&xys[2 * (size_t)id]), y = __ldg(&xys[2 * (size_t)id + 1]);
    const float a = __ldg(&conics[3 * (size_t)id]), b = __ldg(&conics[3 * (size_t)id + 1]), c = __ldg(&conics[3 * (size_t)id + 2]);
    const float ac = a * c;
    const bool regular = fabsf(x) < 1e9f && fabsf(y) < 1e9f && a > 0.f && a < 1e15f && c > 0.f && c < 1e15f &&
                         ac - b * b > 0x1p-16f * ac;
    return {x, y, -0.5f * kLog2e * a, -kLog2e * b, -0.5f * kLog2e * c, regular};
}

// The weight of one slot, for the per-slot path: 0 where sigma is negative, NaN or infinite
__device__ __forceinline__ float slot_weight(const RowGeometry &g, const float px, const float py) {
    const float dx = g.x - px, dy = g.y - py;
    const float e = fmaf(fmaf(g.c, dy, g.b * dx), dy, (g.a * dx) * dx);
    return e <= 0.f ? exp2_approx(e) : 0.f;
}

// Two float operations in one instruction
__device__ __forceinline__ float2 fma2(const float2 a, const float2 b, const float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(r))
        : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)),
          "l"(reinterpret_cast<const uint64_t &>(c)));
    return r;
}
__device__ __forceinline__ float2 mul2(const float2 a, const float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(r))
        : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)));
    return r;
}
__device__ __forceinline__ float2 add2(const float2 a, const float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(r))
        : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)));
    return r;
}

// Sums of magnitudes of a row's values, and of a pixel's, that the row path takes. It multiplies every row of a patch with every pixel and
// leaves out by a weight of zero, so the products have to be finite where they do not count too: at most 2^120 in all.
constexpr float kValueLimit = 0x1p60f;

// The rows of a group with C values f each, in shared memory in pairs: (x x y y) (a' a' b' b') (c' c' f0 f0) (f1 f1 f2 f2) ... Each row is
// read by a lane of its own from the parameters' arrays as they are. (Laid out beforehand as one block per Gaussian, the rows take fewer
// and wider loads; the render is 2 % faster so at 3840x2160, no faster at 1920x1080, and a small one slower by the launch: 4.7 against
// 3.9 us.)
template <int C>
struct Rows {
    static constexpr int kPairQuads = (5 + C + 1) / 2;
    static constexpr int kGroupQuads = kRows / 2 * kPairQuads;

    // value(id, c) gives f_c. False, on all lanes, where a row is not regular or its values are not below kValueLimit.
    template <typename Value>
    static __device__ __forceinline__ bool gather(const PatchRows &rows, const float *xys, const float *conics, Value value,
                                                  float4 *pairs) {
        const int lane = threadIdx.x & 31;
        float q[5 + C];
#pragma unroll
        for (int e = 0; e < 5 + C; ++e) q[e] = 0.f;
        bool good = true;
        if (lane < rows.n) {
            const RowGeometry g = row_geometry(xys, conics, rows.id);
            q[0] = g.x, q[1] = g.y, q[2] = g.a, q[3] = g.b, q[4] = g.c;
            float size = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c) q[5 + c] = value(rows.id, c), size += fabsf(q[5 + c]);
            good = g.regular && size < kValueLimit;  // (not where it is NaN)
        }
        if (lane <= rows.n && lane < kRows) {  // one more, of zeros, to pad the last pair
            float *pair = reinterpret_cast<float *>(pairs + (lane >> 1) * kPairQuads) + (lane & 1);
#pragma unroll
            for (int e = 0; e < 5 + C; ++e) pair[2 * e] = q[e];
        }
        return __all_sync(0xffffffffu, good);
    }

    // The weights of a pair's two rows at the lane's pixels, bits 0 and 1 of held saying which a pixel holds; minus_x is (-px, -px)
    static __device__ __forceinline__ void weights(const float4 *pair, const unsigned (&held)[kPix], const float2 minus_x,
                                                   const float2 (&minus_y)[kPix], float2 (&w)[kPix]) {
        const float4 xy = pair[0], ab = pair[1];
        const float2 c = *reinterpret_cast<const float2 *>(&pair[2]);
        const float2 dx = add2(make_float2(xy.x, xy.y), minus_x);
        const float2 bdx = mul2(make_float2(ab.z, ab.w), dx), adx2 = mul2(mul2(make_float2(ab.x, ab.y), dx), dx);
#pragma unroll
        for (int b = 0; b < kPix; ++b) {
            const float2 dy = add2(make_float2(xy.z, xy.w), minus_y[b]);
            const float2 e = fma2(fma2(c, dy, bdx), dy, adx2);
            w[b] = make_float2((held[b] & 1) ? exp2_approx(e.x) : 0.f, (held[b] & 2) ? exp2_approx(e.y) : 0.f);
        }
    }
    static __device__ __forceinline__ float2 value(const float4 *pair, const int c) {
        return reinterpret_cast<const float2 *>(pair)[5 + c];
    }
};

// Few Gaussians are finished by the last CTA of the patches' kernel instead of a kernel of its own. Both passes of the balance loss in a
// graph: 15.4 against 16.4 us at 100 Gaussians (64x64), 16.0 against 16.8 at 256, but 19.9 against 18.1 at 500 and 22.8 against 17.4 at
// 1000 (256x256); called one by one they gain the host's time for a launch each (48 against 53 us then, at all these sizes).
constexpr int kFinishInLast = 400;  // (igs_b200/pipeline.py counts its kernels by it)

// Whether this CTA is the last to come here, of all CTAs of the grid; what the others wrote before is then visible. All threads together.
__device__ __forceinline__ bool last_cta(unsigned *ticket) {
    __threadfence();
    __syncthreads();
    const bool last = __syncthreads_or(threadIdx.x == 0 && atomicAdd(ticket, 1u) == gridDim.x * gridDim.y - 1);
    if (last) __threadfence();
    return last;
}

// 1 / x to 2 ulp
__device__ __forceinline__ float reciprocal(const float x) { return __fdividef(1.f, x); }

// Host checks of the sizes, shared by the entry points: slots and Gaussians' sums indexed with 32 bits, coordinates exact in float, tiles
// within a grid
constexpr const char *kListsLimit = "at most 2^31 / 10 pixels, 65535 tiles a side and 2^26 Gaussians";
inline bool lists_addressable(int img_height, int img_width, int num_points) {
    return (int64_t)img_height * img_width <= INT32_MAX / kTopK && img_height <= 65535 * kTile && img_width <= 65535 * kTile &&
           num_points <= 1 << 26;
}
inline dim3 tile_grid(int img_height, int img_width) { return dim3(ceil_div(img_width, kTile), ceil_div(img_height, kTile)); }

}  // namespace igs
