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

// The ten 24-bit draws of a pixel, compared with the threshold: bit k is set where slot k is kept. Two calls give eight words: slot k < 8
// takes the upper 24 bits of word k, slots 8 and 9 the low bytes of words 0, 1, 2 and 3, 4, 5 (the first most significant), which no other
// slot uses; a third call for two slots would cost half as much again.
__device__ __forceinline__ unsigned keep_bits(uint32_t pixel, uint64_t seed, uint64_t offset, uint32_t threshold) {
    const uint2 key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
    const uint32_t o0 = (uint32_t)offset, o1 = (uint32_t)(offset >> 32);
    const uint4 a = philox4x32(make_uint4(pixel, 0u, o0, o1), key), b = philox4x32(make_uint4(pixel, 1u, o0, o1), key);
    const uint32_t words[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    unsigned keep = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) keep |= (words[k] >> 8) >= threshold ? 1u << k : 0u;
    const uint32_t d8 = (words[0] & 255u) << 16 | (words[1] & 255u) << 8 | (words[2] & 255u);
    const uint32_t d9 = (words[3] & 255u) << 16 | (words[4] & 255u) << 8 | (words[5] & 255u);
    keep |= d8 >= threshold ? 1u << 8 : 0u;
    keep |= d9 >= threshold ? 1u << 9 : 0u;
    return keep;
}

// ---- a tile's Gaussians as rows --------------------------------------------------------------------------------------------------------
//
// One CTA of 256 threads takes a 16x16 tile, a warp an 8x4 patch of it, a lane one pixel. Neighbouring pixels name nearly the same
// Gaussians (at a trained image's 100 pixels per Gaussian the 2560 slots of a tile name 18 to 23, a patch 13 to 14), so the tile's distinct
// IDs become rows: a hash table in shared memory collects them, they are ranked by ID (so that every sum over rows has one order, whatever
// thread came first), and each row's parameters are staged once. A pixel's slots are then bits of a row mask. A warp takes the rows that
// any of its pixels holds in groups of 16, copied side by side in pairs: it reads them as broadcasts, two rows per packed (f32x2)
// instruction, with no gather per slot, and sums per Gaussian become sums along a row.
constexpr int kTableBits = 10;
constexpr int kTableSize = 1 << kTableBits;
constexpr int kMaxRows = 128;   // more distinct IDs in a tile than this (or an ID twice in a pixel) take the per-slot path
constexpr int kGroup = 16;      // rows of a warp's group
constexpr int kNoRow = 0xFF;
constexpr int kListPitch = 176;  // words per row of 16 pixels: 160, padded so that the 8x4 patches' 8-byte reads do not conflict
constexpr int kListWords = kTile * kListPitch;
constexpr int kWarps = kTilePixels / 32;

struct alignas(16) TileTable {
    int ids[kTableSize];        // -1: free
    uint8_t row[kTableSize];
    int found[kMaxRows];        // distinct IDs in the order found, and their places in the table
    uint16_t place[kMaxRows];
    int sorted[kMaxRows];       // the same by rank
    uint8_t order[kWarps][32];  // a warp's rows of the current 32, closed up
    int count;
    int per_slot;               // set when a row's values ask for the per-slot path
};

// Copies the tile's lists into shared memory (asynchronously; finish_lists waits) and clears the table
__device__ __forceinline__ void load_lists(int *s_lists, TileTable &t, const int *pixel_topk, const int i0, const int j0, const int img_h,
                                           const int img_w) {
    const int pairs = min(kTile, img_w - j0) * (kTopK / 2);  // 8-byte words of a row that lie in the image
    const int rows = min(kTile, img_h - i0);
#pragma unroll
    for (int m = 0; m < kTopK / 2; ++m) {
        const int idx = m * kTilePixels + threadIdx.x;
        const int r = idx / (kTile * kTopK / 2), q = idx % (kTile * kTopK / 2);
        if (r < rows && q < pairs) {
            const int *src = pixel_topk + ((size_t)(i0 + r) * img_w + j0) * kTopK + 2 * q;
            const uint32_t dst = (uint32_t)__cvta_generic_to_shared(s_lists + r * kListPitch + 2 * q);
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
        }
    }
#pragma unroll
    for (int e = 0; e < kTableSize / 4 / kTilePixels; ++e)
        reinterpret_cast<int4 *>(t.ids)[e * kTilePixels + threadIdx.x] = make_int4(-1, -1, -1, -1);
    if (threadIdx.x == 0) t.count = 0, t.per_slot = 0;
}

__device__ __forceinline__ int hash_of(const int id) { return (int)((unsigned)id * 2654435761u >> (32 - kTableBits)); }

// The place of id in the table, found or made. A new ID takes the next entry of found[]; count past kMaxRows means that the tile does not
// fit (the place returned is then meaningless, and so it is when the table is full).
static __device__ __noinline__ int table_place(TileTable &t, const int id) {
    int h = hash_of(id);
    for (int probe = 0; probe < kTableSize; ++probe, h = (h + 1) & (kTableSize - 1)) {
        int v = *(volatile int *)&t.ids[h];
        if (v == id) break;
        if (v == -1) {
            if (*(volatile int *)&t.count > kMaxRows) break;
            v = atomicCAS(&t.ids[h], -1, id);
            if (v == id) break;
            if (v == -1) {
                const int r = atomicAdd(&t.count, 1);
                if (r < kMaxRows) t.found[r] = id, t.place[r] = (uint16_t)h;
                break;
            }
        }
    }
    return h;
}

// Waits for the lists, then enters the IDs of 25 pixels spread over the tile, a thread each: nearly all of the tile's, so that afterwards
// most pixels only look theirs up. (Slots that the caller leaves out may enter too: a row that nobody holds is never visited.)
__device__ __forceinline__ void seed_table(TileTable &t, const int *s_lists, const int i0, const int j0, const int img_h, const int img_w,
                                           const int n) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    const int pixel = threadIdx.x / kTopK, slot = threadIdx.x % kTopK;
    const int y = (pixel / 5) * 15 / 4, x = (pixel % 5) * 15 / 4;  // 0, 3, 7, 11, 15
    if (pixel < 25 && i0 + y < img_h && j0 + x < img_w) {
        const int id = s_lists[y * kListPitch + x * kTopK + slot];
        if ((unsigned)id < (unsigned)n) table_place(t, id);
    }
    __syncthreads();
}

// The pixel of a thread: warp w covers the 8x4 patch (w % 2, w / 2) of the tile, lane l its pixel (l % 8, l / 8)
__device__ __forceinline__ int patch_x() { return (threadIdx.x >> 5 & 1) * 8 + (threadIdx.x & 7); }
__device__ __forceinline__ int patch_y() { return (threadIdx.x >> 6) * 4 + (threadIdx.x >> 3 & 3); }

// A pixel's slots: first their places in the table (-1: empty), then their rows
struct PixelSlots {
    int place[kTopK];
    unsigned rows[3];  // a byte per slot, kNoRow for an empty one
    unsigned bits;     // rows 0-31 as a mask
    int filled;
};

// From the pixel's list in shared memory; keep holds a bit per slot that may be filled
__device__ __forceinline__ void place_slots(PixelSlots &s, TileTable &t, const int *s_lists, const int n, const unsigned keep) {
    const int *list = s_lists + patch_y() * kListPitch + patch_x() * kTopK;
    s.filled = 0;
    unsigned missing = 0;
#pragma unroll
    for (int k = 0; k < kTopK; k += 2) {
        const int2 v = *reinterpret_cast<const int2 *>(list + k);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int id = b ? v.y : v.x;
            const bool filled = (unsigned)id < (unsigned)n && (keep >> (k + b) & 1) != 0;
            const int h = hash_of(id);
            s.place[k + b] = filled ? h : -1;
            s.filled += filled;
            if (filled && t.ids[h] != id) missing |= 1u << (k + b);
        }
    }
    if (__any_sync(0xffffffffu, missing != 0)) {
#pragma unroll
        for (int k = 0; k < kTopK; ++k)
            if (missing >> k & 1) s.place[k] = table_place(t, list[k]);
    }
}

// Ranks the IDs found (count <= kMaxRows), writes each place's row and calls stage(row, id); the caller synchronizes before and after
template <typename Stage>
__device__ __forceinline__ void rank_rows(TileTable &t, const int count, Stage stage) {
    for (int r = threadIdx.x; r < count; r += kTilePixels) {
        const int id = t.found[r];
        int rank = 0;
        for (int o = 0; o < count; ++o) rank += t.found[o] < id ? 1 : 0;
        t.row[t.place[r]] = (uint8_t)rank;
        t.sorted[rank] = id;
        stage(rank, id);
    }
}

// 1 << shift, 0 for a shift of 32 or more (the clamp of PTX's shl; in C++ it would be undefined)
__device__ __forceinline__ unsigned bit_or_nothing(const unsigned shift) {
    unsigned r;
    asm("shl.b32 %0, 1, %1;" : "=r"(r) : "r"(shift));
    return r;
}

// The rows of the slots with first <= row < first + 32 as a mask
__device__ __forceinline__ unsigned row_bits(const PixelSlots &s, const int first) {
    unsigned bits = 0;
#pragma unroll
    for (int k = 0; k < kTopK; ++k) bits |= bit_or_nothing((s.rows[k / 4] >> 8 * (k % 4) & 255) - first);
    return bits;
}

// After rank_rows: the slots' rows. False where an ID stands twice in the list, which the mask cannot say.
__device__ __forceinline__ bool find_rows(PixelSlots &s, const TileTable &t, const int count) {
    s.rows[0] = s.rows[1] = s.rows[2] = 0;
    s.bits = 0;
#pragma unroll
    for (int k = 0; k < kTopK; ++k) {
        const unsigned row = s.place[k] >= 0 ? t.row[s.place[k]] : kNoRow;
        s.rows[k / 4] |= row << 8 * (k % 4);
        s.bits |= bit_or_nothing(row);
    }
    int distinct = __popc(s.bits);
    for (int first = 32; first < count; first += 32) distinct += __popc(row_bits(s, first));
    return distinct == s.filled;
}

// exp2(x) (ex2.approx: 2 ulp; results below 2^-126 are 0, far below what eps leaves of a gate)
__device__ __forceinline__ float exp2_approx(const float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The staged geometry of a row: centre, and the conic times -log2(e) (its outer terms halved too), so that the weight is exp2 of
//   (a' dx) dx + (c' dy + b' dx) dy
// where that is not positive, and 0 where it is positive or NaN. A Gaussian whose parameters are not all finite has no finite sigma
// anywhere; it is staged at the origin with a NaN conic, so that its weights are 0 and its offsets finite.
struct RowGeometry {
    float x, y, a, b, c;
};

__device__ __forceinline__ RowGeometry stage_geometry(const float *xys, const float *conics, const int id) {
    constexpr float kLog2e = 1.4426950408889634f;
    RowGeometry g = {__ldg(&xys[2 * (size_t)id]), __ldg(&xys[2 * (size_t)id + 1]), __ldg(&conics[3 * (size_t)id]),
                     __ldg(&conics[3 * (size_t)id + 1]), __ldg(&conics[3 * (size_t)id + 2])};
    if (isfinite(g.x) && isfinite(g.y) && isfinite(g.a) && isfinite(g.b) && isfinite(g.c))
        return {g.x, g.y, -0.5f * kLog2e * g.a, -kLog2e * g.b, -0.5f * kLog2e * g.c};
    return {0.f, 0.f, __int_as_float(0x7fc00000), 0.f, 0.f};
}

// The weight of one slot, from global memory: the per-slot path
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
        : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)), "l"(reinterpret_cast<const uint64_t &>(c)));
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

// A staged row in the CTA's table: x, y, a', b', c', f[C], padded to whole float4s. A warp's group of 16 rows, in 8 pairs of
// (x x y y) (a' a' b' b') (c' c' m m) (f0 f0 f1 f1) ..., m the row's bit in the mask (0 for a row that pads the last pair).
template <int C>
struct Rows {
    static constexpr int kRowQuads = (5 + C + 3) / 4;
    static constexpr int kPairQuads = 3 + (C + 1) / 2;
    static constexpr int kGroupQuads = kGroup / 2 * kPairQuads;

    // This lane's row (lane % 16) of the group from the table, into registers and, by the first 16 lanes, into the warp's group
    struct Mine {
        int row;
        float x, y, f[C > 0 ? C : 1];
    };
    static __device__ __forceinline__ Mine gather(const float4 *table, const uint8_t *order, const int begin, const int n, const int first,
                                                  float4 *group) {
        const int lane = threadIdx.x & 31, r = lane & (kGroup - 1);
        const int bit = begin + r < n ? order[begin + r] : 0;
        Mine mine;
        mine.row = first + bit;
        float q[4 * kRowQuads];
#pragma unroll
        for (int e = 0; e < kRowQuads; ++e) {
            const float4 v = table[mine.row * kRowQuads + e];
            q[4 * e] = v.x, q[4 * e + 1] = v.y, q[4 * e + 2] = v.z, q[4 * e + 3] = v.w;
        }
        mine.x = q[0], mine.y = q[1];
#pragma unroll
        for (int c = 0; c < C; ++c) mine.f[c] = q[5 + c];
        if (lane < kGroup) {
            float *pair = reinterpret_cast<float *>(group + (r >> 1) * kPairQuads) + (r & 1);
#pragma unroll
            for (int e = 0; e < 5; ++e) pair[2 * e] = q[e];
            reinterpret_cast<unsigned *>(pair)[10] = begin + r < n ? 1u << bit : 0u;
#pragma unroll
            for (int c = 0; c < C; ++c) pair[12 + 2 * c] = q[5 + c];
        }
        return mine;
    }

    // The weights of a pair's two rows at a pixel; minus holds (-px, -px), (-py, -py)
    static __device__ __forceinline__ float2 weights(const float4 *pair, const unsigned bits, const float2 minus_x, const float2 minus_y) {
        const float4 xy = pair[0], ab = pair[1], cm = pair[2];
        const float2 dx = add2(make_float2(xy.x, xy.y), minus_x), dy = add2(make_float2(xy.z, xy.w), minus_y);
        const float2 slope = fma2(make_float2(cm.x, cm.y), dy, mul2(make_float2(ab.z, ab.w), dx));
        const float2 e = fma2(slope, dy, mul2(mul2(make_float2(ab.x, ab.y), dx), dx));
        const bool held0 = (bits & __float_as_uint(cm.z)) != 0, held1 = (bits & __float_as_uint(cm.w)) != 0;
        return make_float2(held0 && e.x <= 0.f ? exp2_approx(e.x) : 0.f, held1 && e.y <= 0.f ? exp2_approx(e.y) : 0.f);
    }
};

// Calls visit(first row of the 32, this lane's mask of them, begin, rows of the 32 that the warp holds) for each group of 16 rows that the
// warp's pixels hold, in order, with t.order closed up for it; all lanes of the warp together. Returns the number of groups.
template <typename Visit>
__device__ __forceinline__ int visit_groups(const PixelSlots &s, TileTable &t, const int count, Visit visit) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int groups = 0;
    for (int first = 0; first < count; first += 32) {
        const unsigned bits = first == 0 ? s.bits : row_bits(s, first);
        const unsigned any = __reduce_or_sync(0xffffffffu, bits);
        const int n = __popc(any);
        __syncwarp();
        if (any >> lane & 1) t.order[warp][__popc(any & ((1u << lane) - 1))] = (uint8_t)lane;
        __syncwarp();
        for (int begin = 0; begin < n; begin += kGroup, ++groups) visit(groups, first, bits, begin, n);
    }
    return groups;
}

// Host checks of the sizes, shared by the entry points: slots and Gaussians' sums indexed with 32 bits, coordinates exact in float
constexpr const char *kListsLimit = "at most 2^31 / 10 pixels, 2^24 pixels a side and 2^26 Gaussians";
inline bool lists_addressable(int img_height, int img_width, int num_points) {
    return (int64_t)img_height * img_width <= INT32_MAX / kTopK && img_height <= 1 << 24 && img_width <= 1 << 24 && num_points <= 1 << 26;
}

}  // namespace igs
