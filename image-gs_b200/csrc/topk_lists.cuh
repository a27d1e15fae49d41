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
// Gaussians (at a trained image's 100 pixels per Gaussian the 2560 slots of a tile name about 25, a patch about 14), so the tile's distinct
// IDs become rows: a hash table in shared memory collects them, they are ranked by ID (so that every sum over rows has one order, whatever
// thread came first), and each row's parameters are staged once. A pixel's slots are then bits of a row mask, and a warp visits the rows
// that any of its pixels holds, reading the parameters as broadcasts: no gather per slot, and sums per Gaussian become sums along a row.
constexpr int kTableBits = 9;
constexpr int kTableSize = 1 << kTableBits;
constexpr int kMaxRows = 128;       // more distinct IDs in a tile than this (or an ID twice in a pixel) take the per-slot path
constexpr int kNoRow = 0xFF;
constexpr int kListPitch = 176;     // words per row of 16 pixels: 160, padded so that the 8x4 patches' 8-byte reads do not conflict
constexpr int kListWords = kTile * kListPitch;

struct alignas(16) TileTable {
    int ids[kTableSize];            // -1: free
    uint8_t row[kTableSize];
    int found[kMaxRows];            // distinct IDs in the order found, and their places in the table
    uint16_t place[kMaxRows];
    int sorted[kMaxRows];           // the same by rank
    int count;
    int per_slot;                   // set when a row's values ask for the per-slot path
};

// Copies the tile's lists into shared memory (asynchronously; wait with finish_lists) and clears the table
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
    for (int e = threadIdx.x; e < kTableSize; e += kTilePixels) t.ids[e] = -1;
    if (threadIdx.x == 0) t.count = 0, t.per_slot = 0;
}

__device__ __forceinline__ void finish_lists() {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
}

// The place of id in the table, found or made. A new ID takes the next entry of found[]; count past kMaxRows means that the tile does not
// fit (the place returned is then meaningless, and so it is when the table is full).
__device__ __forceinline__ int table_place(TileTable &t, const int id) {
    int h = (int)((unsigned)id * 2654435761u >> (32 - kTableBits));
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

// exp2(x) (ex2.approx: 2 ulp, 0 for -inf)
__device__ __forceinline__ float exp2_approx(const float x) {
    float r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
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
    const int2 *list = reinterpret_cast<const int2 *>(s_lists + patch_y() * kListPitch + patch_x() * kTopK);
    s.filled = 0;
#pragma unroll
    for (int k = 0; k < kTopK; k += 2) {
        const int2 v = list[k / 2];
        s.place[k] = (unsigned)v.x < (unsigned)n && (keep >> k & 1) ? table_place(t, v.x) : -1;
        s.place[k + 1] = (unsigned)v.y < (unsigned)n && (keep >> (k + 1) & 1) ? table_place(t, v.y) : -1;
        s.filled += (s.place[k] >= 0) + (s.place[k + 1] >= 0);
    }
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

// Calls visit(row, held) for each row that a pixel of the warp holds, in order, held being whether this lane's pixel does; all lanes of the
// warp together
template <typename Visit>
__device__ __forceinline__ void visit_rows(const PixelSlots &s, const int count, Visit visit) {
    for (int first = 0; first < count; first += 32) {
        const unsigned bits = first == 0 ? s.bits : row_bits(s, first);
        unsigned any = __reduce_or_sync(0xffffffffu, bits);
        while (any) {
            const int b = __ffs(any) - 1;
            any &= any - 1;
            visit(first + b, (bits >> b & 1) != 0);
        }
    }
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

__device__ __forceinline__ float row_exponent(const float4 g, const float c, const float px, const float py) {
    const float dx = g.x - px, dy = g.y - py;
    return fmaf(fmaf(c, dy, g.w * dx), dy, (g.z * dx) * dx);
}

// Host checks of the sizes, shared by the entry points: slots and Gaussians' sums indexed with 32 bits, coordinates exact in float
constexpr const char *kListsLimit = "at most 2^31 / 10 pixels, 2^24 pixels a side and 2^26 Gaussians";
inline bool lists_addressable(int img_height, int img_width, int num_points) {
    return (int64_t)img_height * img_width <= INT32_MAX / kTopK && img_height <= 1 << 24 && img_width <= 1 << 24 && num_points <= 1 << 26;
}

}  // namespace igs
