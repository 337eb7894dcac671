// What the attention of rows that share pages is made of: which keys a group of rows has in common, the items that the work is cut into,
// and where their results go.  See attention_shared.cu.
#pragma once
#include "capped_exp2.cuh"
#include "common.cuh"
#include "tcgen05.cuh"
#include <math_constants.h>

namespace qnn {
namespace shared {

constexpr int TILE = 16;                      // positions
constexpr float LOG2E = 1.4426950408889634f;

using tc::exp2_fast;

struct Shared {
    const int4* groups;                       // first row, rows, first position, position behind the last
    const int* row_group;                     // of a row: its group, or -1
    int n_groups, B;
    int common_ranges, own_ranges;            // S, P: parts 0 .. S - 1 of a row are of C, S .. S + P - 1 its own
    int common_tiles;                         // tiles of query rows of a group
    int most_rows;
    // Group g with the rows that the batch and the launch have room for.
    __device__ __forceinline__ int4 group(int g) const {
        int4 v = groups[g];
        v.y = v.x < 0 || v.x >= B ? 0 : min(min(v.y, most_rows), B - v.x);
        return v;
    }
    // The group of a row that holds it, or one without rows.
    __device__ __forceinline__ int4 group_of(int row) const {
        const int g = row_group[row];
        if (g < 0 || g >= n_groups) return make_int4(0, 0, 0, 0);
        int4 v = group(g);
        if (row < v.x || row - v.x >= v.y) v.y = 0;
        return v;
    }
};

struct Cells {                                // where keys and values lie
    const int* page_table;
    int max_pages, page_shift, ring_pages;    // ring_pages 0: every position kept
    const int* slots;
    const int* slot_len;
    int window;
};

// What an item works on, the same in all threads of its CTA: tiles t0 .. t1 - 1 of 16 positions each, the first `tiles_a` of the walk from
// position a0 on, the others from b0 on (both multiples of 16; a row's own keys lie on both sides of C).  Positions outside lo .. hi - 1 that
// a tile holds do not count.
struct Item {
    int row0, rows;                           // its rows of the batch
    int slot;                                 // whose page table says where the keys are
    int part;                                 // which part of those rows
    int query0;                               // first query of the tile: query m is row row0 + m / G, head m % G of the kv head
    int t0, t1;
    int tiles_a, a0, b0, lo, hi;
    __device__ __forceinline__ int position(int t) const { return t < tiles_a ? a0 + t * TILE : b0 + (t - tiles_a) * TILE; }
};

// The window's start and the length of a row (slot < 0: a row of no sequence, which sees nothing).
__device__ __forceinline__ int2 sees(const Cells& c, int slot) {
    if (slot < 0) return make_int2(0, 0);
    const int n = c.ring_pages > 0 ? c.slot_len[slot] : min(c.slot_len[slot], c.max_pages << c.page_shift);   // no further than its page table
    return make_int2(c.window > 0 && n > c.window ? n - c.window : 0, n);
}

// What the rows of the batch see, four rows a lane, where the batch has no more than 128: asked for before it is known which of them matter.
struct Seen {
    int slot[4];
    int2 w[4];
};
__device__ __forceinline__ bool ask_all(const Shared& sh) { return sh.B <= 128; }
__device__ __forceinline__ void ask_slots(const Shared& sh, const Cells& c, Seen& all) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int r = k * 32 + (threadIdx.x & 31);
        all.slot[k] = ask_all(sh) && r < sh.B ? c.slots[r] : -1;
    }
}
__device__ __forceinline__ void ask_lengths(const Cells& c, Seen& all) {
#pragma unroll
    for (int k = 0; k < 4; ++k) all.w[k] = sees(c, all.slot[k]);
}

// C of a group, by one warp (every lane gets it), and the slot of its first row that belongs to a sequence.  Of what all rows see only
// whole pages: no tile then holds a cell that nobody has written.
static __device__ int3 common_keys(const Shared& sh, const Cells& c, const Seen& all, int4 g) {
    const int lane = threadIdx.x & 31;
    int lo = g.z, hi = g.w, first = 0x7fffffff, slot = -1;    // first: the group's first row with a sequence, and its slot, of this lane's
    const auto count = [&](int r, int s, int2 w) {
        if (s < 0 || r < g.x || r - g.x >= g.y) return;
        lo = max(lo, w.x);
        hi = min(hi, w.y);
        if (r < first) {
            first = r;
            slot = s;
        }
    };
    if (ask_all(sh)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) count(k * 32 + lane, all.slot[k], all.w[k]);
    } else {
        for (int i0 = lane; i0 < g.y; i0 += 128) {
            Seen some;
#pragma unroll
            for (int k = 0; k < 4; ++k) some.slot[k] = i0 + k * 32 < g.y ? c.slots[g.x + i0 + k * 32] : -1;
            ask_lengths(c, some);
#pragma unroll
            for (int k = 0; k < 4; ++k) count(g.x + i0 + k * 32, some.slot[k], some.w[k]);
        }
    }
    lo = __reduce_max_sync(0xffffffffu, lo);
    hi = __reduce_min_sync(0xffffffffu, hi);
    const int leader = __reduce_min_sync(0xffffffffu, first);
    if (leader == 0x7fffffff) return make_int3(0, 0, -1);
    slot = __shfl_sync(0xffffffffu, slot, __ffs(__ballot_sync(0xffffffffu, first == leader)) - 1);
    const int mask = (1 << c.page_shift) - 1;
    lo = (lo + mask) & ~mask;
    hi &= ~mask;
    return make_int3(lo, max(lo, hi), slot);
}

// Range `range` of so many, in whole units of `unit` tiles.
__device__ __forceinline__ void take_range(Item& it, int tiles, int range, int ranges, int unit = 1) {
    const int per = ((tiles + unit - 1) / unit + ranges - 1) / ranges * unit;
    it.t0 = min(range * per, tiles);
    it.t1 = min(it.t0 + per, tiles);
}

// Range `range` of C of group `group` for the queries from tile `q_tile` on.  Every warp works it out.
static __device__ Item common_item(const Shared& sh, const Cells& c, int group, int q_tile, int range, int tile, int unit = 1) {
    Item it;
    Seen all;
    const int4 g = sh.group(group);
    ask_slots(sh, c, all);
    ask_lengths(c, all);
    it.row0 = g.x;
    it.rows = g.y;
    it.query0 = q_tile * tile;
    it.part = range;
    const int3 k = common_keys(sh, c, all, g);
    it.slot = k.z;
    it.tiles_a = 0;
    it.a0 = it.b0 = it.lo = k.x;
    it.hi = k.y;
    take_range(it, (k.y - k.x) / TILE, range, sh.common_ranges, unit);
    return it;
}

// Range `range` of row `row`'s own keys.
static __device__ Item own_item(const Shared& sh, const Cells& c, int row, int q_tile, int range, int tile) {
    Item it;
    Seen all;
    ask_slots(sh, c, all);
    it.row0 = row;
    it.rows = 1;
    it.query0 = q_tile * tile;
    it.part = sh.common_ranges + range;
    it.slot = c.slots[row];
    const int4 group = sh.group_of(row);
    ask_lengths(c, all);
    const int2 w = sees(c, it.slot);
    it.lo = w.x;
    it.hi = w.y;
    it.a0 = w.x & ~(TILE - 1);
    it.tiles_a = 0;
    it.b0 = it.a0;
    if (group.y > 0 && it.slot >= 0) {
        const int3 k = common_keys(sh, c, all, group);
        if (k.y > k.x) {                      // C lies inside what the row sees, and starts and ends with pages
            it.tiles_a = (k.x - it.a0) / TILE;
            it.b0 = k.y;
        }
    }
    take_range(it, it.tiles_a + max(0, it.hi - it.b0 + TILE - 1) / TILE, range, sh.own_ranges);
    return it;
}

// Where part `part` of query m of an item goes.
__device__ __forceinline__ size_t part_of(const Item& it, const Shared& sh, int m, int kh, int G, int nq) {
    return ((size_t)(it.row0 + m / G) * nq + kh * G + m % G) * (sh.common_ranges + sh.own_ranges) + it.part;
}

struct Scores {
    float scale, cap;
    const float* slopes;
};

// ---- the copy engine's view of both pools ---------------------------------------------------------------------------------------
// One tensor map for keys and values: rows of a head's elements, and the pools as a third dimension, whose stride is their distance (encoding
// a map takes the host about 3 us).  KV says which index is whose.
struct KV {
    int k, v;
};
__device__ __forceinline__ void load_rows(unsigned dst, const CUtensorMap* map, unsigned bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
inline int make_pools_map(CUtensorMap* map, KV* kv, const void* k_pool, const void* v_pool, long long rows, int hd, int box_rows) {
    tc::EncodeTiled enc = tc::tensor_map_encoder();
    if (enc == nullptr) return QNN_ERR_UNSUPPORTED;
    const bool v_first = (uintptr_t)v_pool < (uintptr_t)k_pool, one = k_pool == v_pool;
    const void* base = v_first ? v_pool : k_pool;
    *kv = {v_first ? 1 : 0, one || v_first ? 0 : 1};
    const cuuint64_t apart = v_first ? (uintptr_t)k_pool - (uintptr_t)v_pool : (uintptr_t)v_pool - (uintptr_t)k_pool;
    const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)rows, one ? 1u : 2u};
    const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, one ? (cuuint64_t)hd * 2 * rows : apart};
    const cuuint32_t box[3] = {64u, (cuuint32_t)box_rows, 1u}, estr[3] = {1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : QNN_ERR_ARGUMENT;
}

// The items of C on the 5th-generation tensor cores (attention_shared_tcgen05.cu): groups of many rows.
struct SharedLaunch {
    const void* q;
    long long q_stride;
    const void *k_pool, *v_pool;
    long long pool_rows;
    Cells cells;
    Shared sh;
    int nq, nkv, hd;
    Scores sc;
    float* part_o;
    float2* part_ml;
    int* status;
};
int launch_common_tcgen05(const SharedLaunch& a, cudaStream_t st);

}  // namespace shared
}  // namespace qnn
