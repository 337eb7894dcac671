// Decode attention of a batch whose rows hold a stretch of positions in the same pages of the cache: beams of one request, several
// replies to one prompt, requests behind one common text.
//
// One query row per sequence, as in attention.cu:  o_r = sum_j softmax_j(s_rj) v_j  over the keys j that row r sees,
// s_rj = softcap(scale q_r . k_j) - slope (newest_r - j).  The keys of a row fall into two sets: C, which all rows of its group see and
// hold in the same pages, and its own.  With  m = max s,  l = sum e^{s - m},  O = sum e^{s - m} v  of each set (and of any range of it),
//     o_r = sum_i e^{m_i - M} O_i / (sum_i e^{m_i - M} l_i + e^{sink - M}),   M = max_i m_i,
// so the keys of C are read once for all rows of the group: the products with them are matrices of (rows x query heads of a kv head).
//
// C is where the group's common pages (positions begin .. end - 1 of `groups`) meet what every row sees: from the latest window's start to
// the shortest row's length.  No key of C is masked for any row, so whatever a key holds that one row sees and another does not
// (an Inf, a NaN) stays with the rows that see it.  The keys of [begin, end) outside C are among each row's own.
//
// Work is cut into items, a CTA each: (group, tile of query rows, range of C) and (row, tile of query heads, range of its own keys),
// per kv head.  An item leaves (m, l, O) in scratch (m in units of log2), and a second kernel joins a row's items in ascending order:
// results depend on the numbers of ranges, not on what runs when.
#include "attention_generic.cuh"

using namespace qnn;

namespace {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

struct Shared {
    const int4* groups;                       // first row, rows, first position, position behind the last
    const int* row_group;                     // of a row: its group, or -1
    int n_groups, B;
    int common_ranges, own_ranges;            // S, P: parts 0 .. S - 1 of a row are of C, S .. S + P - 1 its own
    int common_tiles;                         // tiles of query rows of a group
};

struct Cells {                                // where keys and values lie
    const int* page_table;
    int max_pages, page_shift, ring_pages;    // ring_pages 0: every position kept
    const int* slots;
    const int* slot_len;
    int window;
};

// What an item works on, the same in all threads of its CTA.
struct Item {
    int row0, rows;                           // its rows of the batch
    int slot;                                 // whose page table says where the keys are
    int part;                                 // which part of those rows
    int query0;                               // first query of the tile: query m is row row0 + m / G, head m % G of the kv head
    int begin, end;                           // logical keys: key i stands at position first + i, from gap_at on gap further
    int first, gap_at, gap;
    __device__ __forceinline__ int position(int i) const { return first + i + (i >= gap_at ? gap : 0); }
};

// The window's start and the length of a row (slot < 0: a row of no sequence, which sees nothing).
__device__ __forceinline__ int2 sees(const Cells& c, int slot) {
    if (slot < 0) return make_int2(0, 0);
    const int n = c.ring_pages > 0 ? c.slot_len[slot] : min(c.slot_len[slot], c.max_pages << c.page_shift);   // no further than its page table
    return make_int2(c.window > 0 && n > c.window ? n - c.window : 0, n);
}

// C of a group, by one warp (every lane gets it), and the slot of its first row that belongs to a sequence.
__device__ int3 common_keys(const Cells& c, int4 g) {
    int lo = g.z, hi = g.w, slot = -1;
    for (int i = threadIdx.x & 31; i < g.y; i += 32) {
        const int s = c.slots[g.x + i];
        if (s < 0) continue;
        const int2 w = sees(c, s);
        lo = max(lo, w.x);
        hi = min(hi, w.y);
        if (slot < 0) slot = s;
    }
    lo = __reduce_max_sync(0xffffffffu, lo);
    hi = __reduce_min_sync(0xffffffffu, hi);
    const unsigned have = __ballot_sync(0xffffffffu, slot >= 0);
    if (have == 0) return make_int3(0, 0, -1);
    slot = __shfl_sync(0xffffffffu, slot, __ffs(have) - 1);
    return make_int3(lo, max(lo, hi), slot);
}

// Item x of the launch: common_tiles x S items of every group first, then own_tiles x P items of every row.  Every warp works it out.
// `tile`: queries of an item.  Ranges are cut to whole multiples of 16 keys.
__device__ Item item_of(const Shared& sh, const Cells& c, int x, int G, int tile) {
    Item it;
    const int common_items = sh.n_groups * sh.common_tiles * sh.common_ranges;
    int ranges, range, keys;
    if (x < common_items) {
        ranges = sh.common_ranges;
        range = x % ranges;
        const int rest = x / ranges;
        const int4 g = sh.groups[rest / sh.common_tiles];
        it.query0 = rest % sh.common_tiles * tile;
        it.row0 = g.x;
        it.rows = g.y;
        it.part = range;
        const int3 k = common_keys(c, g);
        it.slot = k.z;
        it.first = k.x;
        it.gap_at = 0x7fffffff;
        it.gap = 0;
        keys = k.y - k.x;
    } else {
        const int own_tiles = (G + tile - 1) / tile;
        ranges = sh.own_ranges;
        x -= common_items;
        range = x % ranges;
        const int rest = x / ranges;
        it.query0 = rest % own_tiles * tile;
        it.row0 = rest / own_tiles;
        it.rows = 1;
        it.part = sh.common_ranges + range;
        it.slot = c.slots[it.row0];
        const int g = sh.row_group[it.row0];
        const int2 w = sees(c, it.slot);
        it.first = w.x;
        it.gap_at = 0x7fffffff;
        it.gap = 0;
        keys = w.y - w.x;
        if (g >= 0 && it.slot >= 0) {
            const int3 k = common_keys(c, sh.groups[g]);
            it.gap_at = k.x - w.x;            // C lies inside what the row sees
            it.gap = k.y - k.x;
            keys -= it.gap;
        }
    }
    const int per = ((keys + ranges - 1) / ranges + 15) & ~15;
    it.begin = min(range * per, keys);
    it.end = min(it.begin + per, keys);
    return it;
}

// The page ids of an item's keys, pages from that of its first position on; returns the number of that page.
__device__ __forceinline__ int load_pages(const Item& it, const Cells& c, int* pages) {
    const int first = it.position(it.begin) >> c.page_shift, last = it.position(it.end - 1) >> c.page_shift;
    const int* row = c.page_table + (size_t)it.slot * c.max_pages;
    for (int u = threadIdx.x; u <= last - first; u += blockDim.x) {
        const int p = first + u;
        pages[u] = row[c.ring_pages > 0 ? p % c.ring_pages : p];
    }
    return first;
}

// Where part `part` of query m of an item goes.
__device__ __forceinline__ size_t part_of(const Item& it, const Shared& sh, int m, int kh, int G, int nq) {
    return ((size_t)(it.row0 + m / G) * nq + kh * G + m % G) * (sh.common_ranges + sh.own_ranges) + it.part;
}

// ---- tensor cores, bfloat16 -------------------------------------------------------------------------------------------------
// As in attention_decode_mma.cu the keys fill the 16-row side of mma.m16n8k16 and queries the 8-column side,
//     S^T[16 keys x 8 q] = K Q^T,    O^T[hd x 8 q] += V^T P^T,
// here with NT column tiles (8 NT queries) for every fragment of K and V that ldmatrix brings.  A warp walks its own tiles of 16 keys
// (cp.async, a ring of STAGES), so nothing but the last merge is shared between the warps of a CTA.  P^T is the transpose of S^T's
// accumulator, eight by eight (movmatrix).  The exponentials are taken against a reference that is raised only when a score
// exceeds it by more than 8 (in log2): the stale reference cancels in the division, P stays below 2^8.
constexpr int TILE = 16;
constexpr float REFERENCE_STEP = 8.f;

__device__ __forceinline__ void cp_async_16(unsigned dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0));   // 0 bytes: zeros
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t transposed_8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}

constexpr int WARPS = 2, STAGES = 3;

template <int HD, int NT, bool BIAS>
__global__ void __launch_bounds__(WARPS * 32)
attn_shared_mma_kernel(const bf16* __restrict__ q, size_t q_stride, const bf16* __restrict__ k_pool, const bf16* __restrict__ v_pool,
                       const Cells cells, const Shared sh, int nq, int nkv, float scale, float cap, float* __restrict__ part_o,
                       float2* __restrict__ part_ml, const float* __restrict__ slopes) {
    constexpr int KSTEPS = HD / 16, CH = HD / 8, ROW_BYTES = HD * 2, TILE_BYTES = TILE * ROW_BYTES, PER_LANE = TILE * CH / 32, QT = 8 * NT;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    const int kh = blockIdx.y, G = nq / nkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // slots, lengths, page tables and groups come from the host before the step: they are read before the wait for the kernel in front
    const Item it = item_of(sh, cells, blockIdx.x, G, QT);
    const int queries = min(QT, it.rows * G - it.query0);
    const unsigned wbase = (unsigned)__cvta_generic_to_shared(smem_raw) + warp * STAGES * 2 * TILE_BYTES;
    int* pages = reinterpret_cast<int*>(smem_raw + (size_t)WARPS * STAGES * 2 * TILE_BYTES);
    int first_page = 0;
    if (it.begin < it.end) first_page = load_pages(it, cells, pages);
    pdl_wait();
    if (queries <= 0) return;
    if (it.begin >= it.end) {                                 // a range without keys
        for (int m = threadIdx.x; m < queries; m += blockDim.x) part_ml[part_of(it, sh, it.query0 + m, kh, G, nq)] = make_float2(-CUDART_INF_F, 0.f);
        return;
    }
    __syncthreads();

    float o[NT][KSTEPS][4], m0[NT], m1[NT], l0[NT], l1[NT];   // queries 8 nt + 2t and 8 nt + 2t + 1
    uint32_t qf[NT][KSTEPS][2];                               // Q^T: query 8 nt + g, elements 16 ks + 2t, +1 and 16 ks + 8 + 2t, +1
    float slope0[NT], slope1[NT];
    int newest0[NT], newest1[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m0[nt] = m1[nt] = -CUDART_INF_F;
        l0[nt] = l1[nt] = 0.f;
        const int m = it.query0 + nt * 8 + g;
        const bool have = nt * 8 + g < queries;
        const uint32_t* row = reinterpret_cast<const uint32_t*>(q + (have ? (size_t)(it.row0 + m / G) * q_stride + (size_t)(kh * G + m % G) * HD : 0));
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) {
            qf[nt][ks][0] = have ? row[ks * 8 + t] : 0u;
            qf[nt][ks][1] = have ? row[ks * 8 + 4 + t] : 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[nt][ks][j] = 0.f;
        }
        if (BIAS) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int c = nt * 8 + 2 * t + e, mm = it.query0 + c;
                float sl = 0.f;
                int nw = 0;
                if (c < queries) {
                    sl = slopes[kh * G + mm % G] * LOG2E;
                    const int slot = cells.slots[it.row0 + mm / G];
                    nw = slot >= 0 ? cells.slot_len[slot] - 1 : 0;
                }
                (e ? slope1[nt] : slope0[nt]) = sl;
                (e ? newest1[nt] : newest0[nt]) = nw;
            }
        }
    }

    const int first = it.begin + warp * TILE, stride = WARPS * TILE;
    const int my_tiles = first < it.end ? (it.end - first + stride - 1) / stride : 0;
    const int page_mask = (1 << cells.page_shift) - 1;
    auto fetch = [&](int n) {
        if (n < my_tiles) {
            const int base = first + n * stride;
            const unsigned kst = wbase + (n % STAGES) * 2 * TILE_BYTES, vst = kst + TILE_BYTES;
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) {
                const int idx = i * 32 + lane, row = idx / CH, chunk = idx % CH;
                const bool valid = base + row < it.end;
                const int p = it.position(valid ? base + row : it.begin);
                const size_t off = ((((size_t)pages[(p >> cells.page_shift) - first_page] * nkv + kh) << cells.page_shift) + (p & page_mask)) * HD + chunk * 8;
                const unsigned dst = row * ROW_BYTES + ((chunk ^ (row & 7)) << 4);
                cp_async_16(kst + dst, k_pool + off, valid);
                cp_async_16(vst + dst, v_pool + off, valid);
            }
        }
        cp_async_commit();                                    // an empty group keeps the count uniform
    };
#pragma unroll
    for (int n = 0; n < STAGES - 1; ++n) fetch(n);

    const float k1 = cap > 0.f ? scale / cap : scale * LOG2E, k2 = cap * LOG2E;
    for (int n = 0; n < my_tiles; ++n) {
        fetch(n + STAGES - 1);
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const int base = first + n * stride;
        const unsigned kst = wbase + (n % STAGES) * 2 * TILE_BYTES, vst = kst + TILE_BYTES;
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[nt][j] = 0.f;
        {
            const int row = lane & 15, half = lane >> 4;
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks) {
                uint32_t a[4];
                ldmatrix_x4(a, kst + row * ROW_BYTES + (((ks * 2 + half) ^ (row & 7)) << 4));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    if (nt == 0 || nt * 8 < queries) mma_16816(s[nt], a, qf[nt][ks][0], qf[nt][ks][1]);
            }
        }
        // s[nt][0], [1]: key base + g, queries 2t, 2t + 1; [2], [3]: key base + g + 8
        const bool v_lo = base + g < it.end, v_hi = base + g + 8 < it.end;
        int p_lo = 0, p_hi = 0;
        if (BIAS) {
            p_lo = it.position(base + g);
            p_hi = it.position(base + g + 8);
        }
        bool above = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x = s[nt][j] * k1;
                if (cap > 0.f) x = k2 * tanh_approx(x);
                if (BIAS) x -= ((j & 1) ? slope1[nt] : slope0[nt]) * (float)(((j & 1) ? newest1[nt] : newest0[nt]) - ((j < 2) ? p_lo : p_hi));
                s[nt][j] = ((j < 2) ? v_lo : v_hi) ? x : -CUDART_INF_F;
            }
            above |= fmaxf(s[nt][0], s[nt][2]) > m0[nt] + REFERENCE_STEP || fmaxf(s[nt][1], s[nt][3]) > m1[nt] + REFERENCE_STEP;
        }
        if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float x0 = fmaxf(s[nt][0], s[nt][2]), x1 = fmaxf(s[nt][1], s[nt][3]);
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, off));
                    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, off));
                }
                x0 = fmaxf(m0[nt], x0);
                x1 = fmaxf(m1[nt], x1);
                // -inf only before the first key (every tile has one; a score of -inf counts as no key)
                const float c0 = m0[nt] == -CUDART_INF_F ? 0.f : exp2_fast(m0[nt] - x0), c1 = m1[nt] == -CUDART_INF_F ? 0.f : exp2_fast(m1[nt] - x1);
                m0[nt] = x0;
                m1[nt] = x1;
                l0[nt] *= c0;
                l1[nt] *= c1;
#pragma unroll
                for (int i = 0; i < KSTEPS; ++i) {
                    o[nt][i][0] *= c0;
                    o[nt][i][1] *= c1;
                    o[nt][i][2] *= c0;
                    o[nt][i][3] *= c1;
                }
            }
        }
        uint32_t pb[NT][2];                                   // P^T: query g, keys 2t, 2t + 1 and 2t + 8, 2t + 9
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float r0 = m0[nt] == -CUDART_INF_F ? 0.f : m0[nt], r1 = m1[nt] == -CUDART_INF_F ? 0.f : m1[nt];
            const float a0 = exp2_fast(s[nt][0] - r0), a1 = exp2_fast(s[nt][1] - r1), a2 = exp2_fast(s[nt][2] - r0), a3 = exp2_fast(s[nt][3] - r1);
            l0[nt] += a0 + a2;
            l1[nt] += a1 + a3;
            pb[nt][0] = transposed_8x8(pack_bf16(a0, a1));
            pb[nt][1] = transposed_8x8(pack_bf16(a2, a3));
        }
        {
            const int row = (lane & 7) + ((lane >> 4) << 3), sub = (lane >> 3) & 1;
#pragma unroll
            for (int mt = 0; mt < KSTEPS; ++mt) {
                uint32_t a[4];
                ldmatrix_x4_trans(a, vst + row * ROW_BYTES + (((mt * 2 + sub) ^ (row & 7)) << 4));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    if (nt == 0 || nt * 8 < queries) mma_16816(o[nt][mt], a, pb[nt][0], pb[nt][1]);
            }
        }
        __syncwarp();                                         // the stage may be refilled
    }
    cp_async_wait<0>();
    __syncthreads();
    // the warps' states through shared memory, [warp][query][HD + 2], joined in warp order
    float* ms = reinterpret_cast<float*>(smem_raw);
    constexpr int ROW = HD + 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float s0 = l0[nt], s1 = l1[nt];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
            s0 += __shfl_xor_sync(0xffffffffu, s0, off);
            s1 += __shfl_xor_sync(0xffffffffu, s1, off);
        }
        float* r0 = ms + ((size_t)warp * QT + nt * 8 + 2 * t) * ROW;
        float* r1 = r0 + ROW;
#pragma unroll
        for (int mt = 0; mt < KSTEPS; ++mt) {
            r0[mt * 16 + g] = o[nt][mt][0];
            r1[mt * 16 + g] = o[nt][mt][1];
            r0[mt * 16 + g + 8] = o[nt][mt][2];
            r1[mt * 16 + g + 8] = o[nt][mt][3];
        }
        if (g == 0) {
            r0[HD] = m0[nt];
            r0[HD + 1] = s0;
            r1[HD] = m1[nt];
            r1[HD + 1] = s1;
        }
    }
    __syncthreads();
    for (int m = 0; m < queries; ++m) {
        float mm = -CUDART_INF_F, coef[WARPS], ll = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, ms[((size_t)w * QT + m) * ROW + HD]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float mw = ms[((size_t)w * QT + m) * ROW + HD];
            coef[w] = mw == -CUDART_INF_F ? 0.f : exp2_fast(mw - mm);
            ll += coef[w] * ms[((size_t)w * QT + m) * ROW + HD + 1];
        }
        const size_t at = part_of(it, sh, it.query0 + m, kh, G, nq);
        for (int d = threadIdx.x; d < HD; d += blockDim.x) {
            float acc = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) acc += coef[w] * ms[((size_t)w * QT + m) * ROW + d];
            part_o[at * HD + d] = acc;
        }
        if (threadIdx.x == 0) part_ml[at] = make_float2(mm, ll);
    }
}

// ---- any head size, float32 or bfloat16 ----------------------------------------------------------------------------------------
// Tiles of 32 keys as float32 in shared memory (rows an odd number of floats apart); a lane forms the scores of one key, then the lanes
// take the head's elements.  A warp keeps GEN_Q queries; exact exponentials and tanh in float32.
constexpr int GEN_WARPS = 4, GEN_Q = 4, GEN_QT = GEN_WARPS * GEN_Q;

template <typename T, int DPL>                                // elements of a head per lane, at most
__global__ void __launch_bounds__(GEN_WARPS * 32)
attn_shared_generic_kernel(const T* __restrict__ q, size_t q_stride, const T* __restrict__ k_pool, const T* __restrict__ v_pool,
                           const Cells cells, const Shared sh, int nq, int nkv, int hd, int tile_keys, float scale, float cap,
                           float* __restrict__ part_o, float2* __restrict__ part_ml, const float* __restrict__ slopes) {
    constexpr int VEC = Vec16<T>::N;
    extern __shared__ __align__(16) float sm[];
    const int kh = blockIdx.y, G = nq / nkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Item it = item_of(sh, cells, blockIdx.x, G, GEN_QT);
    const int queries = min(GEN_QT, it.rows * G - it.query0);
    pdl_wait();
    if (queries <= 0) return;
    const int pitch = hd + 1;
    float* sk = sm;
    float* sv = sk + tile_keys * pitch;
    float* sq = sv + tile_keys * pitch;                       // [GEN_QT][hd], times the scale
    for (int i = threadIdx.x; i < queries * hd; i += blockDim.x) {
        const int m = it.query0 + i / hd, d = i % hd;
        sq[i] = to_f(q[(size_t)(it.row0 + m / G) * q_stride + (size_t)(kh * G + m % G) * hd + d]) * scale;
    }
    float mx[GEN_Q], l[GEN_Q], o[GEN_Q][DPL], slope[GEN_Q];
    int newest[GEN_Q];
#pragma unroll
    for (int i = 0; i < GEN_Q; ++i) {
        mx[i] = -CUDART_INF_F;
        l[i] = 0.f;
        slope[i] = 0.f;
        newest[i] = 0;
        const int m = warp * GEN_Q + i, mm = it.query0 + m;
        if (slopes != nullptr && m < queries) {
            slope[i] = slopes[kh * G + mm % G];
            const int slot = cells.slots[it.row0 + mm / G];
            newest[i] = slot >= 0 ? cells.slot_len[slot] - 1 : 0;
        }
#pragma unroll
        for (int d = 0; d < DPL; ++d) o[i][d] = 0.f;
    }
    const int chunks = hd / VEC, page_mask = (1 << cells.page_shift) - 1;
    for (int base = it.begin; base < it.end; base += tile_keys) {
        const int n = min(tile_keys, it.end - base);
        __syncthreads();                                      // the tile before has been read
        const int* table = cells.page_table + (size_t)it.slot * cells.max_pages;
        for (int i = threadIdx.x; i < n * chunks; i += blockDim.x) {
            const int j = i / chunks, c = i % chunks, p = it.position(base + j);
            const int pn = p >> cells.page_shift, page = table[cells.ring_pages > 0 ? pn % cells.ring_pages : pn];
            const size_t off = ((((size_t)page * nkv + kh) << cells.page_shift) + (p & page_mask)) * hd + c * VEC;
            Vec16<T> kv, vv;
            kv.load(k_pool + off);
            vv.load(v_pool + off);
            float a[VEC], b[VEC];
            kv.unpack(a);
            vv.unpack(b);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                sk[j * pitch + c * VEC + e] = a[e];
                sv[j * pitch + c * VEC + e] = b[e];
            }
        }
        __syncthreads();
        const bool valid = lane < n;
        const int pos = valid ? it.position(base + lane) : 0;
#pragma unroll
        for (int i = 0; i < GEN_Q; ++i) {
            const int m = warp * GEN_Q + i;
            if (m >= queries) break;
            float s = 0.f;
            if (valid) {
                const float* kr = sk + lane * pitch;
                const float* qr = sq + m * hd;
                for (int d = 0; d < hd; ++d) s = fmaf(qr[d], kr[d], s);
                s = softcap_t<T>(s, cap) - slope[i] * (float)(newest[i] - pos);
            }
            const float top = fmaxf(mx[i], warp_max(valid ? s : -CUDART_INF_F));
            const float keep = mx[i] == -CUDART_INF_F ? 0.f : fexp<T>(mx[i] - top);
            const float w = valid && (top != -CUDART_INF_F || s != s) ? fexp<T>(s - top) : 0.f;
            l[i] = l[i] * keep + warp_sum(w);
            mx[i] = top;
#pragma unroll
            for (int d = 0; d < DPL; ++d) o[i][d] *= keep;
            for (int j = 0; j < n; ++j) {
                const float wj = __shfl_sync(0xffffffffu, w, j);
#pragma unroll
                for (int d = 0; d < DPL; ++d)
                    if (lane + d * 32 < hd) o[i][d] = fmaf(wj, sv[j * pitch + lane + d * 32], o[i][d]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < GEN_Q; ++i) {
        const int m = warp * GEN_Q + i;
        if (m >= queries) break;
        const size_t at = part_of(it, sh, it.query0 + m, kh, G, nq);
        if (l[i] > 0.f || l[i] != l[i])                       // (a NaN among the scores has to come out)
#pragma unroll
            for (int d = 0; d < DPL; ++d)
                if (lane + d * 32 < hd) part_o[at * hd + lane + d * 32] = o[i][d];
        if (lane == 0) part_ml[at] = make_float2(mx[i] * LOG2E, l[i]);
    }
}

// ---- the parts of a row joined ---------------------------------------------------------------------------------------------------
// A block per (row, head): threads in groups of hd / 4, group g adds parts g, g + groups, ...; the groups' sums in ascending order.  Parts
// without keys (l = 0) are not read.
template <typename T>
__global__ void attn_shared_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, T* __restrict__ out, size_t out_stride,
                                        int nq, int hd, int S, int P, const int* __restrict__ row_group, const int* __restrict__ slots,
                                        const float* __restrict__ sinks) {
    pdl_wait();
    extern __shared__ __align__(16) float js[];               // [groups][hd], then the parts' weights
    const int row = blockIdx.x / nq, h = blockIdx.x % nq, parts = S + P;
    const int lpg = hd / 4, groups = blockDim.x / lpg;
    float* weight = js + (size_t)groups * hd;
    float* inverse = weight + parts;
    const int from = row_group[row] >= 0 && slots[row] >= 0 ? 0 : S;      // a row of no group or no sequence has no part in C
    const size_t at = (size_t)blockIdx.x * parts;
    if (threadIdx.x < 32) {
        float M = -CUDART_INF_F;
        for (int p = from + threadIdx.x; p < parts; p += 32) {
            const float2 ml = part_ml[at + p];
            if (ml.y != 0.f) M = fmaxf(M, ml.x);
        }
        M = warp_max(M);
        float sum = 0.f;
        for (int p = from + threadIdx.x; p < parts; p += 32) {
            const float2 ml = part_ml[at + p];
            const float w = ml.y != ml.y ? ml.y : (ml.y != 0.f ? exp2f(ml.x - M) : 0.f);      // a NaN among the scores has to come out
            weight[p] = w;
            sum += w != 0.f ? w * ml.y : 0.f;
        }
        sum = warp_sum(sum);
        if (threadIdx.x == 0) {
            const float all = sinks != nullptr ? sum + exp2f(sinks[h] * LOG2E - M) : sum;
            *inverse = sum != 0.f ? 1.f / all : 0.f;
        }
    }
    __syncthreads();
    const int g = threadIdx.x / lpg, c = (threadIdx.x % lpg) * 4;
    if (g < groups) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = from + g; p < parts; p += groups) {
            const float w = weight[p];
            if (w == 0.f) continue;
            const float4 v = *reinterpret_cast<const float4*>(part_o + (at + p) * hd + c);
            acc.x += w * v.x;
            acc.y += w * v.y;
            acc.z += w * v.z;
            acc.w += w * v.w;
        }
        *reinterpret_cast<float4*>(js + (size_t)g * hd + c) = acc;
    }
    __syncthreads();
    const float inv = *inverse;
    for (int d = threadIdx.x; d < hd; d += blockDim.x) {
        float acc = 0.f;
        for (int i = 0; i < groups; ++i) acc += js[(size_t)i * hd + d];
        out[(size_t)row * out_stride + (size_t)h * hd + d] = from_f<T>(acc * inv);
    }
}

bool on_tensor_cores(int dtype, int hd) { return dtype == QNN_DT_BF16 && (hd == 64 || hd == 128 || hd == 256); }

// Column tiles of an item for so many queries: 1, 2 or, up to head size 128, 4.  More do not fit the registers (O and Q of 16 queries of 256
// elements are 192 registers a thread).
int column_tiles(int hd, int queries) { return queries <= 8 ? 1 : (queries <= 16 || hd > 128 ? 2 : 4); }

template <int HD, int NT, bool BIAS>
int launch_mma(const void* q, long long q_stride, const void* k_pool, const void* v_pool, const Cells& cells, const Shared& sh, int items, int nq,
               int nkv, float scale, float cap, float* part_o, float2* part_ml, const float* slopes, cudaStream_t st) {
    size_t smem = (size_t)WARPS * STAGES * 2 * TILE * HD * 2 + ((size_t)cells.max_pages + 2) * sizeof(int);
    const size_t merge = (size_t)WARPS * 8 * NT * (HD + 2) * sizeof(float);
    if (smem < merge) smem = merge;
    if (smem > 220 * 1024) return QNN_ERR_UNSUPPORTED;
    auto kern = attn_shared_mma_kernel<HD, NT, BIAS>;
    static OncePerDevice asked;
    if (const int rc = allow_shared(asked, kern, 220 * 1024)) return rc;
    launch_pdl(kern, dim3(items, nkv), dim3(WARPS * 32), smem, st, (const bf16*)q, (size_t)q_stride, (const bf16*)k_pool, (const bf16*)v_pool, cells,
               sh, nq, nkv, scale, cap, part_o, part_ml, slopes);
    return (int)cudaGetLastError();
}

template <typename T, int DPL>
int launch_generic(const void* q, long long q_stride, const void* k_pool, const void* v_pool, const Cells& cells, const Shared& sh, int items, int nq,
                   int nkv, int hd, float scale, float cap, float* part_o, float2* part_ml, const float* slopes, cudaStream_t st) {
    const int keys = hd <= 512 ? 32 : 16;
    const size_t smem = ((size_t)2 * keys * (hd + 1) + (size_t)GEN_QT * hd) * sizeof(float);
    auto kern = attn_shared_generic_kernel<T, DPL>;
    static OncePerDevice asked;
    if (const int rc = allow_shared(asked, kern, 220 * 1024)) return rc;
    launch_pdl(kern, dim3(items, nkv), dim3(GEN_WARPS * 32), smem, st, (const T*)q, (size_t)q_stride, (const T*)k_pool, (const T*)v_pool, cells, sh, nq,
               nkv, hd, keys, scale, cap, part_o, part_ml, slopes);
    return (int)cudaGetLastError();
}

template <typename T>
int launch_join(const float* part_o, const float2* part_ml, void* out, long long out_stride, int B, int nq, int hd, int S, int P, const int* row_group,
                const int* slots, const float* sinks, cudaStream_t st) {
    const int lpg = hd / 4;
    int groups = 256 / lpg;
    if (groups > S + P) groups = S + P;
    if (groups < 1) groups = 1;
    int threads = groups * lpg;
    if (threads < 32) threads = 32;
    groups = threads / lpg;                                   // as the kernel counts them
    const size_t smem = ((size_t)groups * hd + S + P + 1) * sizeof(float);
    launch_pdl(attn_shared_join_kernel<T>, dim3((unsigned)(B * nq)), dim3(threads), smem, st, part_o, part_ml, (T*)out, (size_t)out_stride, nq, hd, S, P,
               row_group, slots, sinks);
    return (int)cudaGetLastError();
}

}  // namespace

// Queries that one item takes (what the number of items, and with it the choice of ranges, goes by), or a negative number for a head
// size that is not taken.  `queries`: rows x query heads per kv head of the largest group.
QNN_API int qnn_attn_shared_tile(int dtype, int hd, int queries) {
    const int vec = dtype == QNN_DT_BF16 ? 8 : 4;
    if (hd <= 0 || hd % vec || hd > 1024) return -1;
    return on_tensor_cores(dtype, hd) ? 8 * column_tiles(hd, queries) : GEN_QT;
}

// groups: [n_groups][4] (first row, rows, begin, end): positions begin .. end - 1 lie in the same pages in all the group's rows, as far as a row
// still holds them; row_group: [B], a row's group or -1.  `most_rows`: rows of the largest group.  common_ranges / own_ranges: into how many ranges
// a group's common keys and a row's own keys are cut.  Scratch: part_o B * nq * (common_ranges + own_ranges) * hd floats, part_ml twice as many
// without hd; 16-byte aligned.  page_size: a power of two of at least 16; ring: a multiple of it, or 0.  slots, slot_len, page_table, groups and
// row_group are read before the kernel waits for the one launched in front of it on the stream: that one must not write them.
QNN_API int qnn_attn_decode_shared(const void* q, long long q_stride, int dtype, const void* k_pool, const void* v_pool, const int* page_table,
                                   int max_pages, int page_size, int ring, const int* slots, const int* slot_len, int B, const int* groups,
                                   int n_groups, int most_rows, const int* row_group, int nq, int nkv, int hd, float scale, float cap, int window,
                                   int common_ranges, int own_ranges, float* part_o, float* part_ml, void* out, long long out_stride,
                                   const float* slopes, const float* sinks, cudaStream_t st) {
    if (B <= 0) return 0;
    if (nkv <= 0 || nkv > 65535 || nq <= 0 || nq % nkv || n_groups < 0 || most_rows < 0 || common_ranges < 1 || own_ranges < 1) return QNN_ERR_ARGUMENT;
    if (page_size < 16 || (page_size & (page_size - 1)) || ring < 0 || ring % page_size) return QNN_ERR_ARGUMENT;
    if (ring > 0 && (window <= 0 || window > ring || ring / page_size > max_pages)) return QNN_ERR_ARGUMENT;   // a ring holds no more
    const int G = nq / nkv, esize = dtype == QNN_DT_BF16 ? 2 : 4;
    const int tile = qnn_attn_shared_tile(dtype, hd, most_rows * G);
    if (tile <= 0) return QNN_ERR_UNSUPPORTED;
    if ((q_stride * esize) % 16 || ((uintptr_t)q & 15) || ((uintptr_t)k_pool & 15) || ((uintptr_t)v_pool & 15) || ((uintptr_t)part_o & 15) ||
        ((uintptr_t)part_ml & 7) || ((uintptr_t)groups & 15))
        return QNN_ERR_ARGUMENT;
    const Cells cells = {page_table, max_pages, 31 - __builtin_clz((unsigned)page_size), ring / page_size, slots, slot_len, window};
    const int common_tiles = (most_rows * G + tile - 1) / tile;
    const Shared sh = {(const int4*)groups, row_group, n_groups, B, common_ranges, own_ranges, common_tiles};
    const long long items = (long long)n_groups * common_tiles * common_ranges + (long long)B * ((G + tile - 1) / tile) * own_ranges;
    if (items > 0x7fffffff || (long long)B * nq > 0x7fffffff) return QNN_ERR_UNSUPPORTED;
    float2* ml = (float2*)part_ml;
    int rc = QNN_ERR_UNSUPPORTED;
    if (on_tensor_cores(dtype, hd)) {
        const int nt = tile / 8;
#define QNN_MMA(HDV, NTV)                                                                                                                       \
    if (hd == HDV && nt == NTV)                                                                                                                  \
        rc = slopes != nullptr                                                                                                                   \
                 ? launch_mma<HDV, NTV, true>(q, q_stride, k_pool, v_pool, cells, sh, (int)items, nq, nkv, scale, cap, part_o, ml, slopes, st)   \
                 : launch_mma<HDV, NTV, false>(q, q_stride, k_pool, v_pool, cells, sh, (int)items, nq, nkv, scale, cap, part_o, ml, slopes, st);
        QNN_MMA(64, 1) QNN_MMA(64, 2) QNN_MMA(64, 4) QNN_MMA(128, 1) QNN_MMA(128, 2) QNN_MMA(128, 4) QNN_MMA(256, 1) QNN_MMA(256, 2)
#undef QNN_MMA
    } else {
#define QNN_GENERIC(T, DPLV) \
    launch_generic<T, DPLV>(q, q_stride, k_pool, v_pool, cells, sh, (int)items, nq, nkv, hd, scale, cap, part_o, ml, slopes, st)
        if (dtype == QNN_DT_BF16) rc = hd <= 64 ? QNN_GENERIC(bf16, 2) : (hd <= 256 ? QNN_GENERIC(bf16, 8) : QNN_GENERIC(bf16, 32));
        else rc = hd <= 64 ? QNN_GENERIC(float, 2) : (hd <= 256 ? QNN_GENERIC(float, 8) : QNN_GENERIC(float, 32));
#undef QNN_GENERIC
    }
    if (rc) return rc;
    return dtype == QNN_DT_BF16 ? launch_join<bf16>(part_o, ml, out, out_stride, B, nq, hd, common_ranges, own_ranges, row_group, slots, sinks, st)
                                : launch_join<float>(part_o, ml, out, out_stride, B, nq, hd, common_ranges, own_ranges, row_group, slots, sinks, st);
}
