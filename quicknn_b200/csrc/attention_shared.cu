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
// per kv head; keys are walked in tiles of 16 positions.  An item leaves (m, l, O) in scratch (m in units of log2), and a second kernel joins
// a row's items in ascending order: results depend on the numbers of ranges, not on what runs when.
//
// Bounds, on one B200: memory where keys are many (128 rows of 16 kv heads of 128 behind 6144 common keys, up to 1500 of their own each: 143 us
// for 910 MB, the kernel of the own keys at 6.5 TB/s; 16 groups of 4 rows, window 4096, 8 kv heads of 256: 91 us,
// 6.0 TB/s), else the chain of dependent reads in front of the first key (slot, length, page, query) and the two launches:
// 4 rows of 4 kv heads of 256 behind 448 keys 5.5 us, 8 rows behind 7936 keys 13.4 (5.8 of bytes).
#include "attention_generic.cuh"
#include "attention_shared.cuh"
#include "tcgen05.cuh"

using namespace qnn;
using namespace qnn::shared;

namespace {

// The page ids of an item's keys, pages from that of its first position on; returns the number of that page.
__device__ __forceinline__ int load_pages(const Item& it, const Cells& c, int* pages) {
    const int first = it.position(it.t0) >> c.page_shift, last = it.position(it.t1 - 1) >> c.page_shift;
    const int* row = c.page_table + (size_t)it.slot * c.max_pages;
    for (int u = threadIdx.x; u <= last - first; u += blockDim.x) {
        const int p = first + u;
        pages[u] = row[c.ring_pages > 0 ? p % c.ring_pages : p];
    }
    return first;
}

// ---- tensor cores, bfloat16 -------------------------------------------------------------------------------------------------
// As in attention_decode_mma.cu the keys fill the 16-row side of mma.m16n8k16 and queries the 8-column side,
//     S^T[16 keys x 8 q] = K Q^T,    O^T[hd x 8 q] += V^T P^T,
// here with NT column tiles (8 NT queries) for every fragment of K and V that ldmatrix brings.  A warp walks its own tiles of 16 keys: one
// lane asks the copy engine for them (a tile lies within a page; boxes of 64 elements x 16 positions, 128-byte swizzle, so that ldmatrix does
// not conflict), STAGES deep, an mbarrier each: two, so that 8, 6 and 3 CTAs of head size 64, 128 and 256 fit an SM (three stages, 8, 4 and 2:
// 11 groups of 82 rows with up to 26 keys of their own, 4 kv heads of 128 45 us instead of 38; 14 of 74 with up to 81, 8 kv heads 95 instead of
// 81; long walks the same).  (Rows copied one by one to padded rows, without a tensor map: 16 x 4 rows under a window of 4096 126 us instead of
// 93; cp.async by every lane 114.)  Nothing but the last merge is shared between the warps of a CTA.  P^T is the transpose of S^T's accumulator, eight by eight (movmatrix).  The exponentials are taken against a reference that is raised only when a score
// exceeds it by more than 8 (in log2): the stale reference cancels in the division, P stays below 2^8.
constexpr float REFERENCE_STEP = 8.f;
constexpr int WARPS = 2, STAGES = 2;

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

// The walk of one item.  smem: the warps' rings, which the merge reuses, then the barriers, then the page ids.
template <int HD>
struct Layout {
    static constexpr int TILE_BYTES = TILE * HD * 2, WARP_BYTES = STAGES * 2 * TILE_BYTES;
    static __host__ __device__ constexpr int merge_bytes(int nt) { return WARPS * 8 * nt * (HD + 2) * 4; }
    static __host__ __device__ constexpr int ring_bytes(int nt) { return WARPS * WARP_BYTES > merge_bytes(nt) ? WARPS * WARP_BYTES : (merge_bytes(nt) + 15) / 16 * 16; }
    static constexpr int BARRIERS = WARPS * STAGES * 8;
};

template <int HD, int NT, bool BIAS>
__device__ __forceinline__ void walk(const Item& it, int queries, const CUtensorMap& map, KV kv, const bf16* __restrict__ q, size_t q_stride,
                                     const Cells& cells, const Shared& sh, int kh, int nq, int nkv, const Scores& sc, float* __restrict__ part_o,
                                     float2* __restrict__ part_ml, int* __restrict__ status, unsigned char* smem, const int* pages, int first_page,
                                     unsigned bars) {
    using L = Layout<HD>;
    constexpr int KSTEPS = HD / 16, QT = 8 * NT;
    const int G = nq / nkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const unsigned ring = tc::smem_u32(smem) + warp * L::WARP_BYTES, bar0 = bars + warp * STAGES * 8;
    const int my_tiles = it.t1 - it.t0 > warp ? (it.t1 - it.t0 - warp + WARPS - 1) / WARPS : 0;

    const auto fetch = [&](int n) {                           // one lane
        const int p = it.position(it.t0 + warp + n * WARPS), s = n % STAGES;
        const int y = ((pages[(p >> cells.page_shift) - first_page] * nkv + kh) << cells.page_shift) + (p & ((1 << cells.page_shift) - 1));
        const unsigned kst = ring + s * 2 * L::TILE_BYTES, bar = bar0 + s * 8;
        tc::mbar_expect_tx(bar, 2 * L::TILE_BYTES);
#pragma unroll
        for (int d = 0; d < HD / 64; ++d) load_rows(kst + d * TILE * 128, &map, bar, d * 64, y, kv.k);
#pragma unroll
        for (int d = 0; d < HD / 64; ++d) load_rows(kst + L::TILE_BYTES + d * TILE * 128, &map, bar, d * 64, y, kv.v);
    };
    if (tc::elect_one())
        for (int n = 0; n < STAGES && n < my_tiles; ++n) fetch(n);

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
                    sl = sc.slopes[kh * G + mm % G] * LOG2E;
                    const int slot = cells.slots[it.row0 + mm / G];
                    nw = slot >= 0 ? cells.slot_len[slot] - 1 : 0;
                }
                (e ? slope1[nt] : slope0[nt]) = sl;
                (e ? newest1[nt] : newest0[nt]) = nw;
            }
        }
    }
    const float k1 = sc.cap > 0.f ? sc.scale / sc.cap : sc.scale * LOG2E, k2 = sc.cap * LOG2E;
    for (int n = 0; n < my_tiles; ++n) {
        const int s_at = n % STAGES;
        if (!tc::mbar_wait_warp(bar0 + s_at * 8, (n / STAGES) & 1)) {
            if (lane == 0) atomicOr(status, 512);
            // what else was asked for: wait for it, within the limit, before the memory is used again
            for (int i = n; i < my_tiles && i < n + STAGES; ++i) (void)tc::mbar_wait_warp(bar0 + (i % STAGES) * 8, (i / STAGES) & 1);
            break;
        }
        const int base = it.position(it.t0 + warp + n * WARPS);
        const unsigned kst = ring + s_at * 2 * L::TILE_BYTES, vst = kst + L::TILE_BYTES;
        const bool v_lo = base + g >= it.lo && base + g < it.hi, v_hi = base + g + 8 >= it.lo && base + g + 8 < it.hi;
        if (base < it.lo || base + TILE > it.hi) {
            // positions that do not count: their weights are zero, but zero times what an unused cell holds need not be
            unsigned char* v = smem + (vst - tc::smem_u32(smem));
            for (int i = lane; i < TILE * HD / 8; i += 32) {
                const int r = i / 8 % TILE;                   // 16-byte piece i: block i / (8 TILE), row, piece of the row
                if (base + r < it.lo || base + r >= it.hi) *reinterpret_cast<uint4*>(v + i * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // before the copy engine writes here again
            __syncwarp();
        }
        float s[NT][4], s2[NT][4];                            // two chains of products
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[nt][j] = s2[nt][j] = 0.f;
        {
            const int row = lane & 15, half = lane >> 4;
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks) {
                uint32_t a[4];
                ldmatrix_x4(a, kst + (ks / 4) * (TILE * 128) + row * 128 + ((((ks % 4) * 2 + half) ^ (row & 7)) << 4));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816(ks % 2 ? s2[nt] : s[nt], a, qf[nt][ks][0], qf[nt][ks][1]);
            }
        }
        // s[nt][0], [1]: key base + g, queries 2t, 2t + 1; [2], [3]: key base + g + 8
        bool above = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x = (s[nt][j] + s2[nt][j]) * k1;
                if (sc.cap > 0.f) x = k2 * tanh_approx(x);
                if (BIAS) x -= ((j & 1) ? slope1[nt] : slope0[nt]) * (float)(((j & 1) ? newest1[nt] : newest0[nt]) - (base + g + (j < 2 ? 0 : 8)));
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
                // -inf only before the first key (a score of -inf counts as no key)
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
            pb[nt][0] = transposed_8x8(tc::pack_bf16(a0, a1));
            pb[nt][1] = transposed_8x8(tc::pack_bf16(a2, a3));
        }
        {
            const int row = (lane & 7) + ((lane >> 4) << 3), sub = (lane >> 3) & 1;
#pragma unroll
            for (int mt = 0; mt < KSTEPS; ++mt) {
                uint32_t a[4];
                ldmatrix_x4_trans(a, vst + (mt / 4) * (TILE * 128) + row * 128 + ((((mt % 4) * 2 + sub) ^ (row & 7)) << 4));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816(o[nt][mt], a, pb[nt][0], pb[nt][1]);
            }
        }
        __syncwarp();                                         // everybody has read the stage: it may be filled again
        if (n + STAGES < my_tiles && tc::elect_one()) fetch(n + STAGES);
    }
    __syncthreads();
    // the warps' states through shared memory, [warp][query][HD + 2], joined in warp order
    float* ms = reinterpret_cast<float*>(smem);
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
    // lane m has query m's weights and place; then a warp per query, several on their way
    float coef[WARPS];
    size_t at = 0;
    if (lane < queries) {
        float mm = -CUDART_INF_F, ll = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, ms[((size_t)w * QT + lane) * ROW + HD]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float mw = ms[((size_t)w * QT + lane) * ROW + HD], lw = ms[((size_t)w * QT + lane) * ROW + HD + 1];
            coef[w] = mw == -CUDART_INF_F ? (lw != lw ? lw : 0.f) : exp2_fast(mw - mm);
            ll += coef[w] * lw;
        }
        at = part_of(it, sh, it.query0 + lane, kh, G, nq);
        if (warp == 0) part_ml[at] = make_float2(mm, ll);
    }
#pragma unroll 4
    for (int m = warp; m < queries; m += WARPS) {
        float c[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) c[w] = __shfl_sync(0xffffffffu, coef[w], m);
        float* dst = part_o + __shfl_sync(0xffffffffu, (unsigned long long)at, m) * HD;
#pragma unroll
        for (int d = lane * 2; d < HD; d += 64) {
            float2 acc = make_float2(0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float2 v = *reinterpret_cast<const float2*>(ms + ((size_t)w * QT + m) * ROW + d);
                acc.x += c[w] * v.x;
                acc.y += c[w] * v.y;
            }
            *reinterpret_cast<float2*>(dst + d) = acc;
        }
    }
}

// Items: those of C first (group, tile of queries, range; the range fastest), then the rows' own (row, tile of heads, range).  NT: column tiles
// of an item of C; a row's own heads take one where they fit it.
// BESIDE: the kernel in front is that of the groups' common keys (attention_shared_tcgen05.cu), which nothing here depends on.  Its CTAs have
// all waited for what is in front of them before this kernel can start, so the queries are there and the scratch is free.  One CTA waits
// for it at its end, so that this kernel is over only when that one is.
template <int HD, int NT, bool BIAS, bool BESIDE>
__global__ void __launch_bounds__(WARPS * 32)
attn_shared_mma_kernel(const __grid_constant__ CUtensorMap map, const KV kv, const bf16* __restrict__ q, size_t q_stride,
                       const Cells cells, const Shared sh, int common_items, int own_tile, int nq, int nkv, const Scores sc,
                       float* __restrict__ part_o, float2* __restrict__ part_ml, int* __restrict__ status) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const unsigned bars = tc::smem_u32(smem) + Layout<HD>::ring_bytes(NT);
    int* pages = reinterpret_cast<int*>(smem + Layout<HD>::ring_bytes(NT) + Layout<HD>::BARRIERS);
    const int kh = blockIdx.y, G = nq / nkv;
    const bool own = (int)blockIdx.x >= common_items;
    if (threadIdx.x < WARPS * STAGES) tc::mbar_init(bars + threadIdx.x * 8, 1);
    // slots, lengths, page tables and groups come from the host before the step: they are read before the wait for the kernel in front
    Item it;
    int tile;
    if (own) {
        const int own_tiles = (G + own_tile - 1) / own_tile, x = (int)blockIdx.x - common_items, rest = x / sh.own_ranges;
        tile = own_tile;
        it = own_item(sh, cells, rest / own_tiles, rest % own_tiles, x % sh.own_ranges, own_tile);
    } else {
        const int rest = blockIdx.x / sh.common_ranges;
        tile = 8 * NT;
        it = common_item(sh, cells, rest / sh.common_tiles, rest % sh.common_tiles, blockIdx.x % sh.common_ranges, 8 * NT);
    }
    const int queries = min(tile, it.rows * G - it.query0);
    int first_page = 0;
    if (it.t0 < it.t1) first_page = load_pages(it, cells, pages);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    if (!BESIDE) pdl_wait();
    const bool last = BESIDE && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1;
    if (queries <= 0) {
        if (last) pdl_wait();
        return;
    }
    if (it.t0 >= it.t1) {                                     // a range without keys
        for (int m = threadIdx.x; m < queries; m += blockDim.x) part_ml[part_of(it, sh, it.query0 + m, kh, G, nq)] = make_float2(-CUDART_INF_F, 0.f);
        if (last) pdl_wait();
        return;
    }
    if (NT > 1 && own && own_tile == 8)
        walk<HD, 1, BIAS>(it, queries, map, kv, q, q_stride, cells, sh, kh, nq, nkv, sc, part_o, part_ml, status, smem, pages, first_page, bars);
    else
        walk<HD, NT, BIAS>(it, queries, map, kv, q, q_stride, cells, sh, kh, nq, nkv, sc, part_o, part_ml, status, smem, pages, first_page, bars);
    if (last) pdl_wait();
}

// ---- any head size, float32 or bfloat16 ----------------------------------------------------------------------------------------
// Tiles of 32 keys as float32 in shared memory (rows an odd number of 16-byte pieces apart).  A warp keeps GEN_Q queries: a lane forms their
// scores with one key, the weights go to shared memory, and then the lanes take the head's elements, so that what is read of K and V serves
// all the warp's queries.  Exact exponentials and tanh in float32.  Bound by instructions (half of them products, four for each row of 16 bytes read)
// and the wait for a tile, which no other is fetched behind: six groups of 16 rows, 16 heads of 64 on 2 kv heads, 2112 keys 64 us (11 of
// float32 arithmetic); three groups of 5 rows, 6 heads of 24 on one, 960 keys 8.1.  (Four pieces of keys and values asked for at once: 90 us, for
// what it adds in instructions.)  bfloat16 at other head sizes than the tensor cores': 6 heads of 40 on 2, 32 rows, 2048 keys 18 us; 8 heads of 96 on 4,
// 32 rows, 2048 keys 50; 16 heads of 576 on one, 8 rows, 4096 keys 319.  An item holds 16 queries, so a row's own keys cost what 16 queries' would.
// Above head size 256 an accumulator of 4 x 32 elements a lane does not fit 255 registers (444 bytes of spills in float32, 204 in bfloat16; 8 to 24
// bytes up to head size 64, where six CTAs an SM are asked for), and above 64 an SM holds one or two CTAs.
constexpr int GEN_WARPS = 4, GEN_Q = 4, GEN_QT = GEN_WARPS * GEN_Q;

__device__ __forceinline__ float redux_max(float x) {         // the largest of the warp's that is a number
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

template <typename T, int DPL>                                // elements of a head per lane, at most
__global__ void __launch_bounds__(GEN_WARPS * 32, DPL <= 2 ? 6 : 1)
attn_shared_generic_kernel(const T* __restrict__ q, size_t q_stride, const T* __restrict__ k_pool, const T* __restrict__ v_pool,
                           const Cells cells, const Shared sh, int nq, int nkv, int hd, int tile_keys, bool staged, float scale, float cap,
                           float* __restrict__ part_o, float2* __restrict__ part_ml, const float* __restrict__ slopes) {
    constexpr int VEC = Vec16<T>::N;
    extern __shared__ __align__(16) float sm[];
    const int kh = blockIdx.y, G = nq / nkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int common_items = sh.n_groups * sh.common_tiles * sh.common_ranges;
    Item it;
    if ((int)blockIdx.x < common_items) {
        const int rest = blockIdx.x / sh.common_ranges;
        it = common_item(sh, cells, rest / sh.common_tiles, rest % sh.common_tiles, blockIdx.x % sh.common_ranges, GEN_QT);
    } else {
        const int own_tiles = (G + GEN_QT - 1) / GEN_QT, x = (int)blockIdx.x - common_items, rest = x / sh.own_ranges;
        it = own_item(sh, cells, rest / own_tiles, rest % own_tiles, x % sh.own_ranges, GEN_QT);
    }
    const int queries = min(GEN_QT, it.rows * G - it.query0);
    const int pitch = (hd / 4 | 1) * 4;
    float* sk = sm;
    float* sv = sk + tile_keys * pitch;
    float* sq = sv + tile_keys * pitch;                       // [GEN_QT][hd], times the scale; zeros for queries that are not there
    float4* sw = reinterpret_cast<float4*>(sq + GEN_QT * hd) + warp * 32;      // the warp's weights: key, then query
    int* pages = reinterpret_cast<int*>(reinterpret_cast<float4*>(sq + GEN_QT * hd) + GEN_WARPS * 32);      // the item's page ids, where there is room
    int first_page = 0;
    if (staged && queries > 0 && it.t0 < it.t1) first_page = load_pages(it, cells, pages);
    pdl_wait();
    if (queries <= 0) return;
    static_assert(GEN_Q == 4, "a float4 of weights");
    for (int i = threadIdx.x; i < GEN_QT * hd; i += blockDim.x) {
        const int m = it.query0 + i / hd, d = i % hd;
        sq[i] = i / hd < queries ? to_f(q[(size_t)(it.row0 + m / G) * q_stride + (size_t)(kh * G + m % G) * hd + d]) * scale : 0.f;
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
    const int chunks = hd / VEC, j0 = threadIdx.x / chunks, c0 = threadIdx.x % chunks, step_j = blockDim.x / chunks, step_c = blockDim.x % chunks;
    const int page_mask = (1 << cells.page_shift) - 1;
    for (int t = it.t0; t < it.t1; t += tile_keys / TILE) {
        const int n = min(tile_keys, (it.t1 - t) * TILE);
        __syncthreads();                                      // the tiles before have been read
        const int* table = cells.page_table + (size_t)it.slot * cells.max_pages;
        for (int j = j0, c = c0; j < n;) {
            const int p = it.position(t + j / TILE) + j % TILE;
            float* const kd = sk + j * pitch + c * VEC;
            float* const vd = sv + j * pitch + c * VEC;
            if (p >= it.lo && p < it.hi) {
                const int pn = p >> cells.page_shift, page = staged ? pages[pn - first_page] : table[cells.ring_pages > 0 ? pn % cells.ring_pages : pn];
                const size_t off = ((((size_t)page * nkv + kh) << cells.page_shift) + (p & page_mask)) * hd + c * VEC;
                Vec16<T> kv, vv;
                kv.load(k_pool + off);
                vv.load(v_pool + off);
                float a[VEC], b[VEC];
                kv.unpack(a);
                vv.unpack(b);
#pragma unroll
                for (int e = 0; e < VEC; e += 4) {
                    *reinterpret_cast<float4*>(kd + e) = make_float4(a[e], a[e + 1], a[e + 2], a[e + 3]);
                    *reinterpret_cast<float4*>(vd + e) = make_float4(b[e], b[e + 1], b[e + 2], b[e + 3]);
                }
            } else {                                          // zero weights, and zeros for them to meet
#pragma unroll
                for (int e = 0; e < VEC; e += 4) *reinterpret_cast<float4*>(vd + e) = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            c += step_c;
            j += step_j;
            if (c >= chunks) {
                c -= chunks;
                ++j;
            }
        }
        __syncthreads();
        const int pos = lane < n ? it.position(t + lane / TILE) + lane % TILE : 0;
        const bool valid = lane < n && pos >= it.lo && pos < it.hi;
        if (warp * GEN_Q >= queries) continue;                // (the warp still brings keys)
        float s[GEN_Q] = {0.f, 0.f, 0.f, 0.f}, w[GEN_Q];
        {
            const float* kr = sk + (valid ? lane : 0) * pitch;
            const float* qr = sq + warp * GEN_Q * hd;
#pragma unroll 4
            for (int d = 0; d < hd; d += 4) {
                const float4 k = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
                for (int i = 0; i < GEN_Q; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(qr + i * hd + d);
                    s[i] = fmaf(x.w, k.w, fmaf(x.z, k.z, fmaf(x.y, k.y, fmaf(x.x, k.x, s[i]))));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < GEN_Q; ++i) {
            s[i] = softcap_t<T>(s[i], cap) - slope[i] * (float)(newest[i] - pos);
            const float top = fmaxf(mx[i], redux_max(valid ? s[i] : -CUDART_INF_F));
            if (top > mx[i]) {                                // (the same in all lanes)
                const float keep = mx[i] == -CUDART_INF_F ? 0.f : fexp<T>(mx[i] - top);
                mx[i] = top;
                l[i] *= keep;
#pragma unroll
                for (int d = 0; d < DPL; ++d) o[i][d] *= keep;
            }
            w[i] = valid && (top != -CUDART_INF_F || s[i] != s[i]) ? fexp<T>(s[i] - top) : 0.f;
            l[i] += w[i];                                     // the lane's keys
        }
        sw[lane] = make_float4(w[0], w[1], w[2], w[3]);
        __syncwarp();
#pragma unroll 8
        for (int j = 0; j < n; ++j) {
            const float4 wj = sw[j];
#pragma unroll
            for (int d = 0; d < DPL; ++d) {
                const float v = lane + d * 32 < hd ? sv[j * pitch + lane + d * 32] : 0.f;
                o[0][d] = fmaf(wj.x, v, o[0][d]);
                o[1][d] = fmaf(wj.y, v, o[1][d]);
                o[2][d] = fmaf(wj.z, v, o[2][d]);
                o[3][d] = fmaf(wj.w, v, o[3][d]);
            }
        }
        __syncwarp();                                         // before the weights are written again
    }
#pragma unroll
    for (int i = 0; i < GEN_Q; ++i) {
        const int m = warp * GEN_Q + i;
        if (m >= queries) break;
        const size_t at = part_of(it, sh, it.query0 + m, kh, G, nq);
        l[i] = warp_sum(l[i]);
        if (l[i] > 0.f || l[i] != l[i])                       // (a NaN among the scores has to come out)
#pragma unroll
            for (int d = 0; d < DPL; ++d)
                if (lane + d * 32 < hd) part_o[at * hd + lane + d * 32] = o[i][d];
        if (lane == 0) part_ml[at] = make_float2(mx[i] * LOG2E, l[i]);
    }
}

// ---- the parts of a row joined ---------------------------------------------------------------------------------------------------
// JOIN_WARPS warps per (row, head): warp i adds parts i, i + JOIN_WARPS, ...; then the warps' sums in ascending order.  Weights are in the
// lanes' registers (part p: lane p % 32), the first parts are asked for before the weights are known.  Of parts without keys (l = 0) nothing counts.
constexpr int JOIN_WARPS = 8, MOST_PARTS = 128;

template <typename T, int PIECES>                             // pieces of 128 elements that a head has, at most
__global__ void __launch_bounds__(JOIN_WARPS * 32)
attn_shared_join_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, T* __restrict__ out, size_t out_stride, int nq, int hd,
                        const Shared sh, const int* __restrict__ slots, const float* __restrict__ sinks) {
    extern __shared__ __align__(16) float js[];               // [JOIN_WARPS][hd]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, S = sh.common_ranges, parts = S + sh.own_ranges;
    const int i = blockIdx.x, row = i / nq, h = i % nq;
    const int from = sh.group_of(row).y > 0 && slots[row] >= 0 ? 0 : S;      // a row of no group or no sequence has no part in C
    pdl_wait();
    const size_t at = (size_t)i * parts;
    float2 ml[MOST_PARTS / 32];
#pragma unroll
    for (int k = 0; k < MOST_PARTS / 32; ++k) {
        const int p = k * 32 + lane;
        ml[k] = p >= from && p < parts ? part_ml[at + p] : make_float2(-CUDART_INF_F, 0.f);
    }
    constexpr int AHEAD = PIECES <= 2 ? 8 : 4;
    float4 v[AHEAD][PIECES];
    const auto ask = [&](int p0) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int p = p0 + j * JOIN_WARPS;
#pragma unroll
            for (int k = 0; k < PIECES; ++k) {
                const int c = k * 128 + lane * 4;
                v[j][k] = p < parts && c < hd ? *reinterpret_cast<const float4*>(part_o + (at + p) * hd + c) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
    };
    ask(from + warp);
    float M = -CUDART_INF_F, sum = 0.f, w[MOST_PARTS / 32];
#pragma unroll
    for (int k = 0; k < MOST_PARTS / 32; ++k)
        if (ml[k].y != 0.f) M = fmaxf(M, ml[k].x);
    M = warp_max(M);
#pragma unroll
    for (int k = 0; k < MOST_PARTS / 32; ++k) {
        w[k] = ml[k].y != ml[k].y ? ml[k].y : (ml[k].y != 0.f ? exp2f(ml[k].x - M) : 0.f);       // a NaN among the scores has to come out
        sum += w[k] != 0.f ? w[k] * ml[k].y : 0.f;
    }
    sum = warp_sum(sum);
    const float all = sinks != nullptr ? sum + exp2f(sinks[h] * LOG2E - M) : sum;
    const float inverse = sum != 0.f ? 1.f / all : 0.f;
    float4 acc[PIECES];
#pragma unroll
    for (int k = 0; k < PIECES; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = from + warp; p0 < parts; p0 += AHEAD * JOIN_WARPS) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int p = p0 + j * JOIN_WARPS;
            float mine_w = 0.f;
#pragma unroll
            for (int k = 0; k < MOST_PARTS / 32; ++k) {
                const float x = __shfl_sync(0xffffffffu, w[k], p & 31);
                if (p >> 5 == k) mine_w = x;
            }
            if (mine_w != 0.f)
#pragma unroll
                for (int k = 0; k < PIECES; ++k) {
                    acc[k].x += mine_w * v[j][k].x;
                    acc[k].y += mine_w * v[j][k].y;
                    acc[k].z += mine_w * v[j][k].z;
                    acc[k].w += mine_w * v[j][k].w;
                }
        }
        if (p0 + AHEAD * JOIN_WARPS < parts) ask(p0 + AHEAD * JOIN_WARPS);
    }
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
        const int c = k * 128 + lane * 4;
        if (c < hd) *reinterpret_cast<float4*>(js + (size_t)warp * hd + c) = acc[k];
    }
    __syncthreads();
    for (int d = threadIdx.x; d < hd; d += blockDim.x) {
        float a = 0.f;
#pragma unroll
        for (int x = 0; x < JOIN_WARPS; ++x) a += js[(size_t)x * hd + d];
        out[(size_t)row * out_stride + (size_t)h * hd + d] = from_f<T>(a * inverse);
    }
}

// The same where a row has few parts: a thread per four elements of an output, which asks for all of them at once (a part that nobody has written is
// read all the same and does not count).  59,520 outputs of 64 from two parts: 46 us with a warp each, 13 so.
constexpr int FEW_PARTS = 8;

template <typename T, int PARTS>                              // at most
__global__ void __launch_bounds__(JOIN_WARPS * 32)
attn_shared_join_few_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, T* __restrict__ out, size_t out_stride, long long pieces, int nq,
                            int hd, const Shared sh, const int* __restrict__ slots, const float* __restrict__ sinks) {
    const long long x = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int chunks = hd / 4, S = sh.common_ranges, parts = S + sh.own_ranges;
    const bool mine = x < pieces;
    const long long i = mine ? x / chunks : 0;
    const int c = mine ? (int)(x - i * chunks) * 4 : 0, row = (int)(i / nq), h = (int)(i - (long long)row * nq);
    const int from = sh.group_of(row).y > 0 && slots[row] >= 0 ? 0 : S;      // a row of no group or no sequence has no part in C
    const float sink = sinks != nullptr ? sinks[h] * LOG2E : -CUDART_INF_F;
    pdl_wait();
    if (!mine) return;
    const size_t at = (size_t)i * parts;
    float2 ml[PARTS];
    float4 v[PARTS];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        ml[p] = p < parts ? part_ml[at + p] : make_float2(-CUDART_INF_F, 0.f);
        v[p] = p < parts ? *reinterpret_cast<const float4*>(part_o + (at + p) * hd + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float M = -CUDART_INF_F, sum = 0.f;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        if (p < from) ml[p] = make_float2(-CUDART_INF_F, 0.f);
        if (ml[p].y != 0.f) M = fmaxf(M, ml[p].x);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        const float w = ml[p].y != ml[p].y ? ml[p].y : (ml[p].y != 0.f ? exp2f(ml[p].x - M) : 0.f);   // a NaN among the scores has to come out
        if (w == 0.f) continue;
        sum += w * ml[p].y;
        acc.x += w * v[p].x;
        acc.y += w * v[p].y;
        acc.z += w * v[p].z;
        acc.w += w * v[p].w;
    }
    const float inverse = sum != 0.f ? 1.f / (sum + exp2f(sink - M)) : 0.f;
    T* dst = out + (size_t)row * out_stride + (size_t)h * hd + c;
    const float r[4] = {acc.x * inverse, acc.y * inverse, acc.z * inverse, acc.w * inverse};
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(tc::pack_bf16(r[0], r[1]), tc::pack_bf16(r[2], r[3]));
    } else {
        *reinterpret_cast<float4*>(dst) = make_float4(r[0], r[1], r[2], r[3]);
    }
}

bool on_tensor_cores(int dtype, int hd) { return dtype == QNN_DT_BF16 && (hd == 64 || hd == 128 || hd == 256); }

// Column tiles of an item for so many queries: 1 or 2.  (4, up to head size 128, were slower wherever they would have been taken: 18 queries, 8 kv
// heads of 128, 2048 keys 12.7 us against 9.9.)
int column_tiles(int queries) { return queries <= 8 ? 1 : 2; }

// Groups of more query rows than an item of the mma.sync kernel takes go to the 5th-generation tensor cores, where a CTA takes 128, if the work is
// enough for what a kernel of its own costs (3 to 4 us): `walks` walks (groups x kv heads) over `keys` keys, times the items beside one another
// that the queries would take here.  Both take the same time at 22,000 (128 queries of 256) to 100,000 (18 queries of 128).  us there and here,
// 4 kv heads of 256: 64 queries on 1024 keys 14.5 / 12.8, on 4096 17.3 / 25.2; 18 queries on 4096 16.6 / 12.5; 2 kv heads of 128: 64 queries on
// 2048 11.5 / 9.3; four groups of 24 queries, 8 kv heads of 128, 8192 keys 35 / 48.
constexpr int MANY_TILE = 128;
constexpr long long MANY_WORK = 50000;
bool many_rows(int dtype, int hd, int queries, long long walks, int keys) {
    return on_tensor_cores(dtype, hd) && queries > 16 && (queries + 15) / 16 * walks * keys >= MANY_WORK;
}

// Shared memory of a CTA of the mma.sync kernel: rings, barriers, and the page ids of an item, with room for all of a sequence's.  The 8, 6 and 3 CTAs
// an SM of head size 64, 128 and 256 fit up to page tables of 2500, 780 and 2150 pages (160,000, 50,000 and 137,000 positions); with longer ones
// fewer do.
template <int HD>
size_t mma_bytes(int nt, int max_pages) { return 1024 + Layout<HD>::ring_bytes(nt) + Layout<HD>::BARRIERS + ((size_t)max_pages + 2) * sizeof(int); }
constexpr size_t MMA_MOST_BYTES = 220 * 1024;

// Whether the tensor cores take these sizes.  Page tables of more than 38,000 pages (2.4 million positions) leave no room for the tiles: they go to
// the kernel for any head size, which then reads its page ids from the table.
bool takes_tensor_cores(int dtype, int hd, int max_pages) {
    if (!on_tensor_cores(dtype, hd)) return false;
    return (hd == 64 ? mma_bytes<64>(2, max_pages) : hd == 128 ? mma_bytes<128>(2, max_pages) : mma_bytes<256>(2, max_pages)) <= MMA_MOST_BYTES;
}

template <int HD, int NT, bool BIAS, bool BESIDE>
int launch_mma(const void* q, long long q_stride, const void* k_pool, const void* v_pool, long long pool_rows, const Cells& cells, const Shared& sh,
               int B, int nq, int nkv, const Scores& sc, float* part_o, float2* part_ml, int* status, cudaStream_t st) {
    const int G = nq / nkv, own_tile = G <= 8 ? 8 : 8 * NT;
    const long long common = BESIDE ? 0 : (long long)sh.n_groups * sh.common_tiles * sh.common_ranges, own = (long long)B * ((G + own_tile - 1) / own_tile) * sh.own_ranges;
    if (common + own > 0x7fffffff) return QNN_ERR_UNSUPPORTED;
    const size_t smem = mma_bytes<HD>(NT, cells.max_pages);
    CUtensorMap map;
    KV kv;
    if (const int rc = make_pools_map(&map, &kv, k_pool, v_pool, pool_rows, HD, TILE)) return rc;
    auto kern = attn_shared_mma_kernel<HD, NT, BIAS, BESIDE>;
    static OncePerDevice asked;
    if (const int rc = allow_shared(asked, kern, MMA_MOST_BYTES)) return rc;
    // (beside the kernel of the common keys also where the grid is larger than others are launched early with)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(common + own), nkv);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = (BESIDE && pdl_enabled()) || (pdl_enabled() && (common + own) * nkv <= pdl_max_grid()) ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, map, kv, (const bf16*)q, (size_t)q_stride, cells, sh, (int)common, own_tile, nq, nkv, sc,
                                             part_o, part_ml, status);
    return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

template <typename T, int DPL>
int launch_generic(const void* q, long long q_stride, const void* k_pool, const void* v_pool, const Cells& cells, const Shared& sh, int items, int nq,
                   int nkv, int hd, float scale, float cap, float* part_o, float2* part_ml, const float* slopes, cudaStream_t st) {
    const int keys = hd <= 512 ? 32 : 16;
    size_t smem = ((size_t)2 * keys * ((hd / 4) | 1) * 4 + (size_t)GEN_QT * hd + GEN_WARPS * 32 * 4) * sizeof(float);
    const size_t pages = ((size_t)cells.max_pages + 2) * sizeof(int);
    const bool staged = hd <= 256 && smem + pages <= 220 * 1024;
    if (staged) smem += pages;
    auto kern = attn_shared_generic_kernel<T, DPL>;
    static OncePerDevice asked;
    if (const int rc = allow_shared(asked, kern, 220 * 1024)) return rc;
    launch_pdl(kern, dim3(items, nkv), dim3(GEN_WARPS * 32), smem, st, (const T*)q, (size_t)q_stride, (const T*)k_pool, (const T*)v_pool, cells, sh, nq,
               nkv, hd, keys, staged, scale, cap, part_o, part_ml, slopes);
    return (int)cudaGetLastError();
}

template <typename T>
int launch_join(const float* part_o, const float2* part_ml, void* out, long long out_stride, int nq, int hd, const Shared& sh, const int* slots,
                const float* sinks, cudaStream_t st) {
    const int outputs = sh.B * nq, parts = sh.common_ranges + sh.own_ranges;
    if (parts <= FEW_PARTS) {
        const long long pieces = (long long)outputs * (hd / 4);
        const dim3 blocks((unsigned)((pieces + JOIN_WARPS * 32 - 1) / (JOIN_WARPS * 32)));
#define QNN_JOIN(PARTS)                                                                                                                          \
    launch_pdl(attn_shared_join_few_kernel<T, PARTS>, blocks, dim3(JOIN_WARPS * 32), 0, st, part_o, part_ml, (T*)out, (size_t)out_stride, pieces, nq, hd, sh, \
               slots, sinks)
        if (parts <= 2) QNN_JOIN(2);
        else if (parts <= 4) QNN_JOIN(4);
        else QNN_JOIN(FEW_PARTS);
#undef QNN_JOIN
        return (int)cudaGetLastError();
    }
    const size_t smem = (size_t)JOIN_WARPS * hd * sizeof(float);
#define QNN_JOIN(PIECES)                                                                                                                         \
    launch_pdl(attn_shared_join_kernel<T, PIECES>, dim3(outputs), dim3(JOIN_WARPS * 32), smem, st, part_o, part_ml, (T*)out, (size_t)out_stride, nq, hd, sh, \
               slots, sinks)
    if (hd <= 128) QNN_JOIN(1);
    else if (hd <= 256) QNN_JOIN(2);
    else QNN_JOIN(8);
#undef QNN_JOIN
    return (int)cudaGetLastError();
}

}  // namespace

// Queries that one item takes (what the number of items, and with it the choice of ranges, goes by), or a negative number for a head
// size that is not taken.  queries: rows x query heads per kv head of the largest group; walks: groups x kv heads; keys: of a group, at most.
QNN_API int qnn_attn_shared_tile(int dtype, int hd, int queries, int walks, int keys) {
    const int vec = dtype == QNN_DT_BF16 ? 8 : 4;
    if (hd <= 0 || hd % vec || hd > 1024) return -1;
    return many_rows(dtype, hd, queries, walks, keys) ? MANY_TILE : (on_tensor_cores(dtype, hd) ? 8 * column_tiles(queries) : GEN_QT);
}

// groups: [n_groups][4] (first row, rows, begin, end): positions begin .. end - 1 lie in the same pages in all the group's rows, as far as a row
// still holds them; row_group: [B], a row's group or -1.  `most_rows`: rows of the largest group; `most_keys`: positions of the
// longest (a matter of speed).  common_ranges / own_ranges: into how many ranges
// a group's common keys and a row's own keys are cut.  Scratch: part_o B * nq * (common_ranges + own_ranges) * hd floats, part_ml twice as many
// without hd; 16-byte aligned.  pool_pages: pages of
// the pools; status: as in qnn_gemm_tcgen05 (bit 512: keys or values did not arrive).  page_size: a power of two of at least 16; ring: a
// multiple of it, or 0.  slots, slot_len, page_table, groups and row_group are read before the kernel waits for the one launched in front of
// it on the stream: that one must not write them.
QNN_API int qnn_attn_decode_shared(const void* q, long long q_stride, int dtype, const void* k_pool, const void* v_pool, const int* page_table,
                                   int max_pages, int page_size, int ring, const int* slots, const int* slot_len, int B, const int* groups,
                                   int n_groups, int most_rows, int most_keys, const int* row_group, int nq, int nkv, int hd, float scale, float cap, int window,
                                   int common_ranges, int own_ranges, float* part_o, float* part_ml, void* out, long long out_stride,
                                   const float* slopes, const float* sinks, long long pool_pages, int* status, cudaStream_t st) {
    if (B <= 0) return 0;
    if (nkv <= 0 || nkv > 65535 || nq <= 0 || nq % nkv || n_groups < 0 || most_rows < 0 || most_keys < 0 || common_ranges < 1 || own_ranges < 1 ||
        common_ranges + own_ranges > MOST_PARTS)
        return QNN_ERR_ARGUMENT;
    if (n_groups > 0 && most_rows < 1) return QNN_ERR_ARGUMENT;
    if (page_size < 16 || (page_size & (page_size - 1)) || ring < 0 || ring % page_size) return QNN_ERR_ARGUMENT;
    if (ring > 0 && (window <= 0 || window > ring || ring / page_size > max_pages)) return QNN_ERR_ARGUMENT;   // a ring holds no more
    const int G = nq / nkv, esize = dtype == QNN_DT_BF16 ? 2 : 4;
    const bool tensor = takes_tensor_cores(dtype, hd, max_pages);
    const bool many = tensor && n_groups > 0 && page_size >= 64 && many_rows(dtype, hd, most_rows * G, (long long)n_groups * nkv, most_keys);
    const int tile = many ? MANY_TILE : tensor ? 8 * column_tiles(most_rows * G) : on_tensor_cores(dtype, hd) ? GEN_QT : qnn_attn_shared_tile(dtype, hd, most_rows * G, 0, 0);
    if (tile <= 0) return QNN_ERR_UNSUPPORTED;
    if ((q_stride * esize) % 16 || ((uintptr_t)q & 15) || ((uintptr_t)k_pool & 15) || ((uintptr_t)v_pool & 15) || ((uintptr_t)part_o & 15) ||
        ((uintptr_t)part_ml & 7) || ((uintptr_t)groups & 15) || ((uintptr_t)out & 15) || (out_stride * esize) % 16)
        return QNN_ERR_ARGUMENT;
    const Cells cells = {page_table, max_pages, 31 - __builtin_clz((unsigned)page_size), ring / page_size, slots, slot_len, window};
    const int common_tiles = (most_rows * G + tile - 1) / tile;
    const Shared sh = {(const int4*)groups, row_group, n_groups, B, common_ranges, own_ranges, common_tiles, most_rows};
    const int own_tile = tensor ? 8 : GEN_QT;
    const long long items = (long long)n_groups * common_tiles * common_ranges + (long long)B * ((G + own_tile - 1) / own_tile) * own_ranges;
    const long long pool_rows = pool_pages * nkv * page_size;         // of the pools as matrices of head rows
    if (items > 0x7fffffff || (long long)B * nq > 0x7fffffff || pool_rows <= 0 || pool_rows > 0x7fffffff) return QNN_ERR_UNSUPPORTED;
    const Scores sc = {scale, cap, slopes};
    float2* ml = (float2*)part_ml;
    int rc = QNN_ERR_UNSUPPORTED;
    if (tensor) {
        if (many) {
            const SharedLaunch a = {q, q_stride, k_pool, v_pool, pool_rows, cells, sh, nq, nkv, hd, sc, part_o, ml, status};
            if (const int err = launch_common_tcgen05(a, st)) return err;
        }
        const int nt = many ? column_tiles(G) : tile / 8;
#define QNN_MMA_AS(HDV, NTV, BIAS, BESIDE) launch_mma<HDV, NTV, BIAS, BESIDE>(q, q_stride, k_pool, v_pool, pool_rows, cells, sh, B, nq, nkv, sc, part_o, ml, status, st)
#define QNN_MMA(HDV, NTV)                                                                                                                       \
    if (hd == HDV && nt == NTV)                                                                                                                  \
        rc = slopes != nullptr ? (many ? QNN_MMA_AS(HDV, NTV, true, true) : QNN_MMA_AS(HDV, NTV, true, false))                                   \
                               : (many ? QNN_MMA_AS(HDV, NTV, false, true) : QNN_MMA_AS(HDV, NTV, false, false));
        QNN_MMA(64, 1) QNN_MMA(64, 2) QNN_MMA(128, 1) QNN_MMA(128, 2) QNN_MMA(256, 1) QNN_MMA(256, 2)
#undef QNN_MMA
#undef QNN_MMA_AS
    } else {
#define QNN_GENERIC(T, DPLV) \
    launch_generic<T, DPLV>(q, q_stride, k_pool, v_pool, cells, sh, (int)items, nq, nkv, hd, scale, cap, part_o, ml, slopes, st)
        if (dtype == QNN_DT_BF16) rc = hd <= 32 ? QNN_GENERIC(bf16, 1) : hd <= 64 ? QNN_GENERIC(bf16, 2) : (hd <= 256 ? QNN_GENERIC(bf16, 8) : QNN_GENERIC(bf16, 32));
        else rc = hd <= 32 ? QNN_GENERIC(float, 1) : hd <= 64 ? QNN_GENERIC(float, 2) : (hd <= 256 ? QNN_GENERIC(float, 8) : QNN_GENERIC(float, 32));
#undef QNN_GENERIC
    }
    if (rc) return rc;
    return dtype == QNN_DT_BF16 ? launch_join<bf16>(part_o, ml, out, out_stride, nq, hd, sh, slots, sinks, st)
                                : launch_join<float>(part_o, ml, out, out_stride, nq, hd, sh, slots, sinks, st);
}
