// The keys that many rows hold in the same pages, on the 5th-generation tensor cores: the items of C of attention_shared.cu for groups with more
// query rows (rows x query heads of a kv head) than a warp's registers hold.  bfloat16, head sizes 64, 128 and 256, pages of whole 64
// positions.
//
// A CTA owns up to 128 query rows of one group and kv head and a range of C, and leaves (m, l, O) of each row in scratch.  The roles and the
// pipeline are those of attention_prefill_tcgen05.cu, twelve warps: a producer of K (pairs of pages, one operand of 128 keys), one of V
// (a page at a time), an issuer of S = Q K^T (Q from tensor memory), one of O += P V, and two softmax groups of four warps (thread = query
// row) that take the lower and the upper page of each pair.  What differs: the query rows lie apart (row, head), so each thread brings its
// own from global memory to tensor memory; every key counts for every row, so nothing is masked but the half of a last pair that is not
// there; results go out as float32 with their reference and sum.
// With a softcap up to 70 the exponentials are taken against 0 (FIXED), else against a running maximum that both groups share.  Weights are rounded
// to bfloat16 before they meet V, as in the library's other attention on tensor cores: up to 2^-8 of a weight, as the results are.
// Bounds: the softmax between two products of a pair (special functions, two a score with a softcap, some of the exponentials on the FMA pipe
// instead: 54 % of their pipe; tensor cores 35 %), and about 8 us a CTA in front of its first and behind its last page.  32 CTAs over 6144 keys
// (128 rows, 2 heads of 128 on each of 16 kv heads) 83 us beside 134 of the rows' own keys, which hide it; 64 queries on 4096 keys of 4 kv heads of
// 256 17 us.  The keys themselves come from memory once per 128 query rows.
// Every mbarrier wait is bounded in time; on expiry a status word is set and the CTA winds down.
#include "attention_shared.cuh"
#include "capped_exp2.cuh"
#include "tcgen05.cuh"
#include <math_constants.h>

using namespace qnn;
using namespace qnn::shared;
using namespace qnn::tc;

namespace {

constexpr int BM = 128, BN = 64, UMMA_K = 16, MAX_STAGES = 6, THREADS = 384;
constexpr int P_BYTES = BM * BN * 2;
constexpr int S_COL = 0, O_COL = 128;         // tensor-memory columns of S (two halves of 64) and of O; Q follows O
constexpr float STEP = 8.f;                   // how far (in e) a maximum may rise before O is rescaled
// Depth of the rings.  Up to head size 128 they leave room for a CTA of the rows' own keys on the same SM.
__host__ __device__ constexpr int k_stages(int hd) { return hd >= 128 ? 2 : 4; }                        // pairs of pages
__host__ __device__ constexpr int v_stages(int hd) { return hd >= 256 ? 2 : (hd >= 128 ? 3 : 6); }       // pages

// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void umma_a_tmem(unsigned tmem_d, unsigned tmem_a, uint64_t bdesc, unsigned idesc, unsigned accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
struct __align__(8) Barriers {
    uint64_t q_tmem;          // Q is in tensor memory
    uint64_t k_full[MAX_STAGES], k_empty[MAX_STAGES];
    uint64_t v_full[MAX_STAGES], v_empty[MAX_STAGES];
    uint64_t s_ready;         // S of a pair is complete
    uint64_t s_free;          // the softmax warps have read it
    uint64_t p_ready[2];      // P of a page is in shared memory and O has been corrected
    uint64_t pv_done[2];      // O += P V of a page has completed
    uint64_t max_ready[4];    // both groups' maxima of a pair are there (one for each 32 rows)
    uint32_t tmem_base, failed;
    float row_max[2][2][BM];  // what the groups tell each other: by pair parity and group
};
__device__ __forceinline__ bool has_failed(Barriers* b) { return *reinterpret_cast<volatile uint32_t*>(&b->failed) != 0; }

template <int HD, bool FIXED>
__global__ void __launch_bounds__(THREADS)
attn_shared_tcgen05_kernel(const __grid_constant__ CUtensorMap map, const KV kv, const bf16* __restrict__ q, size_t q_stride,
                           const Cells cells, const Shared sh, int nq, int nkv, const Scores sc, float* __restrict__ part_o, float2* __restrict__ part_ml,
                           int* __restrict__ status) {
    constexpr int KS = k_stages(HD), VS = v_stages(HD);
    constexpr int KP_BYTES = 2 * BN * HD * 2, V_BYTES = BN * HD * 2;
    constexpr int Q_COL = O_COL + HD;                                // HD / 2 columns, two bfloat16 each
    constexpr int TMEM_COLS = HD > 64 ? 512 : 256;
    constexpr int BLOCKS = HD / 64, Q_GROUPS = BLOCKS > 1 ? 2 : 1;    // both softmax groups bring queries, alternate blocks of 64 elements
    static_assert(BM * HD * 4 <= KS * KP_BYTES, "the results are staged in the K ring");
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* sK = smem;
    unsigned char* sV = sK + KS * KP_BYTES;
    unsigned char* sP = sV + VS * V_BYTES;
    Barriers* bars = reinterpret_cast<Barriers*>(sP + 2 * P_BYTES);
    unsigned dynamic_bytes;
    asm("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dynamic_bytes));
    if ((unsigned)(reinterpret_cast<unsigned char*>(bars + 1) - smem_raw) > dynamic_bytes) {       // (at head size 256 there is no room to align it)
        if (threadIdx.x == 0) atomicOr(status, 256);
        pdl_wait();
        return;
    }
    const int kh = blockIdx.y, G = nq / nkv, rest = blockIdx.x / sh.common_ranges;
    const Item it = common_item(sh, cells, rest / sh.common_tiles, rest % sh.common_tiles, blockIdx.x % sh.common_ranges, BM, BN / TILE);
    const int queries = min(BM, it.rows * G - it.query0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nt = (it.t1 - it.t0) / (BN / TILE), np = (nt + 1) / 2; // pages and pairs of them
    if (queries <= 0 || nt <= 0) {                                   // before any barrier or tensor memory
        pdl_wait();                                                  // (what follows in the stream waits for this kernel, not for those before it)
        for (int m = threadIdx.x; m < queries; m += THREADS) part_ml[part_of(it, sh, it.query0 + m, kh, G, nq)] = make_float2(-CUDART_INF_F, 0.f);
        return;
    }
    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&bars->q_tmem), 4 * Q_GROUPS);
        for (int s = 0; s < KS; ++s) {
            mbar_init(smem_u32(&bars->k_full[s]), 1);
            mbar_init(smem_u32(&bars->k_empty[s]), 1);
        }
        for (int s = 0; s < VS; ++s) {
            mbar_init(smem_u32(&bars->v_full[s]), 1);
            mbar_init(smem_u32(&bars->v_empty[s]), 1);
        }
        mbar_init(smem_u32(&bars->s_ready), 1);
        mbar_init(smem_u32(&bars->s_free), 8);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&bars->p_ready[i]), 4);
            mbar_init(smem_u32(&bars->pv_done[i]), 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&bars->max_ready[i]), 2);
        bars->failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = bars->tmem_base;
    pdl_wait();

    const int quarter = warp & 3, group = (warp >= 6 && warp < 10) ? 1 : 0;
    const int rloc = quarter * 32 + lane;                            // query of the tile = tensor-memory lane
    const unsigned lane_base = tmem + ((unsigned)(quarter * 32) << 16);
    const int* const table = cells.page_table + (size_t)it.slot * cells.max_pages;
    // the pools' row of page-sized tile j of the range (behind the last: the last again)
    const auto tile_row = [&](int j) {
        const int p = it.position(it.t0) + min(j, nt - 1) * BN, n = p >> cells.page_shift;
        return ((table[cells.ring_pages > 0 ? n % cells.ring_pages : n] * nkv + kh) << cells.page_shift) + (p & ((1 << cells.page_shift) - 1));
    };
    const auto give_up = [&](int bit) {
        atomicOr(status, bit);
        bars->failed = 1;
    };

    if (warp == 0) {
        if (elect_one()) {
            // ---- K: a pair of pages is one operand of 128 rows; its stage is free once S is formed
            int lower = tile_row(0), upper = tile_row(1), J = 0;
            for (; J < np; ++J) {
                const int s = J % KS;
                if (J >= KS && !mbar_wait(smem_u32(&bars->k_empty[s]), ((J / KS) - 1) & 1)) { give_up(16); break; }
                const unsigned full = smem_u32(&bars->k_full[s]), dst = smem_u32(sK + s * KP_BYTES);
                mbar_expect_tx(full, KP_BYTES);
                for (int d = 0; d < HD / 64; ++d) {
                    load_rows(dst + d * (2 * BN * 128), &map, full, d * 64, lower, kv.k);
                    load_rows(dst + d * (2 * BN * 128) + BN * 128, &map, full, d * 64, upper, kv.k);
                }
                lower = tile_row(2 * J + 2);
                upper = tile_row(2 * J + 3);
            }
            if (has_failed(bars))                                    // what was asked for arrives before the memory is given back
                for (int i = max(0, J - KS); i < J; ++i) (void)mbar_wait(smem_u32(&bars->k_full[i % KS]), (i / KS) & 1);
        }
    } else if (warp == 10) {
        if (elect_one()) {
            // ---- V: a stage is free once O += P V is done
            int row = tile_row(0), j = 0;
            for (; j < nt; ++j) {
                const int s = j % VS;
                if (j >= VS && !mbar_wait(smem_u32(&bars->v_empty[s]), ((j / VS) - 1) & 1)) { give_up(16); break; }
                const unsigned full = smem_u32(&bars->v_full[s]), dst = smem_u32(sV + s * V_BYTES);
                mbar_expect_tx(full, V_BYTES);
                for (int d = 0; d < HD / 64; ++d) load_rows(dst + d * (BN * 128), &map, full, d * 64, row, kv.v);
                row = tile_row(j + 1);
            }
            if (has_failed(bars))
                for (int i = max(0, j - VS); i < j; ++i) (void)mbar_wait(smem_u32(&bars->v_full[i % VS]), (i / VS) & 1);
        }
    } else if (warp == 1) {
        if (elect_one()) {
            // ---- S of a pair: products of N = 128 with Q from tensor memory
            const unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)((2 * BN) >> 3) << 17) | ((unsigned)(BM >> 4) << 24);
            const uint64_t desc0 = umma_desc(smem_u32(sK), 16, 1024);
            bool ok = mbar_wait(smem_u32(&bars->q_tmem), 0);
            if (!ok) give_up(32);
            for (int J = 0; J < np && ok; ++J) {
                if (!mbar_wait(smem_u32(&bars->k_full[J % KS]), (J / KS) & 1)) { give_up(2); break; }
                if (J >= 1 && !mbar_wait(smem_u32(&bars->s_free), (J - 1) & 1)) { give_up(8); break; }
                if (has_failed(bars)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t desc = desc0 + (uint64_t)(((J % KS) * KP_BYTES) >> 4);
#pragma unroll
                for (int d = 0; d < HD / 64; ++d)
#pragma unroll
                    for (int k = 0; k < 64 / UMMA_K; ++k)
                        umma_a_tmem(tmem + S_COL, tmem + Q_COL + d * 32 + k * (UMMA_K / 2), desc + (uint64_t)((d * (2 * BN * 128) + k * 32) >> 4), idesc,
                                    (d > 0 || k > 0) ? 1u : 0u);
                umma_commit_cta1(smem_u32(&bars->k_empty[J % KS]));
                umma_commit_cta1(smem_u32(&bars->s_ready));
            }
        }
    } else if (warp == 11) {
        if (elect_one()) {
            // ---- O += P V: A (P) K-major, B (V) MN-major
            const unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((unsigned)(HD >> 3) << 17) | ((unsigned)(BM >> 4) << 24);
            const uint64_t v_desc0 = umma_desc(smem_u32(sV), BN * 128, 1024), p_desc0 = umma_desc(smem_u32(sP), 16, 1024);
            for (int j = 0; j < nt; ++j) {
                if (!mbar_wait(smem_u32(&bars->p_ready[j & 1]), (j >> 1) & 1)) { give_up(8); break; }
                if (has_failed(bars)) break;
                if (!mbar_wait(smem_u32(&bars->v_full[j % VS]), (j / VS) & 1)) { give_up(2); break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t v_desc = v_desc0 + (uint64_t)(((j % VS) * V_BYTES) >> 4), p_desc = p_desc0 + (uint64_t)(((j & 1) * P_BYTES) >> 4);
#pragma unroll
                for (int k = 0; k < BN / UMMA_K; ++k)
                    umma_bf16_cta1(tmem + O_COL, p_desc + (uint64_t)((k * 32) >> 4), v_desc + (uint64_t)((k * UMMA_K * 128) >> 4), idesc, (j > 0 || k > 0) ? 1u : 0u);
                umma_commit_cta1(smem_u32(&bars->v_empty[j % VS]));
                umma_commit_cta1(smem_u32(&bars->pv_done[j & 1]));
            }
        }
    } else {
        // ---- softmax: thread = query.  First its query goes to tensor memory, 64 elements (32 columns) at a time.
        bool alive = true;
        const int m = it.query0 + rloc, row = it.row0 + m / G, head = kh * G + m % G;
        const bool have = rloc < queries;
        if (group < Q_GROUPS) {
            constexpr int MINE = BLOCKS / Q_GROUPS;
            const uint4* src = reinterpret_cast<const uint4*>(q + (have ? (size_t)row * q_stride + (size_t)head * HD : 0));
            uint4 w[MINE][8];
#pragma unroll
            for (int i = 0; i < MINE; ++i)
#pragma unroll
                for (int c = 0; c < 8; ++c) w[i][c] = have ? src[(i * Q_GROUPS + group) * 8 + c] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                uint32_t v[32];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    v[c * 4 + 0] = w[i][c].x; v[c * 4 + 1] = w[i][c].y; v[c * 4 + 2] = w[i][c].z; v[c * 4 + 3] = w[i][c].w;
                }
                tmem_st32(lane_base + Q_COL + (i * Q_GROUPS + group) * 32, v);
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars->q_tmem));
        }
        const float cap = sc.cap;
        const float k1 = cap > 0.f ? sc.scale / cap : sc.scale;      // scores in the unit of the maximum: tanh(score / cap), or the scaled score
        const float k2 = (cap > 0.f ? cap : 1.f) * LOG2E;            // times this: the exponent to base 2
        const uint64_t k1_2 = two(k1, k1), k2_2 = two(k2, k2);
        const float slope = !FIXED && sc.slopes != nullptr && have ? sc.slopes[head] / (cap > 0.f ? cap : 1.f) : 0.f;
        int newest = 0;
        if (!FIXED && sc.slopes != nullptr && have) {
            const int slot = cells.slots[row];
            newest = slot >= 0 ? cells.slot_len[slot] - 1 : 0;
        }
        const float step = STEP / (cap > 0.f ? cap : 1.f);
        const int first = it.position(it.t0);
        float m_run = -CUDART_INF_F, m_used = 0.f, l_sum = 0.f;
        bool started = false;
        for (int j = group; j < nt && alive; j += 2) {
            const int J = j >> 1;
            if (!mbar_wait_warp(smem_u32(&bars->s_ready), J & 1)) {
                give_up(4);
                alive = false;
                break;
            }
            if (__any_sync(0xffffffffu, has_failed(bars))) {
                alive = false;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float s[BN];
            {
                uint32_t v0[32], v1[32];
                tmem_ld32_nowait(lane_base + S_COL + group * BN, v0);
                tmem_ld32_nowait(lane_base + S_COL + group * BN + 32, v1);
                tmem_ld_wait();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars->s_free));
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                    s[c] = __uint_as_float(v0[c]);
                    s[32 + c] = __uint_as_float(v1[c]);
                }
            }
            float corr = 1.f;
            bool rescale = false;
            uint64_t rs01 = two(0.f, 0.f), rs23 = two(0.f, 0.f);     // sums of the columns c % 4
            if (FIXED) {
#pragma unroll
                for (int c = 0; c < BN; c += 4) {
                    rs01 = add2(rs01, capped_exp2(s[c], s[c + 1], k1_2, k2_2, (c & 7) < POLY));
                    rs23 = add2(rs23, capped_exp2(s[c + 2], s[c + 3], k1_2, k2_2, (c & 7) < POLY));
                }
            } else {
                const float bias0 = slope * (float)(first + j * BN - newest);
                float mx4[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
                for (int c = 0; c < BN; ++c) {
                    const float bias = fmaf(slope, (float)c, bias0);
                    s[c] = cap > 0.f ? tanh_approx(s[c] * k1) + bias : fmaf(s[c], k1, bias);
                    mx4[c & 3] = fmaxf(mx4[c & 3], s[c]);
                }
                const float mine = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                m_run = fmaxf(m_run, mine);
                if (2 * J + 1 < nt) {
                    // Both groups take their exponentials against one reference.  A group writes the place of pair J + 2 only when the
                    // other has arrived for J + 1, that is, has read J.
                    float(*const told)[BM] = bars->row_max[J & 1];
                    told[group][rloc] = mine;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&bars->max_ready[quarter]));
                    if (!mbar_wait_warp(smem_u32(&bars->max_ready[quarter]), J & 1)) {
                        give_up(4);
                        alive = false;
                        break;
                    }
                    m_run = fmaxf(m_run, told[group ^ 1][rloc]);
                }
                if (m_run != -CUDART_INF_F && (!started || m_run > m_used + step)) {
                    corr = started ? exp2_fast((m_used - m_run) * k2) : 0.f;
                    rescale = started;
                    m_used = m_run;
                    started = true;
                }
                const float moff = m_used * k2;
                const uint64_t less = two(-moff, -moff);
#pragma unroll
                for (int c = 0; c < BN; c += 4) {
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        float x, y;
                        one_by_one(fma2(two(s[c + i], s[c + i + 1]), k2_2, less), x, y);
                        s[c + i] = exp2_fast(x);
                        s[c + i + 1] = exp2_fast(y);
                    }
                    rs01 = add2(rs01, two(s[c], s[c + 1]));
                    rs23 = add2(rs23, two(s[c + 2], s[c + 3]));
                }
            }
            if (FIXED) {
                l_sum += capped_sum(rs01, rs23);
            } else {
                float a, b, c, d;
                one_by_one(rs01, a, b);
                one_by_one(rs23, c, d);
                l_sum = l_sum * corr + ((a + b) + (c + d));
            }
            // P_j overwrites what P_{j-2} V_{j-2} read
            if (j >= 2 && !mbar_wait_warp(smem_u32(&bars->pv_done[group]), ((j - 2) >> 1) & 1)) {
                give_up(64);
                alive = false;
                break;
            }
            {
                unsigned char* prow = sP + group * P_BYTES + rloc * 128;
#pragma unroll
                for (int ch = 0; ch < BN / 8; ++ch)
                    *reinterpret_cast<uint4*>(prow + ((ch ^ (rloc & 7)) << 4)) =
                        make_uint4(pack_bf16(s[ch * 8 + 0], s[ch * 8 + 1]), pack_bf16(s[ch * 8 + 2], s[ch * 8 + 3]), pack_bf16(s[ch * 8 + 4], s[ch * 8 + 5]),
                                   pack_bf16(s[ch * 8 + 6], s[ch * 8 + 7]));
            }
            // group 0 rescales: P V of the second group's page comes after its own
            if (!FIXED && group == 0 && __any_sync(0xffffffffu, rescale)) {
                if (j >= 1 && !mbar_wait_warp(smem_u32(&bars->pv_done[1]), ((j - 1) >> 1) & 1)) {
                    give_up(64);
                    alive = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const float f = rescale ? corr : 1.f;
#pragma unroll 1
                for (int c0 = 0; c0 < HD; c0 += 32) {
                    uint32_t v[32];
                    tmem_ld32_sync(lane_base + O_COL + c0, v);
#pragma unroll
                    for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * f);
                    tmem_st32(lane_base + O_COL + c0, v);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars->p_ready[group]));
        }
        // Each group waits for its own last product first (a parity says nothing about a phase that has not begun; of its own pages it
        // has seen every phase before); products are done in order, so after that the very last may be asked for.
        if (alive) {
            const int jl = nt - 1, jmine = (jl & 1) != group ? jl - 1 : jl;
            if (jmine >= 0 && jmine != jl && !mbar_wait_warp(smem_u32(&bars->pv_done[jmine & 1]), (jmine >> 1) & 1)) {
                give_up(64);
                alive = false;
            }
            if (alive && !mbar_wait_warp(smem_u32(&bars->pv_done[jl & 1]), (jl >> 1) & 1)) {
                give_up(64);
                alive = false;
            }
        }
        // a row's sum is that of both groups (against the same reference); without a softcap the second group's reference may lag behind
        // in the last pair when there is no upper page, and then it has nothing newer to add
        // (Their places are those of the maxima: the last product is done, so group 0 has read what it was told.)
        float *const l_second = bars->row_max[0][0], *const m_second = bars->row_max[0][1];
        if (group == 1) {
            l_second[rloc] = l_sum;
            m_second[rloc] = m_used;
        }
        asm volatile("bar.sync 2, 256;" ::: "memory");               // the eight softmax warps
        if (__any_sync(0xffffffffu, has_failed(bars))) alive = false;
        if (alive) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const size_t at = have ? part_of(it, sh, m, kh, G, nq) : 0;
            if (group == 0 && have) {
                float l_other = l_second[rloc];
                if (!FIXED && l_other != 0.f) l_other *= exp2_fast((m_second[rloc] - m_used) * k2);      // (without a weight it has no reference)
                part_ml[at] = make_float2(FIXED ? 0.f : m_used * k2, l_sum + l_other);
            }
            // Half of the head by each group, through the K ring (16-byte pieces XOR-ed with the row), so that whole rows are written.
            constexpr int HALF = HD / 2;
            unsigned char* const mine = sK + rloc * (HD * 4);
#pragma unroll 1
            for (int c0 = group * HALF; c0 < (group + 1) * HALF; c0 += 32) {
                uint32_t v[32];
                tmem_ld32_sync(lane_base + O_COL + c0, v);
#pragma unroll
                for (int c = 0; c < 32; c += 4)
                    *reinterpret_cast<uint4*>(mine + (((c0 + c) / 4 ^ (rloc & 7)) << 4)) = make_uint4(v[c], v[c + 1], v[c + 2], v[c + 3]);
            }
        }
        asm volatile("bar.sync 2, 256;" ::: "memory");
        if (alive) {
            constexpr int CPR = HD / 4, RPI = CPR < 32 ? 32 / CPR : 1, PPR = CPR < 32 ? 1 : CPR / 32;       // pieces of a row; rows, pieces per lane at a time
            const int first_row = (warp - 2) * 16;                   // each of the eight warps writes sixteen rows
#pragma unroll 4
            for (int rr = 0; rr < 16; rr += RPI) {
                const int r = first_row + rr + (CPR < 32 ? lane / CPR : 0);
                if (r >= queries) continue;
                float* dst = part_o + part_of(it, sh, it.query0 + r, kh, G, nq) * HD;
#pragma unroll
                for (int i = 0; i < PPR; ++i) {
                    const int c = i * 32 + lane % (CPR < 32 ? CPR : 32);
                    *reinterpret_cast<uint4*>(dst + c * 4) = *reinterpret_cast<const uint4*>(sK + r * (HD * 4) + ((c ^ (r & 7)) << 4));
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

template <int HD, bool FIXED>
int launch(const SharedLaunch& a, cudaStream_t st) {
    CUtensorMap map;
    KV kv;
    if (const int rc = make_pools_map(&map, &kv, a.k_pool, a.v_pool, a.pool_rows, HD, BN)) return rc;
    constexpr size_t layout = (size_t)k_stages(HD) * 2 * BN * HD * 2 + (size_t)v_stages(HD) * BN * HD * 2 + 2 * P_BYTES + sizeof(Barriers);
    static_assert(layout <= 227 * 1024, "a block's shared memory");
    const size_t smem = layout + 1024 < 227 * 1024 ? layout + 1024 : 227 * 1024;
    auto kern = attn_shared_tcgen05_kernel<HD, FIXED>;
    static OncePerDevice asked;
    if (const int rc = allow_shared(asked, kern, smem)) return rc;
    const long long items = (long long)a.sh.n_groups * a.sh.common_tiles * a.sh.common_ranges;
    if (items <= 0) return 0;
    if (items > 0x7fffffff) return QNN_ERR_UNSUPPORTED;
    launch_pdl(kern, dim3((unsigned)items, a.nkv), dim3(THREADS), smem, st, map, kv, (const bf16*)a.q, (size_t)a.q_stride, a.cells, a.sh, a.nq, a.nkv, a.sc,
               a.part_o, a.part_ml, a.status);
    return (int)cudaGetLastError();
}

}  // namespace

int qnn::shared::launch_common_tcgen05(const SharedLaunch& a, cudaStream_t st) {
    const bool fixed = a.sc.cap > 0.f && a.sc.cap <= 70.f && a.sc.slopes == nullptr;       // exp(cap) times any number of keys stays in float32
    switch (a.hd) {
        case 64: return fixed ? launch<64, true>(a, st) : launch<64, false>(a, st);
        case 128: return fixed ? launch<128, true>(a, st) : launch<128, false>(a, st);
        case 256: return fixed ? launch<256, true>(a, st) : launch<256, false>(a, st);
        default: return QNN_ERR_UNSUPPORTED;
    }
}
