// Copies inside the cache, for sequences that go on from another's: fixed-size states from slot to slot, and the filled part of pages
// of keys and values.  Any number of tensors and pairs (source, destination) in few launches: both lists travel as kernel arguments, so
// nothing is uploaded before a launch and nothing has to outlive it.  Destinations are never sources (the caller sees to it), so the
// order of the copies does not matter.
//
// Bound by memory: every byte is read once and written once.  32 of 64 slots, 153 MB read and written: 44.7 us, 6.8 TB/s with what
// stays in L2 (5.7 TB/s of it at the memory); 63 pages of 13 lines 36.7 us, 5.8 TB/s.  Few bytes: one launch, 1.3 us, behind 9 us of host time.
#include "common.cuh"

using namespace qnn;

namespace {

constexpr int MOST_PAIRS = 128, MOST_TENSORS = 64;
constexpr int COPY_THREADS = 256, AHEAD = 4;                  // loads of a thread in flight
constexpr int COPY_BYTES = COPY_THREADS * AHEAD * 16;         // of a block

struct Pairs {
    int src[MOST_PAIRS], dst[MOST_PAIRS];
};
struct Tensors {
    char* base[MOST_TENSORS];
    long long bytes[MOST_TENSORS];                            // of one slot
    int blocks[MOST_TENSORS + 1];                             // blocks before tensor i
};

// `bytes` from src to dst, from byte `at` on COPY_BYTES of them at most, by a block; 16 bytes at a time where both allow it.
__device__ __forceinline__ void copy_piece(char* __restrict__ dst, const char* __restrict__ src, long long bytes, long long at) {
    const long long end = min(bytes, at + COPY_BYTES);
    const uintptr_t both = (uintptr_t)dst | (uintptr_t)src;
    if (((both | (uintptr_t)bytes) & 15) == 0) {
        uint4 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const long long p = at + (long long)(i * COPY_THREADS + threadIdx.x) * 16;
            if (p < end) v[i] = *reinterpret_cast<const uint4*>(src + p);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const long long p = at + (long long)(i * COPY_THREADS + threadIdx.x) * 16;
            if (p < end) *reinterpret_cast<uint4*>(dst + p) = v[i];
        }
    } else if (((both | (uintptr_t)bytes) & 3) == 0) {
        for (long long p = at + threadIdx.x * 4; p < end; p += COPY_THREADS * 4) *reinterpret_cast<uint32_t*>(dst + p) = *reinterpret_cast<const uint32_t*>(src + p);
    } else {
        for (long long p = at + threadIdx.x; p < end; p += COPY_THREADS) dst[p] = src[p];
    }
}

// grid (blocks of all tensors, pairs)
__global__ void __launch_bounds__(COPY_THREADS) copy_slots_kernel(const __grid_constant__ Tensors t, const __grid_constant__ Pairs pairs, int n_tensors) {
    pdl_wait();
    int i = 0;
    while (i + 1 < n_tensors && (int)blockIdx.x >= t.blocks[i + 1]) ++i;
    const long long bytes = t.bytes[i];
    copy_piece(t.base[i] + pairs.dst[blockIdx.y] * bytes, t.base[i] + pairs.src[blockIdx.y] * bytes, bytes,
               (long long)(blockIdx.x - t.blocks[i]) * COPY_BYTES);
}

struct PagePairs {
    int src[MOST_PAIRS], dst[MOST_PAIRS];
    int used[MOST_PAIRS];                                     // positions of the page that are copied
};

// grid (lines x kv heads x pieces of a head's page, pairs, K and V)
__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(char* __restrict__ k, char* __restrict__ v, const __grid_constant__ PagePairs pairs,
                                                                  long long pages, int heads, int page_bytes, int position_bytes, int pieces) {
    pdl_wait();
    const int run = blockIdx.x / pieces, piece = blockIdx.x % pieces, line = run / heads, head = run % heads;
    const int bytes = pairs.used[blockIdx.y] * position_bytes;
    const long long at = (long long)piece * COPY_BYTES;
    if (at >= bytes) return;
    char* base = blockIdx.z ? v : k;
    const auto place = [&](int page) { return base + (((long long)line * pages + page) * heads + head) * page_bytes; };
    copy_piece(place(pairs.dst[blockIdx.y]), place(pairs.src[blockIdx.y]), bytes, at);
}

}  // namespace

// tensors: n_tensors x (address, bytes of a row); row dst[p] = row src[p] of every tensor, for every pair.  pairs: n_pairs sources, then as many
// destinations.  Both are host arrays, read before the call returns.
QNN_API int qnn_copy_slots(const long long* tensors, int n_tensors, const int* pairs_of, int n_pairs, cudaStream_t st) {
    for (int t0 = 0; t0 < n_tensors; t0 += MOST_TENSORS) {
        Tensors t;
        const int nt = n_tensors - t0 < MOST_TENSORS ? n_tensors - t0 : MOST_TENSORS;
        long long blocks = 0;
        for (int i = 0; i < nt; ++i) {
            t.base[i] = (char*)tensors[2 * (t0 + i)];
            t.bytes[i] = tensors[2 * (t0 + i) + 1];
            t.blocks[i] = (int)blocks;
            blocks += (t.bytes[i] + COPY_BYTES - 1) / COPY_BYTES;
            if (blocks > 0x7fffffff) return QNN_ERR_UNSUPPORTED;
        }
        t.blocks[nt] = (int)blocks;
        if (blocks == 0) continue;
        for (int p0 = 0; p0 < n_pairs; p0 += MOST_PAIRS) {
            Pairs pairs;
            const int np = n_pairs - p0 < MOST_PAIRS ? n_pairs - p0 : MOST_PAIRS;
            for (int i = 0; i < np; ++i) {
                pairs.src[i] = pairs_of[p0 + i];
                pairs.dst[i] = pairs_of[n_pairs + p0 + i];
            }
            launch_pdl(copy_slots_kernel, dim3((unsigned)blocks, np), dim3(COPY_THREADS), 0, st, t, pairs, nt);
            if (const cudaError_t e = cudaGetLastError()) return (int)e;
        }
    }
    return 0;
}

// Pools [lines][pages][heads][page_size][head_dim] of esize-byte elements (v == k: one pool): the first used positions of page src go to page
// dst, in every line and head, for every pair.  moves: n_pairs sources, as many destinations, as many numbers of positions: a host array, read
// before the call returns.
QNN_API int qnn_copy_pages(void* k, void* v, int lines, long long pages, int heads, int page_size, int head_dim, int esize, const int* moves,
                           int n_pairs, cudaStream_t st) {
    if (lines <= 0 || n_pairs <= 0) return 0;
    const long long page_bytes = (long long)page_size * head_dim * esize;
    if (page_bytes > 0x7fffffff) return QNN_ERR_UNSUPPORTED;
    const int *src = moves, *dst = moves + n_pairs, *used = moves + 2 * n_pairs;
    for (int p0 = 0; p0 < n_pairs; p0 += MOST_PAIRS) {
        PagePairs pairs;
        const int np = n_pairs - p0 < MOST_PAIRS ? n_pairs - p0 : MOST_PAIRS;
        int most = 0;
        for (int i = 0; i < np; ++i) {
            pairs.src[i] = src[p0 + i];
            pairs.dst[i] = dst[p0 + i];
            pairs.used[i] = used[p0 + i];
            most = used[p0 + i] > most ? used[p0 + i] : most;
        }
        const int pieces = (int)(((long long)most * head_dim * esize + COPY_BYTES - 1) / COPY_BYTES);
        if (pieces == 0) continue;
        const long long runs = (long long)lines * heads * pieces;
        if (runs > 0x7fffffff) return QNN_ERR_UNSUPPORTED;
        launch_pdl(copy_pages_kernel, dim3((unsigned)runs, np, v != k ? 2 : 1), dim3(COPY_THREADS), 0, st, (char*)k, (char*)v, pairs, pages, heads,
                   (int)page_bytes, head_dim * esize, pieces);
        if (const cudaError_t e = cudaGetLastError()) return (int)e;
    }
    return 0;
}
