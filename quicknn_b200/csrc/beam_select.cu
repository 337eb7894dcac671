// The best continuations of every request over its beams and the vocabulary, for beam search.
//
// Beam b of a request has the score t_b (a sum of logarithms of probabilities); with z = logits[b] its continuation by token v scores
//     t_b + z_v - log(sum_u exp(z_u)).
// Wanted are the `take` best of a request's beams x V continuations in descending order, equal scores by the lowest (beam, token).
//
// Within a beam the order of the scores is that of the logits, so one pass over the logits is enough for everything but a few of them:
//   1. a warp per segment of a row (SEGMENT logits) leaves the segment's maximum and sum of exp(z - maximum);
//   2. a block per request joins them to log(sum exp) of every beam, turns the segments' maxima into scores, and takes as a threshold the
//      `take`-th largest of 128 groups' maxima, so that at least `take` segments reach it.  As each of these holds a score that reaches it, so do
//      the `take` best of all; they lie in the segments that reach it, which are read again (a few KB) into a short list, whose best are
//      found by counting.  Where a request has few logits, that block does the first pass too, and the groups are of logits.
// Scores are formed in 64 bits: those of different beams may differ by less than 32 bits resolve after a sum over the vocabulary.
// A logit that is not finite is no continuation and not in the sum (bit 0 of the error word says so); nor is any of a beam whose score is
// -inf or NaN.  Where fewer than `take` are left, the places behind them hold score -inf, beam -1, token -1.
#include "common.cuh"
#include <float.h>
#include <math_constants.h>

using namespace qnn;

namespace {

constexpr int SELECT_MOST = 64;               // continuations per request, at most
// Of the second kernel's block.  It is short code that every warp runs once, so what it takes is instructions times warps: 4 beams x 1000 words 6.4 us
// with 512 (when that took 6.2, 1024 took 7.7); 10 beams x 1015 10.8 (when that took 9.6, 256 took 13).  Of its 11,000 cycles (8 beams x 99,521)
// 4,500 go to the logarithms of the sums, 2,000 to the threshold, 3,000 to the second look, 1,500 to the order.
constexpr int THREADS = 512;
constexpr int LIST = 2048;                    // places of the short list
constexpr int MOST_REACHED = 512;             // segments that are looked at again

// Segment `s` of a row starts at its logit s * SEGMENT - shift, shift the row's distance from a 16-byte boundary: segments then start on
// one, and the row's first and last segments hold a few logits less.
__device__ __forceinline__ int segment_start(const float* row, int s, int segment) { return s * segment - (int)(((uintptr_t)row >> 2) & 3); }

// One maximum and sum per segment: warp w of the grid takes segments w, w + warps, ... of all rows, and asks for the next one's logits before it
// works on those it has.  Whether all are finite is read off the maximum, the minimum and the sum; only where they are not does a
// second look leave the others out.  Exponentials are the fast ones of z - m: with the logit's distance d from the maximum they are off by at
// most |d| 2^-23 + 2^-22, of weight e^d in the sum, which moves the sum's logarithm by less than 2^-20 however the logits lie.
// Bound by memory, and by how much of it a short kernel keeps in flight: 80 rows of 255,029 (82 MB, 12.5 us at the copy rate), us, by segment and
// loads: 512, 4 bytes a lane 21.5; 1024, 16 bytes 19.6; the same with the fast exponentials 17.3 (torch's amax alone: 24.7).
template <int SEGMENT>
struct Segment {
    static constexpr int PER = SEGMENT / 128;                 // 16-byte pieces a lane
    float4 ahead[PER];

    __device__ __forceinline__ static int place(const float* logits, int V, int segments, int i, const float*& row) {
        const int r = i / segments;
        row = logits + (size_t)r * V;
        return segment_start(row, i - r * segments, SEGMENT);
    }
    // asks for segment i's logits
    __device__ __forceinline__ void ask(const float* __restrict__ logits, int V, int segments, int total, int i) {
        if (i >= total) return;
        const int lane = threadIdx.x & 31;
        const float* row;
        const int v0 = place(logits, V, segments, i, row);
        if (v0 >= 0 && v0 + SEGMENT <= V) {
            const float4* p = reinterpret_cast<const float4*>(row + v0) + lane;
#pragma unroll
            for (int j = 0; j < PER; ++j) ahead[j] = p[j * 32];
        } else {                                              // outside the row: its nearest logit, taken out later
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = row[min(max(v0 + (j * 32 + lane) * 4 + e, 0), V - 1)];
                ahead[j] = make_float4(x[0], x[1], x[2], x[3]);
            }
        }
    }
    // the maximum and sum of segment i, whose logits are here, and asks for those of segment `next`; `keep`: a place for the logits, -inf for
    // those that do not count
    __device__ __forceinline__ float2 stats(const float* __restrict__ logits, int V, int segments, int total, int i, int next, int* __restrict__ error_flag,
                                            float4* __restrict__ keep = nullptr) {
        const int lane = threadIdx.x & 31;
        float z[PER * 4];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            z[j * 4] = ahead[j].x;
            z[j * 4 + 1] = ahead[j].y;
            z[j * 4 + 2] = ahead[j].z;
            z[j * 4 + 3] = ahead[j].w;
        }
        ask(logits, V, segments, total, next);
        const float* row;
        const int v0 = place(logits, V, segments, i, row);
        float m = -CUDART_INF_F, least = CUDART_INF_F;
        if (v0 < 0 || v0 + SEGMENT > V) {
#pragma unroll
            for (int j = 0; j < PER * 4; ++j) {
                const int v = v0 + (j / 4 * 32 + lane) * 4 + j % 4;
                if (v >= 0 && v < V) {
                    m = fmaxf(m, z[j]);
                    least = fminf(least, z[j]);
                } else {
                    z[j] = -CUDART_INF_F;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < PER * 4; ++j) {
                m = fmaxf(m, z[j]);
                least = fminf(least, z[j]);
            }
        }
        m = warp_max(m);
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < PER * 4; ++j) s += __expf(z[j] - m);
        s = warp_sum(s);
        if (__any_sync(0xffffffffu, least == -CUDART_INF_F) || !(s < CUDART_INF_F)) {      // (NaN, or an infinity in the maximum, make s a NaN)
            float finite = -CUDART_INF_F;
            bool bad = false;
#pragma unroll
            for (int j = 0; j < PER * 4; ++j) {
                const int v = v0 + (j / 4 * 32 + lane) * 4 + j % 4;
                if (!isfinite(z[j])) {
                    bad = bad || (v >= 0 && v < V);
                    z[j] = -CUDART_INF_F;
                }
                finite = fmaxf(finite, z[j]);
            }
            m = warp_max(finite);
            s = 0.f;
            if (m != -CUDART_INF_F)
#pragma unroll
                for (int j = 0; j < PER * 4; ++j) s += __expf(z[j] - m);
            s = warp_sum(s);
            if (__any_sync(0xffffffffu, bad) && lane == 0 && error_flag != nullptr) atomicOr(error_flag, 1);
        }
        if (keep != nullptr)
#pragma unroll
            for (int j = 0; j < PER; ++j) keep[j * 32 + lane] = make_float4(z[j * 4], z[j * 4 + 1], z[j * 4 + 2], z[j * 4 + 3]);
        return make_float2(m, s);
    }
};

template <int SEGMENT>
__global__ void __launch_bounds__(256, SEGMENT >= 1024 ? 2 : 4)
beam_segments_kernel(const float* __restrict__ logits, int V, int segments, int total, float2* __restrict__ stats, int* __restrict__ error_flag) {
    pdl_wait();
    const int warps = gridDim.x * 8;
    Segment<SEGMENT> seg;
    int i = blockIdx.x * 8 + (threadIdx.x >> 5);
    seg.ask(logits, V, segments, total, i);
    for (; i < total; i += warps) {
        const float2 ms = seg.stats(logits, V, segments, total, i, i + warps, error_flag);
        if ((threadIdx.x & 31) == 0) stats[i] = ms;
    }
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// a score in 32 bits, finite
__device__ __forceinline__ float rounded(double score) { return fmaxf((float)score, -FLT_MAX); }
__device__ __forceinline__ bool before(double a, unsigned ia, double b, unsigned ib) { return a > b || (a == b && ia < ib); }

// The `take`-th largest of 128 groups' maxima, value i of n in group i % 128, found by counting, into `result` (which stays as it is where
// fewer groups hold anything above -inf).  By the whole block; what it reads is written, and what it writes is there, in all threads.
constexpr int GROUPS = 128;
template <typename F>
__device__ __forceinline__ void nth_of_groups(int n, int take, F value, float* group_best, float& result) {
    constexpr int EACH = THREADS / GROUPS;    // threads a group
    const int g = threadIdx.x / EACH, e = threadIdx.x % EACH;
    __syncthreads();
    float most = -CUDART_INF_F;
    for (int i = g + e * GROUPS; i < n; i += THREADS) most = fmaxf(most, value(i));
#pragma unroll
    for (int o = 1; o < EACH; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (e == 0) group_best[g] = most;
    __syncthreads();
    int rank = 0;                             // each of a group's threads counts against its share
#pragma unroll 16
    for (int o = e; o < GROUPS; o += EACH) {
        const float other = group_best[o];
        rank += other > most || (other == most && o < g);
    }
#pragma unroll
    for (int o = 1; o < EACH; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (rank == take - 1 && e == 0 && most > -CUDART_INF_F) result = most;
    __syncthreads();
}

struct Found {
    double score[LIST];
    unsigned at[LIST];                        // beam * V + token
};

// ALONE: a request's logits are few enough for this block to do the first pass as well (`stats` is not used then), and to keep them: the threshold
// is that of groups of single logits (of a few segments' maxima it would be a low one and let thousands pass).
template <int SEGMENT, bool ALONE>
__global__ void __launch_bounds__(THREADS)
beam_pick_kernel(const float* __restrict__ logits, int V, int beams, int take, int segments, const float* __restrict__ scores,
                 const float2* __restrict__ stats, float* __restrict__ out_scores, int* __restrict__ out_beams, int* __restrict__ out_tokens,
                 const int* __restrict__ status_in, int* __restrict__ error_flag) {
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0 && status_in != nullptr && error_flag != nullptr) {
        const int s = *status_in;             // what the step's kernels reported: bit 1 and their status from bit 8 up
        if (s != 0) atomicOr(error_flag, 2 | (s << 8));
    }
    extern __shared__ __align__(16) unsigned char smem[];
    Found* found = reinterpret_cast<Found*>(smem);
    double* base = reinterpret_cast<double*>(found + 1);      // [beams] t_b - log(sum exp)
    float* best = reinterpret_cast<float*>(base + (beams + 1) / 2 * 2);   // [beams * segments] the segments' best scores; -inf: none
    constexpr int WARPS = THREADS / 32, KEPT = 4;
    __shared__ float part_m[WARPS];
    __shared__ double part_s[WARPS];
    __shared__ float group_best[GROUPS], threshold_s;
    __shared__ int reached[MOST_REACHED], n_reached, n_found;
    __shared__ double last_score;
    __shared__ unsigned last_at;
    const int q = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const size_t row0 = (size_t)q * beams;
    const float2* mine_stats = stats + row0 * segments;       // of this request's beams
    float4* logits_here = reinterpret_cast<float4*>(best + (beams * segments + 3) / 4 * 4);
    float2* here = reinterpret_cast<float2*>(logits_here + beams * segments * (SEGMENT / 4));
    if (ALONE) {
        Segment<SEGMENT> seg;
        const int total = beams * segments;
        seg.ask(logits + row0 * V, V, segments, total, warp);
        for (int i = warp; i < total; i += WARPS) {
            const float2 ms = seg.stats(logits + row0 * V, V, segments, total, i, i + WARPS, error_flag, logits_here + i * (SEGMENT / 4));
            if (lane == 0) here[i] = ms;
        }
        mine_stats = here;
    }
    if (threadIdx.x == 0) {
        n_found = n_reached = 0;
        threshold_s = -FLT_MAX;               // fewer groups than wanted: all that hold anything
    }
    if (ALONE) __syncthreads();
    // log(sum exp) of every beam, by a warp each or, where it has many segments, by as many as there are; a lane keeps its segments' numbers where they fit
    const int share = max(1, min(WARPS / beams, (segments + 32 * KEPT - 1) / (32 * KEPT)));
    for (int b0 = 0; b0 < beams; b0 += WARPS / share) {
        const int b = b0 + warp / share, p = warp % share, i0 = p * 32 + lane, step = share * 32;
        const bool mine = warp / share < WARPS / share && b < beams;
        const float2* st = mine_stats + (size_t)(mine ? b : 0) * segments;
        const double t = mine ? (double)scores[row0 + b] : 0.0;
        float2 kept[KEPT];
        float m = -CUDART_INF_F;
#pragma unroll
        for (int k = 0; k < KEPT; ++k) {
            kept[k] = mine && i0 + k * step < segments ? st[i0 + k * step] : make_float2(-CUDART_INF_F, 0.f);
            m = fmaxf(m, kept[k].x);
        }
        if (mine)
            for (int i = i0 + KEPT * step; i < segments; i += step) m = fmaxf(m, st[i].x);
        m = qnn::warp_max(m);
        if (share > 1) {
            if (lane == 0) part_m[warp] = m;
            __syncthreads();
            if (mine)
                for (int i = 0; i < share; ++i) m = fmaxf(m, part_m[warp / share * share + i]);
        }
        double s = 0.0;
        if (mine && m != -CUDART_INF_F) {
#pragma unroll
            for (int k = 0; k < KEPT; ++k) s += (double)(kept[k].y * expf(kept[k].x - m));       // (0 times exp(-inf) where there is none)
            for (int i = i0 + KEPT * step; i < segments; i += step) s += (double)(st[i].y * expf(st[i].x - m));
        }
        s = warp_sum(s);
        if (share > 1) {
            if (lane == 0) part_s[warp] = s;
            __syncthreads();
            s = 0.0;
            if (mine)
                for (int i = 0; i < share; ++i) s += part_s[warp / share * share + i];
        }
        // (one lane a beam takes the logarithm, which is long in 64 bits)
        if (mine && p == 0 && lane == 0) base[b] = m != -CUDART_INF_F && t > -CUDART_INF && t < CUDART_INF ? t - (double)m - log(s) : -CUDART_INF;
        __syncthreads();
        if (mine) {
            const double add = base[b];
            const auto note = [&](int i, float z) {
                const bool holds = add != -CUDART_INF && z != -CUDART_INF_F;
                best[b * segments + i] = holds ? rounded(add + (double)z) : -CUDART_INF_F;
                if (ALONE) reinterpret_cast<double*>(here)[b * segments + i] = holds ? add : -CUDART_INF;       // (nobody else reads these numbers)
            };
#pragma unroll
            for (int k = 0; k < KEPT; ++k)
                if (i0 + k * step < segments) note(i0 + k * step, kept[k].x);
            for (int i = i0 + KEPT * step; i < segments; i += step) note(i, st[i].x);
        }
        if (b0 + WARPS / share < beams) __syncthreads();      // the partial results have been read
    }
    const int n = beams * segments;
    // Logits of a beam below this are out, whatever the roundings (of those that are not, the scores are formed in 64 bits).
    const auto limit_of = [&](double add, float threshold) {
        const double top = (double)threshold, exactly = top - add;
        return threshold > -FLT_MAX ? rounded(exactly - 1e-5 * (fabs(exactly) + fabs(top))) : -FLT_MAX;
    };
    // The threshold is compared with the segments' best scores and with scores of other beams, so single logits, too, become scores in 64 bits that are
    // rounded once.  (t_b - log(sum exp) rounded before the sum would move all of a beam's scores together, by more than their distances to
    // another's where logits are large.)
    if (ALONE) nth_of_groups(n * SEGMENT, take, [&](int i) {
                                 const double s = reinterpret_cast<const double*>(here)[i / SEGMENT] + (double)reinterpret_cast<const float*>(logits_here)[i];
                                 return s > -CUDART_INF ? rounded(s) : -CUDART_INF_F;
                             }, group_best, threshold_s);
    else nth_of_groups(n, take, [&](int i) { return best[i]; }, group_best, threshold_s);
    const float threshold = threshold_s;
    if (ALONE) {
        for (int l = warp; l < n; l += WARPS) {
            if (best[l] == -CUDART_INF_F) continue;
            const int b = l / segments;
            const double add = base[b];
            const float limit = limit_of(add, threshold);
            const int v0 = segment_start(logits + (row0 + b) * V, l - b * segments, SEGMENT);
#pragma unroll
            for (int j = 0; j < SEGMENT / 32; ++j) {
                const float z = reinterpret_cast<const float*>(logits_here)[l * SEGMENT + j * 32 + lane];
                if (!(z >= limit)) continue;                  // (limit is finite, what is no continuation -inf)
                const double s = add + (double)z;
                if (rounded(s) < threshold) continue;
                const int at = atomicAdd(&n_found, 1);
                if (at < LIST) {
                    found->score[at] = s;
                    found->at[at] = (unsigned)b * (unsigned)V + (unsigned)(v0 + j * 32 + lane);
                }
            }
        }
    } else {
        for (int i = threadIdx.x; i < n; i += THREADS)
            if (best[i] >= threshold) {
                const int at = atomicAdd(&n_reached, 1);
                if (at < MOST_REACHED) reached[at] = i;
            }
        __syncthreads();
        // (of more than the list holds every segment is looked at)
        const int n_look = n_reached <= MOST_REACHED ? n_reached : n;
        for (int l = warp; l < n_look; l += WARPS) {
            const int i = n_reached <= MOST_REACHED ? reached[l] : l;
            if (best[i] < threshold) continue;
            const int b = i / segments;
            const float* row = logits + (row0 + b) * V;
            const int v0 = segment_start(row, i - b * segments, SEGMENT);
            const double add = base[b];
            const float limit = limit_of(add, threshold);
            float4 z[SEGMENT / 128];
            const bool whole = v0 >= 0 && v0 + SEGMENT <= V;
            if (whole) {
                const float4* src = reinterpret_cast<const float4*>(row + v0) + lane;
#pragma unroll
                for (int j = 0; j < SEGMENT / 128; ++j) z[j] = src[j * 32];
            } else {
#pragma unroll
                for (int j = 0; j < SEGMENT / 128; ++j) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int v = v0 + (j * 32 + lane) * 4 + e;
                        x[e] = v >= 0 && v < V ? row[v] : -CUDART_INF_F;
                    }
                    z[j] = make_float4(x[0], x[1], x[2], x[3]);
                }
            }
#pragma unroll
            for (int j = 0; j < SEGMENT / 128; ++j) {
                if (!(fmaxf(fmaxf(z[j].x, z[j].y), fmaxf(z[j].z, z[j].w)) >= limit)) continue;      // (the maximum of those that are numbers)
                const float x[4] = {z[j].x, z[j].y, z[j].z, z[j].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (!(x[e] >= limit) || x[e] > FLT_MAX) continue;
                    const double s = add + (double)x[e];
                    if (rounded(s) < threshold) continue;
                    const int at = atomicAdd(&n_found, 1);
                    if (at < LIST) {
                        found->score[at] = s;
                        found->at[at] = (unsigned)b * (unsigned)V + (unsigned)(v0 + (j * 32 + lane) * 4 + e);
                    }
                }
            }
        }
    }
    __syncthreads();
    const int have = n_found;
    float* os = out_scores + (size_t)q * take;
    int* ob = out_beams + (size_t)q * take;
    int* ot = out_tokens + (size_t)q * take;
    if (have <= LIST) {
        for (int i = warp; i < have; i += WARPS) {
            const double s = found->score[i];
            const unsigned a = found->at[i];
            int rank = 0;
            for (int j = lane; j < have; j += 32) rank += before(found->score[j], found->at[j], s, a);
            rank = __reduce_add_sync(0xffffffffu, rank);
            if (rank < take && lane == 0) {
                os[rank] = (float)s;
                ob[rank] = (int)(a / (unsigned)V);
                ot[rank] = (int)(a % (unsigned)V);
            }
        }
        for (int i = have + threadIdx.x; i < take; i += THREADS) {
            os[i] = -CUDART_INF_F;
            ob[i] = ot[i] = -1;
        }
        return;
    }
    // More scores at the threshold than the list holds (thousands of equal ones): `take` rounds over the segments that reach it, each for
    // the best behind the one before.  (Thousands reach it, so no round ends with nothing.)
    for (int k = 0; k < take; ++k) {
        double s_best = -CUDART_INF;
        unsigned a_best = 0xffffffffu;
        for (int i = warp; i < n; i += THREADS / 32) {
            if (best[i] < threshold) continue;
            const int b = i / segments;
            const float* row = logits + (row0 + b) * V;
            const int v0 = segment_start(row, i - b * segments, SEGMENT);
            for (int j = 0; j < SEGMENT / 32; ++j) {
                const int v = v0 + j * 32 + lane;
                if (v < 0 || v >= V) continue;
                const float z = row[v];
                if (!isfinite(z)) continue;
                const double s = base[b] + (double)z;
                const unsigned a = (unsigned)b * (unsigned)V + (unsigned)v;
                if ((k == 0 || before(last_score, last_at, s, a)) && before(s, a, s_best, a_best)) {
                    s_best = s;
                    a_best = a;
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double s = __shfl_xor_sync(0xffffffffu, s_best, o);
            const unsigned a = __shfl_xor_sync(0xffffffffu, a_best, o);
            if (before(s, a, s_best, a_best)) {
                s_best = s;
                a_best = a;
            }
        }
        __syncthreads();                      // the round before has been read
        if (lane == 0) {
            found->score[warp] = s_best;
            found->at[warp] = a_best;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < THREADS / 32; ++w)
                if (before(found->score[w], found->at[w], s_best, a_best)) {
                    s_best = found->score[w];
                    a_best = found->at[w];
                }
            last_score = s_best;
            last_at = a_best;
            os[k] = (float)s_best;
            ob[k] = (int)(a_best / (unsigned)V);
            ot[k] = (int)(a_best % (unsigned)V);
        }
        __syncthreads();
    }
}

// Logits per segment.  Small vocabularies get short ones, so that the threshold, the `take`-th best of 128 groups, stays near the best.
// Where 512 would keep every warp of the device busy, 1024 leave half as many numbers behind (8 x 256,000: 10.3 us, 12.1 by 512).
int least_segment(int V) { return V < 16384 ? 128 : 512; }
int segment_of(int rows, int V) { return least_segment(V) == 512 && (long long)rows * V > 148LL * 16 * 512 ? 1024 : least_segment(V); }
int segments_of(int V, int segment) { return (V + 3 + segment - 1) / segment; }
// One block does it all for few logits: a launch less, and a threshold from single logits.  us so and by two kernels: 4 beams x 1000, 8 best 6.4 /
// 8.0; 11 x 515, 22 best 9.4 / 15; 10 x 1015, 20 best 10.8 / 15.8 (where segments are few, the `take`-th of their maxima lets hundreds pass).
bool one_block(int segment, int segments, int take) { return segment == 128 && (segments <= 64 || segments <= (4 * take < 128 ? 4 * take : 128)); }

}  // namespace

// the most segments that a row is cut into, however many rows there are
QNN_API int qnn_beam_select_segments(int V) { return V <= 0 ? 0 : segments_of(V, least_segment(V)); }

// Launches of a call with these sizes.
QNN_API int qnn_beam_select_kernels(int requests, int beams, int V, int take) {
    if (requests <= 0 || V <= 0) return 0;
    const int segment = segment_of(requests * beams, V);
    return one_block(segment, beams * segments_of(V, segment), take) ? 1 : 2;
}

// logits: [requests * beams, V] float32; scores: [requests * beams]; the outputs [requests, take].  Scratch: requests * beams *
// qnn_beam_select_segments(V) float2.  take <= 64; beams * V < 2^32.
QNN_API int qnn_beam_select(const float* logits, const float* scores, int requests, int beams, int V, int take, void* scratch, float* out_scores,
                            int* out_beams, int* out_tokens, const int* status_in, int* error_flag, cudaStream_t st) {
    if (requests <= 0) return 0;
    if (beams < 1 || V < 1 || take < 1 || take > SELECT_MOST || ((uintptr_t)logits & 3)) return QNN_ERR_ARGUMENT;
    if ((long long)requests * beams > 65535 || (long long)beams * V >= 0xffffffffLL) return QNN_ERR_UNSUPPORTED;
    const int rows = requests * beams, segment = segment_of(rows, V), segments = segments_of(V, segment);
    const bool alone = one_block(segment, beams * segments, take);
    const size_t smem = sizeof(Found) + (size_t)(beams + 1) / 2 * 2 * sizeof(double) + (size_t)(beams * segments + 3) / 4 * 4 * sizeof(unsigned) +
                        (alone ? (size_t)beams * segments * (sizeof(float2) + 128 * sizeof(float)) : 0);
    if (smem > 200 * 1024 || (long long)rows * segments > 0x7fffffff) return QNN_ERR_UNSUPPORTED;
    const int total = rows * segments, wave = device_sms() * (segment >= 1024 ? 2 : 4);       // blocks of the first kernel at a time
    const int blocks = (total + 7) / 8 < wave ? (total + 7) / 8 : wave;
    float2* stats = (float2*)scratch;
#define QNN_PICK(SEG, ALONE)                                                                                                                   \
    {                                                                                                                                          \
        static OncePerDevice asked;                                                                                                            \
        if (const int rc = allow_shared(asked, beam_pick_kernel<SEG, ALONE>, 200 * 1024)) return rc;                                           \
        launch_pdl(beam_pick_kernel<SEG, ALONE>, dim3(requests), dim3(THREADS), smem, st, logits, V, beams, take, segments, scores,      \
                   (const float2*)stats, out_scores, out_beams, out_tokens, status_in, error_flag);                                            \
    }
#define QNN_SELECT(SEG)                                                                                                                        \
    {                                                                                                                                          \
        launch_pdl(beam_segments_kernel<SEG>, dim3(blocks), dim3(256), 0, st, logits, V, segments, total, stats, error_flag);                  \
        QNN_PICK(SEG, false)                                                                                                                   \
    }
    if (alone) QNN_PICK(128, true)
    else if (segment == 1024) QNN_SELECT(1024)
    else if (segment == 512) QNN_SELECT(512)
    else QNN_SELECT(128)
#undef QNN_PICK
#undef QNN_SELECT
    QNN_LAUNCH_CHECK();
}
