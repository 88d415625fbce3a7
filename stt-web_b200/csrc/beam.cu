// Beam search's selection over beams and vocabulary, and the reordering of the beams' states.
//
// Selection.  With x_b the logits of beam b and s_b its score so far, the `beams` best of
//   s_b + (x_bv - log sum_w exp(x_bw)),   ties to the lowest b * vocab + v.
// The logits are read once.  A CTA takes a chunk of a row, tile by tile through registers, and leaves a
// reference value, its sum of exponentials over it, and its `beams` best logits (no more of one row can
// be among the best of all); the last CTA of an utterance joins the rows' sums and picks among the
// chunks' bests.  The order of two beams' candidates can hang on the last digits, so sums are joined and
// candidates compared in 64 bits; the exponentials themselves are f32 over the largest logit so far, 16 or
// 32 of a thread added at a time in two chains: a sum is off by 16 * 2^-24 of itself at most, and where
// many terms are alike their roundings average out (1e-8 of the sum at 8000 normally distributed logits).
//
// The best of a chunk: the k-th largest of the maxima of its 32 groups of 4 lanes bounds the k-th best
// logit from below, and little more than the k best reach it; those few go to a list in shared memory,
// with the list's and the tiles' bounds carried from tile to tile, and are ranked by counting.  A tile
// costs a maximum, an exponential and a comparison per logit.  Where more reach the bound than the list
// takes (ties, masked rows), the warps sort them 32 at a time by a bitonic network instead.
//
// What bounds it: the latency of a CTA's chain (copy, two passes over a tile, ranking, a ticket, the last CTA's
// join) rather than memory or issue: the two batches below keep the issue slots 48% and 43% busy with 28
// instructions a logit and lane in f32 (16 logits of a thread in a tile) and 21 in bf16 (32), joins included,
// and 36% and 29% of the warps resident.  So CTAs are small, 7 or 8 of them share an SM, and tiles come by bulk
// copies, which hold no registers.  128 x 8 rows of 8000 f32 logits (32.8 MB) take 16 us with the logits in L2 and
// 19.4 us from memory, 16 x 16 rows of 65,537 bf16 logits, some ended, 26 and 29.5 us (16 logits to a thread
// cost 4 us more, CTAs of 512 threads, two to an SM, and tiles through registers 10 us more).  One utterance of 4
// beams and 8000 tokens takes 8.4 us, half of it the last CTA's join.
#include <algorithm>

#include "beam.h"
#include "kv8.cuh"
#include "tcgen05.cuh"

namespace stt {

namespace {

constexpr int kWarps = kBeamThreads / 32;
constexpr int kGroup = kBeamThreads / 32;  // lanes of a group: 32 groups give a tile's bound
static_assert(kGroup == 4, "a group lies in a warp");

// Order-preserving 32 bits of an f32 (no NaN; -0 counts as +0).
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
// Larger key: larger value, then lower index.
__device__ __forceinline__ uint64_t make_key(float x, uint32_t index) {
    return (uint64_t)ordered(x) << 32 | (uint32_t)~index;
}

// The warp's 32 keys in descending order over its lanes (bitonic).
template <class Key, class Greater, class Shuffle>
__device__ __forceinline__ Key warp_sort(Key k, int lane, Greater greater, Shuffle shuffle) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d > 0; d >>= 1) {
            const Key o = shuffle(k, d);
            const bool keep_large = ((lane & d) == 0) == ((lane & size) == 0);
            if (greater(o, k) == keep_large) k = o;
        }
    return k;
}

// A candidate of the whole utterance: its total as 64 bits that order like the f64, and beam * vocab + token.
struct Cand {
    int64_t order;
    int32_t at;  // 0x7FFFFFFF: none
};
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
    return (a.order > b.order) | ((a.order == b.order) & (a.at < b.at));  // (no branches)
}
// (no NaN; -0 counts as +0.  The map is its own inverse.)
__device__ __forceinline__ int64_t order_of(double x) {
    const int64_t u = __double_as_longlong(x + 0.0);
    return u ^ (u >> 63 & 0x7FFFFFFFFFFFFFFFll);
}
__device__ __forceinline__ double total_of(int64_t order) {
    return __longlong_as_double(order ^ (order >> 63 & 0x7FFFFFFFFFFFFFFFll));
}
// How many of the n candidates are better than c.
__device__ __forceinline__ int rank_of(const Cand& c, const Cand* cands, int n) {
    int rank = 0, j = 0;
    for (; j + 8 <= n; j += 8) {
        Cand o[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) o[u] = cands[j + u];
#pragma unroll
        for (int u = 0; u < 8; ++u) rank += better(o[u], c);
    }
    for (; j < n; ++j) rank += better(cands[j], c);
    return rank;
}

template <int DT>
__device__ __forceinline__ float to_f32(typename Elem<DT>::T x) {
    if constexpr (DT == DT_F32) return x;
    else if constexpr (DT == DT_BF16) return __bfloat162float(x);
    else return __half2float(x);
}
constexpr float kLog2e = 1.4426950408889634f;
// Maximum that a NaN wins.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A warp's best keys: lane l holds the l-th best.
struct Best {
    uint64_t top = 0;
    // Takes the 32 best of the two sets; `o` sorted as `top` is.
    __device__ __forceinline__ void merge_sorted(uint64_t o, int lane) {
        o = __shfl_sync(0xFFFFFFFFu, o, 31 - lane);
        top = o > top ? o : top;  // the 32 best of the 64, as a bitonic sequence
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const uint64_t p = __shfl_xor_sync(0xFFFFFFFFu, top, d);
            if ((p > top) == ((lane & d) == 0)) top = p;
        }
    }
    // Adds up to 32 keys (0: none), one per lane.
    __device__ __forceinline__ void merge(uint64_t k, int lane) {
        merge_sorted(warp_sort(k, lane, [](uint64_t p, uint64_t q) { return p > q; },
                               [](uint64_t p, int d) { return __shfl_xor_sync(0xFFFFFFFFu, p, d); }), lane);
    }
};

constexpr int kList = 512;      // keys of the list
constexpr int kCounted = 256;   // up to this many stay there, and are ranked by counting; more are sorted

struct Lists {
    uint64_t list[kList], pending[kWarps][64], top[kWarps][32];
};
struct Sorted {
    int listed;
    float bound;
};
// Leaves the k best, descending, of the list's first `from` keys and (row != NULL) of the row's logits
// from index v0 on, one tile, that reach the bound.  Rarely needed and long: kept out of the tile loop's
// code, whose instruction fetches it would stretch (it did: 900 cycles a tile).
template <int DT>
__device__ __noinline__ Sorted sort_list(Lists& s, int from, const typename Elem<DT>::T* row, int v0, int vocab,
                                         float bound, int k) {
    constexpr int kPerThread = beam_per_thread(DT);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    Best best;
    for (int j = 0; j < from; j += kBeamThreads) best.merge(j + tid < from ? s.list[j + tid] : 0, lane);
    if (row) {
        uint64_t* pending = s.pending[warp];
        uint64_t kth = 0;  // the warp's k-th best
        int pend = 0;
        for (int i = 0; i < kPerThread || pend > 0; ++i) {
            if (i < kPerThread) {
                const int v = v0 + (warp * kPerThread + i) * 32 + lane;
                uint64_t key = 0;
                if (v >= 0 && v < vocab) {
                    const float x = to_f32<DT>(row[v]);
                    if (x >= bound) key = make_key(x, (uint32_t)v);
                }
                const uint32_t vote = __ballot_sync(0xFFFFFFFFu, key > kth);
                if (key > kth) pending[pend + __popc(vote & ((1u << lane) - 1u))] = key;
                pend += __popc(vote);
                if (pend < 32) continue;
            }
            __syncwarp();
            best.merge(lane < pend ? pending[lane] : 0, lane);
            const uint64_t rest = lane + 32 < pend ? pending[lane + 32] : 0;
            __syncwarp();
            pending[lane] = rest;
            pend = max(0, pend - 32);
            kth = __shfl_sync(0xFFFFFFFFu, best.top, k - 1);
        }
    }
    s.top[warp][lane] = best.top;
    for (int d = kWarps / 2; d > 0; d >>= 1) {  // a tree of merges
        __syncthreads();
        if (warp < d) {
            best.merge_sorted(s.top[warp + d][lane], lane);
            s.top[warp][lane] = best.top;
        }
    }
    __syncthreads();
    Sorted r{0, bound};
    for (int j = 0; j < k; ++j) r.listed += s.top[0][j] != 0;
    if (tid < k) s.list[tid] = s.top[0][tid];
    if (r.listed == k) r.bound = fmaxf(bound, from_ordered((uint32_t)(s.top[0][k - 1] >> 32)));
    __syncthreads();
    return r;
}

template <int DT>
__global__ void __launch_bounds__(kBeamThreads, beam_ctas(DT)) select_kernel(BeamArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int VEC = 16 / (int)sizeof(T);            // elements of a 16-byte load
    constexpr int kPerThread = beam_per_thread(DT), kTile = beam_tile(DT);
    constexpr int LOADS = kPerThread / VEC;
    constexpr int kRoom = 1024;                         // candidates of an utterance that are ranked at once
    constexpr int kSlots = kRoom * sizeof(Cand) / (kTile * sizeof(T));
    static_assert(kSlots >= 2, "a tile is fetched while another is worked on");
    __shared__ __align__(128) union {
        T tiles[kSlots][kTile];                    // as they come from memory
        Cand cands[kRoom];
    } sm;
    __shared__ Lists lists_of;
    __shared__ uint64_t full[kSlots];
    __shared__ int late;
    __shared__ float wref[kWarps], group_max[2][32];
    __shared__ double wsum[kWarps];
    __shared__ uint32_t many, last, found, pushed[3];  // pushed: by the tiles, in turn
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int chunk = blockIdx.x % a.chunks, r = blockIdx.x / a.chunks;
    const int g = r / a.beams, k = a.beams;
    const int64_t part = (int64_t)r * a.chunks + chunk;
    if (tid == 0) {
        many = found = late = 0;
        pushed[0] = pushed[1] = pushed[2] = 0;
        for (int j = 0; j < kSlots; ++j) mbar_init(&full[j], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (!(a.done && a.done[r])) {
        // Tiles are cut at 16-byte boundaries of memory, whatever the row's own alignment: vector j of
        // thread t of a tile covers elements -lead + tile * kTile + (j * kBeamThreads + t) * VEC on.
        const T* row = static_cast<const T*>(a.logits) + r * a.row_stride;
        const int lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
        float ref = -INFINITY;    // the sum's reference: the warp's largest so far
        double sum = 0.0;
        float bound = -INFINITY;  // the chunk has at least k logits that reach it
        int listed = 0;           // keys of the list
        uint64_t* const list = lists_of.list;
        const int tile0 = chunk * a.tiles_per_chunk;
        const int tile1 = min(tile0 + a.tiles_per_chunk, (a.vocab + lead + kTile - 1) / kTile);
        // Vectors that lie inside the row come by a bulk copy of the tile; the row's ragged ends are put in
        // element by element.
        auto first = [&](int tile) { return tile * kTile + tid * VEC - lead; };
        auto whole = [&](int v0) { return v0 >= 0 && v0 + VEC <= a.vocab; };
        auto issue = [&](int tile) {  // by one thread
            const int v0 = tile * kTile - lead, from = v0 < 0 ? VEC : 0;
            const int to = min(kTile, (a.vocab - v0) / VEC * VEC);
            const uint32_t bytes = to > from ? (uint32_t)(to - from) * sizeof(T) : 0;
            mbar_expect_tx(&full[(tile - tile0) % kSlots], bytes);
            if (bytes) bulk_g2s(&sm.tiles[(tile - tile0) % kSlots][from], row + v0 + from, bytes, &full[(tile - tile0) % kSlots]);
        };
        auto unpack = [&](int tile, float (&x)[kPerThread]) {
            const bool inner = tile * kTile >= lead && (tile + 1) * kTile - lead <= a.vocab;
            const uint4* raw = reinterpret_cast<const uint4*>(sm.tiles[(tile - tile0) % kSlots]);
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                const int v0 = first(tile) + j * kBeamThreads * VEC;
                const uint4 r4 = raw[j * kBeamThreads + tid];
                const uint32_t w[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    float y;
                    if constexpr (DT == DT_F32) {
                        y = __uint_as_float(w[e]);
                    } else {
                        const float2 f = unpack2(w[e / 2], Elem<DT>());
                        y = e % 2 ? f.y : f.x;
                    }
                    x[j * VEC + e] = y;
                }
                if (!inner && !whole(v0)) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        x[j * VEC + e] = v0 + e >= 0 && v0 + e < a.vocab ? to_f32<DT>(row[v0 + e]) : -INFINITY;
                }
            }
        };
        if (tid == 0)
            for (int tile = tile0; tile < min(tile0 + kSlots, tile1); ++tile) issue(tile);
        // What a tile pushed is looked at after the next one's barrier (the tile's counter is its own until
        // every thread has seen it), so that a tile takes one barrier.
        uint32_t *counter = pushed, *counter1 = pushed + 1, *counter2 = pushed + 2;  // this tile's, the next's, the last's
        auto settle = [&](int tile) {
            const int now = listed + (int)*counter2;
            if (now <= kCounted) {
                listed = now;
            } else {
                const Sorted s = sort_list<DT>(lists_of, now <= kList ? now : listed, now <= kList ? nullptr : row,
                                               tile * kTile - lead, a.vocab, bound, k);
                listed = s.listed;
                bound = s.bound;
            }
        };
        float group = -INFINITY;  // the greatest of the lane's group so far
        for (int tile = tile0; tile < tile1; ++tile) {
            float x[kPerThread];
            const int base = first(tile);
            auto index = [&](int e) { return base + e / VEC * (kBeamThreads * VEC) + e % VEC; };
            mbar_wait(&full[(tile - tile0) % kSlots], (tile - tile0) / kSlots & 1, &late);
            unpack(tile, x);
            float m0 = max_nan(x[0], x[1]), m1 = max_nan(x[2], x[3]);  // (two chains)
#pragma unroll
            for (int e = 4; e < kPerThread; e += 4) m0 = max3_nan(m0, x[e], x[e + 1]), m1 = max3_nan(m1, x[e + 2], x[e + 3]);
            const float lane_max = max_nan(m0, m1);
            float mx = lane_max;
#pragma unroll
            for (int o = 1; o < kGroup; o <<= 1) mx = max_nan(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
            group = max_nan(group, mx);
            if (lane % kGroup == 0) group_max[tile & 1][tid / kGroup] = group;
#pragma unroll
            for (int o = kGroup; o < 32; o <<= 1) mx = max_nan(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
            // the warp's sum; NaN and +inf carry into it and mark the row
            if (!(mx < INFINITY)) {
                ref = INFINITY;
            } else if (mx > -INFINITY && ref < INFINITY) {
                // every larger maximum becomes the reference: a term e^d above an older one would carry the
                // rounding of its argument, 3 d 2^-24 of it (rows with a peak of 30 .. 59 in a later tile: the
                // log sum 2.7e-6 .. 5.3e-6 off; a peak that is the reference itself is exact)
                if (mx > ref) {
                    if (sum != 0.0) sum *= exp((double)ref - (double)mx);
                    ref = mx;
                }
                // e^(x - ref) as 2^((x - ref) log2 e): the argument is off by 2^-23 of its size, the power
                // by 2^-22; the difference first, since ref may be the type's lowest value
                const float2 less = make_float2(-ref, -ref), log2e = make_float2(kLog2e, kLog2e);
                float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int e = 0; e < kPerThread; e += 2) {
                    const float2 y = mul2(add2(make_float2(x[e], x[e + 1]), less), log2e);
                    s = add2(s, make_float2(exp2_approx(y.x), exp2_approx(y.y)));
                }
                sum += s.x + s.y;
            }
            if (tile + 1 == tile1) {
                double total = sum;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
                if (lane == 0) wref[warp] = ref, wsum[warp] = total;
            }
            __syncthreads();
            if (tid == 0 && tile + kSlots < tile1) issue(tile + kSlots);  // every thread has read the slot
            if (tile > tile0) settle(tile - 1);
            if (tid == 0) *counter1 = 0;
            const float gm = group_max[tile & 1][lane];
            if (bound == -INFINITY || __popc(__ballot_sync(0xFFFFFFFFu, gm > bound)) >= k) {  // (else it stays)
                // k or more sets of neighbouring groups: the least of their maxima
                uint32_t hm = ordered(gm);
                for (int o = 1, sets = 16; sets >= k && sets > 0; o <<= 1, sets >>= 1)
                    hm = max(hm, __shfl_xor_sync(0xFFFFFFFFu, hm, o));
                float least = from_ordered(__reduce_min_sync(0xFFFFFFFFu, hm));
                if (k > 8 || least == -INFINITY) {
                    // more sets than half of the groups, or sets that a short or masked row leaves empty: the
                    // k-th largest of the groups is worth the sort (at 16 beams 23 logits reach it, 54 the
                    // least of 16)
                    const uint32_t sorted = warp_sort(
                        ordered(gm), lane, [](uint32_t p, uint32_t q) { return p > q; },
                        [](uint32_t p, int d) { return __shfl_xor_sync(0xFFFFFFFFu, p, d); });
                    least = from_ordered(__shfl_sync(0xFFFFFFFFu, sorted, k - 1));
                }
                bound = fmaxf(bound, least);
            }
            if (lane_max >= bound) {
                uint32_t reach = 0;
#pragma unroll
                for (int e = 0; e < kPerThread; ++e) reach |= (uint32_t)(x[e] >= bound) << e;
                if (bound == -INFINITY) {  // the places outside the row count as -inf: not candidates
#pragma unroll
                    for (int e = 0; e < kPerThread; ++e)
                        if (index(e) < 0 || index(e) >= a.vocab) reach &= ~(1u << e);
                }
                const uint32_t mine = __popc(reach);
                uint32_t at = listed + atomicAdd(counter, mine);
                if (mine == 1) {  // as a rule
                    if (at < kList) list[at] = make_key(lane_max, (uint32_t)index(__ffs(reach) - 1));
                } else {
                    for (; reach; reach &= reach - 1, ++at) {
                        const int v = index(__ffs(reach) - 1);
                        if (at < kList) list[at] = make_key(to_f32<DT>(row[v]), (uint32_t)v);
                    }
                }
            }
            uint32_t* const t = counter2;
            counter2 = counter, counter = counter1, counter1 = t;
        }
        __syncthreads();
        if (tile1 > tile0) settle(tile1 - 1);
        if (tile1 <= tile0) {  // the row ends before this chunk
            if (lane == 0) wref[warp] = -INFINITY, wsum[warp] = 0.0;
            __syncthreads();
        }
        if (warp == kWarps - 1) {
            const float m = lane < kWarps ? wref[lane] : -INFINITY;
            float top = m;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            double s = m > -INFINITY && top < INFINITY ? wsum[lane] * exp((double)m - (double)top) : 0.0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            if (lane == 0) a.part_max[part] = top, a.part_sum[part] = s;
        }
        // the k best of the list, among those that reach the last bound: a key's rank is the number of larger ones
        uint64_t* out = a.part_keys + part * a.key_stride;
        uint64_t* const left = lists_of.pending[0];
        static_assert(kWarps * 64 >= kCounted, "the list's keys have room");
        for (int q = tid; q < listed; q += kBeamThreads)
            if ((uint32_t)(list[q] >> 32) >= ordered(bound)) left[atomicAdd(&found, 1u)] = list[q];
        __syncthreads();
        listed = (int)found;
        for (int q = tid; q < listed; q += kBeamThreads) {
            const uint64_t key = left[q];
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < listed; ++j) rank += left[j] > key;
            if (rank < k) out[rank] = key;
        }
        if (tid >= listed && tid < k) out[tid] = 0;  // a chunk of fewer elements
    }
    __syncthreads();
    if (tid == 0 && late) atomicCAS(a.err, 0, -5);  // STT_E_DEVICE_FLAG: a copy that never came
    if (tid == 0) last = ticket(a.tickets + g) == (uint32_t)(a.beams * a.chunks - 1);
    __syncthreads();
    if (!last) return;

    // ---- the utterance: log sums of its beams, then the best of the chunks' bests
    __shared__ double lse[kMaxBeams], score[kMaxBeams];
    __shared__ float rmax[kMaxBeams];
    __shared__ uint8_t state[kMaxBeams], over[kMaxBeams];  // state 0 live, 1 ended, 2 all candidates at -inf
    const int64_t row0 = (int64_t)g * k;
    static_assert(kBeamMaxChunks <= 32, "a lane joins one chunk");
    int per_beam = 1;  // lanes of a beam
    while (per_beam < a.chunks) per_beam <<= 1;
    for (int b0 = warp * (32 / per_beam); b0 < k; b0 += kBeamThreads / per_beam) {
        const int b = b0 + lane / per_beam, at = lane % per_beam;
        const bool real = b < k;
        const bool end_b = real && a.done && a.done[row0 + b], here = real && !end_b && at < a.chunks;
        const int64_t p = (row0 + b) * a.chunks + at;
        const float s = real ? a.scores[row0 + b] : 0.0f;
        const float mc = here ? __ldcg(a.part_max + p) : -INFINITY;
        double sum = here ? __ldcg(a.part_sum + p) : 0.0;
        float m = mc;
        if (a.chunks > 1) {
            for (int o = per_beam / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            sum = mc > -INFINITY && m < INFINITY ? sum * exp((double)mc - (double)m) : 0.0;
            for (int o = per_beam / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        }
        if (real && at == 0) {
            const bool bad = !(s < INFINITY) || (!end_b && m == INFINITY);
            if (bad) atomicCAS(a.err, 0, -5);  // STT_E_DEVICE_FLAG
            const int st = bad || s == -INFINITY || (!end_b && m == -INFINITY) ? 2 : end_b ? 1 : 0;
            state[b] = (uint8_t)st;
            over[b] = end_b;
            score[b] = s;
            rmax[b] = m;
            if (st == 0) lse[b] = log(sum);
        }
    }
    __syncthreads();
    // List l = beam * chunks + chunk holds k candidates, best first.
    const int lists = k * a.chunks;
    const int64_t lowest = order_of(-INFINITY);
    const Cand kNone{lowest, 0x7FFFFFFF};
    auto candidate = [&](int l, int j) {
        const int b = l / a.chunks;
        Cand c = kNone;
        if (state[b] == 0) {
            const uint64_t key = __ldcg(a.part_keys + (row0 * a.chunks + l) * a.key_stride + j);
            if (key == 0) return c;
            const double x = from_ordered((uint32_t)(key >> 32));
            c.order = order_of(((x - (double)rmax[b]) - lse[b]) + score[b]);
            c.at = b * a.vocab + (int)~(uint32_t)key;
            return c;
        }
        // a beam that ended offers its end token, then the lowest of the others at -inf; a beam with
        // nothing to offer its lowest tokens at -inf
        if (l % a.chunks != 0) return c;
        int token = j;
        if (state[b] == 1 && a.eos >= 0 && a.eos < a.vocab) {
            if (j == 0) c.order = order_of(score[b]);
            token = j == 0 ? a.eos : j - 1 < a.eos ? j - 1 : j;
        }
        if (token < a.vocab) c.at = b * a.vocab + token;
        return c;
    };
    auto write = [&](int rank, const Cand& c) {
        const int b = c.at / a.vocab, token = c.at % a.vocab;
        const int64_t o = row0 + rank;
        a.next_scores[o] = (float)total_of(c.order);
        a.parents[o] = b;
        a.tokens[o] = token;
        if (a.next_done) a.next_done[o] = over[b] || token == a.eos;
    };
    // The lists that can hold one of the k best: where there are more than k, those with the k best first
    // candidates (fewer than k may have one), best first; then candidate j of the list at place p counts if
    // p + j < k and it reaches the k-th best of the first ones.
    Cand L = kNone;
    Cand* cands = sm.cands;
    __shared__ Cand limit;
    __shared__ int alive[kMaxBeams];
    int places = lists;
    if (lists > k) {
        if (tid == 0) limit = kNone, found = 0;
        for (int l = tid; l < lists; l += kBeamThreads) cands[l] = candidate(l, 0);
        __syncthreads();
        for (int l = tid; l < lists; l += kBeamThreads) {
            const Cand c = cands[l];
            if (c.at == 0x7FFFFFFF) continue;
            const int rank = rank_of(c, cands, lists);
            if (rank < k) alive[rank] = l, atomicAdd(&found, 1u);
            if (rank == k - 1) limit = c;
        }
        __syncthreads();
        L = limit;
        places = (int)found;
    }
    for (int q = tid; q < places * k; q += kBeamThreads) {
        const int p = q / k, j = q % k;
        if (lists > k && p + j >= k) continue;
        const Cand c = candidate(lists > k ? alive[p] : p, j);
        if (c.at == 0x7FFFFFFF || better(L, c)) continue;
        cands[atomicAdd(&many, 1u)] = c;
    }
    static_assert(kMaxBeams * kMaxBeams <= kRoom && kBeamThreads <= kRoom, "all that count, and the lists' first ones, have room");
    __syncthreads();
    const int n = (int)many;
    for (int q = tid; q < n; q += kBeamThreads) {
        const Cand c = cands[q];
        const int rank = rank_of(c, cands, n);
        if (rank < k) write(rank, c);
    }
    if (tid == 0) a.tickets[g] = 0u;
}

// ---- reordering

// Units of a group's rows are moved position by position: a thread loads its position of every row
// that another beam takes, then stores it to the beams that change.  All of a position is read
// before any of it is written, and no other thread touches it, so the rows are permuted in place,
// with each source read once (a beam that two others take is read twice, the second time from L1).
// HBM bounds it: 32 x 8 rows of 64 pieces of up to 751 x 256 bytes take 565 us for 3.4 GB, 5.9 TB/s.
// FLAT: segments that do not fill a CTA are taken one after another, so that its threads all have work
// (64 x 16 rows of 200 segments of 3 units of 144 bytes: 22 us, with a CTA to each segment 102 us).
template <int B, class V, int U, bool FLAT>
__global__ void __launch_bounds__(256) reorder_kernel(ReorderArgs a, int64_t per_segment) {
    __shared__ int parent[B];
    __shared__ int64_t place[B];
    __shared__ int64_t limit[B];
    const int g = blockIdx.z;
    const int64_t row0 = (int64_t)g * a.beams;
    const int64_t per_unit = a.unit_bytes / (int64_t)sizeof(V);
    for (int b = threadIdx.x; b < B; b += 256) {
        int p = b < a.beams ? __ldg(a.parents + row0 + b) : b;
        if (p < 0 || p >= a.beams) p = b;  // keeps its own
        int64_t m = a.units;
        if (a.held && b < a.beams) {
            const int64_t held = __ldg(a.held + row0 + b);
            m = held <= 0 ? 0 : min((held + a.per_unit - 1) / a.per_unit, a.units);
        }
        parent[b] = p;
        place[b] = (a.rows && b < a.beams ? __ldg(a.rows + row0 + b) : row0 + b) * a.row_stride;
        limit[b] = p == b ? 0 : m * per_unit;
    }
    __syncthreads();
    uint8_t* base[U];  // of the thread's U segments, and its positions in them
    int64_t q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        q[u] = (int64_t)blockIdx.x * 256 * U + u * 256 + threadIdx.x;
        int s = blockIdx.y;
        if constexpr (FLAT) {  // (fewer than 2^31: 65535 segments of fewer than 1024 positions)
            const uint32_t at = (uint32_t)q[u], per = (uint32_t)per_segment;
            s = (int)(at / per);
            q[u] = s < a.segments ? (int64_t)(at % per) : INT64_MAX;
        }
        s += a.first_segment;
        base[u] = a.states + (s / a.inner) * a.outer_stride + (s % a.inner) * a.segment_stride;
    }
    V v[U][B];
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (q[u] < limit[b]) v[u][b] = *reinterpret_cast<const V*>(base[u] + place[parent[b]] + q[u] * sizeof(V));
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (q[u] < limit[b]) *reinterpret_cast<V*>(base[u] + place[b] + q[u] * sizeof(V)) = v[u][b];
}

template <int B, class V, int U>
cudaError_t reorder_t(const ReorderArgs& a, cudaStream_t st) {
    const int64_t per_segment = a.units * a.unit_bytes / (int64_t)sizeof(V);
    const bool flat = per_segment < 256 * U;
    // grid y and z end at 65535: more segments or groups than that go in several launches
    for (int g0 = 0; g0 < a.groups; g0 += 65535)
        for (int s0 = 0; s0 < a.segments; s0 += 65535) {
            ReorderArgs b = a;
            b.groups = std::min(65535, a.groups - g0);
            b.segments = std::min(65535, a.segments - s0);
            if (b.rows) b.rows += (int64_t)g0 * a.beams;
            else b.states += (int64_t)g0 * a.beams * a.row_stride;
            b.first_segment = s0;
            b.parents += (int64_t)g0 * a.beams;
            if (b.held) b.held += (int64_t)g0 * a.beams;
            const int64_t x = ((flat ? b.segments * per_segment : per_segment) + 256 * U - 1) / (256 * U);
            if (flat) reorder_kernel<B, V, U, true><<<dim3((unsigned)x, 1, b.groups), 256, 0, st>>>(b, per_segment);
            else reorder_kernel<B, V, U, false><<<dim3((unsigned)x, b.segments, b.groups), 256, 0, st>>>(b, per_segment);
            const cudaError_t e = cudaGetLastError();
            if (e != cudaSuccess) return e;
        }
    return cudaSuccess;
}

template <class V>
cudaError_t reorder_v(const ReorderArgs& a, cudaStream_t st) {
    if (a.beams <= 4) return reorder_t<4, V, 4>(a, st);
    if (a.beams <= 8) return reorder_t<8, V, 2>(a, st);
    if (a.beams <= 16) return reorder_t<16, V, 1>(a, st);
    return reorder_t<32, V, 1>(a, st);
}

}  // namespace

cudaError_t launch_beam_select(const BeamArgs& a, int dtype, cudaStream_t st) {
    const unsigned grid = (unsigned)((int64_t)a.batch * a.beams * a.chunks);
    if (dtype == DT_F32) select_kernel<DT_F32><<<grid, kBeamThreads, 0, st>>>(a);
    else if (dtype == DT_BF16) select_kernel<DT_BF16><<<grid, kBeamThreads, 0, st>>>(a);
    else select_kernel<DT_F16><<<grid, kBeamThreads, 0, st>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_reorder(const ReorderArgs& a, cudaStream_t st) {
    if (a.units <= 0 || a.segments <= 0 || a.groups <= 0 || a.beams <= 1) return cudaSuccess;
    // the widest access that the base, the strides and the unit allow
    const uint64_t bits = reinterpret_cast<uintptr_t>(a.states) | (uint64_t)a.row_stride | (uint64_t)a.segment_stride |
                          (uint64_t)a.outer_stride | (uint64_t)a.unit_bytes;
    if (bits % 16 == 0) return reorder_v<uint4>(a, st);
    if (bits % 4 == 0) return reorder_v<uint32_t>(a, st);
    return reorder_v<uint8_t>(a, st);
}

}  // namespace stt
