// Beam search's selection over beams and vocabulary, and the reordering of the beams' states.
//
// Selection.  With x_b the logits of beam b and s_b its score so far, the `beams` best of
//   s_b + (x_bv - max x_b - log sum_w exp(x_bw - max x_b)),   ties to the lowest b * vocab + v.
// The logits are read once.  A CTA takes a chunk of a row into registers and leaves its maximum, its
// sum of exponentials and its `beams` best logits (no more of one row can be among the best of all);
// the last CTA of an utterance adds up the rows' sums and picks among the chunks' bests.  The order
// of two beams' candidates can hang on the last digits, so sums are joined and candidates compared in
// 64 bits; the exponentials themselves are f32 (their rounding errors, 2^-24 each, average out).
//
// The `beams` best of a chunk without sorting it: each warp sorts its 32 lanes' maxima, the beams-th of
// them is a lower bound of the chunk's beams-th best, the largest bound of the 8 warps leaves little
// more than the `beams` best themselves, and those few are ranked by counting.
#include "beam.h"

#include <algorithm>

#include "kv8.cuh"

namespace stt {

namespace {

constexpr int kWarps = kBeamThreads / 32;

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

// A candidate of the whole utterance.
struct Cand {
    double total;
    int32_t at;  // beam * vocab + token; 0x7FFFFFFF: none
};
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
    return a.total > b.total || (a.total == b.total && a.at < b.at);
}

template <int DT>
__device__ __forceinline__ float to_f32(typename Elem<DT>::T x) {
    if constexpr (DT == DT_F32) return x;
    else if constexpr (DT == DT_BF16) return __bfloat162float(x);
    else return __half2float(x);
}

template <int DT>
__global__ void __launch_bounds__(kBeamThreads) select_kernel(BeamArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int VEC = 16 / (int)sizeof(T);            // elements of a 16-byte load
    constexpr int LOADS = kBeamPerThread / VEC;
    __shared__ uint64_t list[kBeamChunk];
    __shared__ uint64_t bound[kWarps];
    __shared__ float wmax[kWarps];
    __shared__ double wsum[kWarps];
    __shared__ uint32_t many, last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int chunk = blockIdx.x % a.chunks, r = blockIdx.x / a.chunks;
    const int g = r / a.beams, k = a.beams;
    const int64_t part = (int64_t)r * a.chunks + chunk;
    const bool ended = a.done && a.done[r];
    if (tid == 0) many = 0;
    if (!ended) {
        // The chunk is cut at 16-byte boundaries of memory, whatever the row's own alignment: vector j
        // of thread t covers elements from -lead + (chunk * CTA + j * 256 + t) * VEC on.
        const T* row = static_cast<const T*>(a.logits) + r * a.row_stride;
        const int lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
        float x[kBeamPerThread];
        int base[LOADS];
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            base[j] = (chunk * (kBeamChunk / VEC) + j * kBeamThreads + tid) * VEC - lead;
            if (base[j] >= 0 && base[j] + VEC <= a.vocab) {
                float y[VEC];
                if constexpr (DT == DT_F32) load_elems<DT, 4>(row + base[j], y);
                else load_elems<DT, 8>(row + base[j], y);
#pragma unroll
                for (int e = 0; e < VEC; ++e) x[j * VEC + e] = y[e];
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int v = base[j] + e;
                    x[j * VEC + e] = v >= 0 && v < a.vocab ? to_f32<DT>(row[v]) : -INFINITY;
                }
            }
        }
        uint64_t best = 0;
        float mx = -INFINITY;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < kBeamPerThread; ++e) {
            const int v = base[e / VEC] + e % VEC;
            bad |= !(x[e] < INFINITY);  // NaN or +inf
            mx = fmaxf(mx, x[e]);
            if (v >= 0 && v < a.vocab) {
                const uint64_t key = make_key(x[e], (uint32_t)v);
                best = key > best ? key : best;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
        float sum = 0.0f;
        if (mx > -INFINITY) {
#pragma unroll
            for (int e = 0; e < kBeamPerThread; ++e) sum += expf(x[e] - mx);
        }
        double total = sum;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
        const uint64_t sorted = warp_sort(
            best, lane, [](uint64_t p, uint64_t q) { return p > q; },
            [](uint64_t p, int d) { return __shfl_xor_sync(0xFFFFFFFFu, p, d); });
        const uint64_t mine = __shfl_sync(0xFFFFFFFFu, sorted, k - 1);
        if (__any_sync(0xFFFFFFFFu, bad)) mx = INFINITY;  // marks the row
        if (lane == 0) wmax[warp] = mx, wsum[warp] = total, bound[warp] = mine;
        __syncthreads();
        uint64_t T0 = 1;  // every element's key is above 0, the key of no element
#pragma unroll
        for (int w = 0; w < kWarps; ++w) T0 = bound[w] > T0 ? bound[w] : T0;
#pragma unroll
        for (int e = 0; e < kBeamPerThread; ++e) {
            const int v = base[e / VEC] + e % VEC;
            if (v < 0 || v >= a.vocab) continue;
            const uint64_t key = make_key(x[e], (uint32_t)v);
            if (key >= T0) list[atomicAdd(&many, 1u)] = key;
        }
        __syncthreads();
        const int n = (int)many;
        uint64_t* out = a.part_keys + part * a.key_stride;
        for (int q = tid; q < n; q += kBeamThreads) {
            const uint64_t key = list[q];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += list[j] > key;
            if (rank < k) out[rank] = key;
        }
        for (int q = n + tid; q < k; q += kBeamThreads) out[q] = 0;  // a chunk of fewer elements
        if (tid == 0) {
            float m = wmax[0];
            for (int w = 1; w < kWarps; ++w) m = fmaxf(m, wmax[w]);
            double s = 0.0;
            if (m > -INFINITY && m < INFINITY)
                for (int w = 0; w < kWarps; ++w)
                    if (wmax[w] > -INFINITY) s += wsum[w] * exp((double)wmax[w] - (double)m);
            a.part_max[part] = m;
            a.part_sum[part] = s;
        }
    }
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicAdd(a.tickets + g, 1u) == (uint32_t)(a.beams * a.chunks - 1);
    __syncthreads();
    if (!last) return;
    __threadfence();

    // ---- the utterance: log sums of its beams, then the best of the chunks' bests
    __shared__ double lse[kMaxBeams], score[kMaxBeams];
    __shared__ float rmax[kMaxBeams];
    __shared__ uint8_t state[kMaxBeams], over[kMaxBeams];  // state 0 live, 1 ended, 2 all candidates at -inf
    const int64_t row0 = (int64_t)g * k;
    for (int b = warp; b < k; b += kWarps) {
        const int64_t p0 = (row0 + b) * a.chunks;
        const bool end_b = a.done && a.done[row0 + b];
        const float s = a.scores[row0 + b];
        float m = -INFINITY;
        if (!end_b)
            for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, __ldcg(a.part_max + p0 + c));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        double sum = 0.0;
        if (!end_b && m > -INFINITY && m < INFINITY)
            for (int c = lane; c < a.chunks; c += 32) {
                const float mc = __ldcg(a.part_max + p0 + c);
                if (mc > -INFINITY) sum += __ldcg(a.part_sum + p0 + c) * exp((double)mc - (double)m);
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (lane == 0) {
            const bool bad = !(s < INFINITY) || (!end_b && m == INFINITY);
            if (bad) atomicCAS(a.err, 0, -5);  // STT_E_DEVICE_FLAG
            state[b] = bad || s == -INFINITY || (!end_b && m == -INFINITY) ? 2 : end_b ? 1 : 0;
            over[b] = end_b;
            score[b] = s;
            rmax[b] = m;
            lse[b] = log(sum);
        }
    }
    if (tid == 0) many = 0;
    __syncthreads();
    // List l = beam * chunks + chunk holds k candidates, best first.
    const int lists = k * a.chunks;
    constexpr Cand kNone{-INFINITY, 0x7FFFFFFF};
    auto candidate = [&](int l, int j) {
        const int b = l / a.chunks;
        Cand c = kNone;
        if (state[b] == 0) {
            const uint64_t key = __ldcg(a.part_keys + (row0 * a.chunks + l) * a.key_stride + j);
            if (key == 0) return c;
            const double x = from_ordered((uint32_t)(key >> 32));
            c.total = ((x - (double)rmax[b]) - lse[b]) + score[b];
            c.at = b * a.vocab + (int)~(uint32_t)key;
            return c;
        }
        // a beam that ended offers its end token, then the lowest of the others at -inf; a beam with
        // nothing to offer its lowest tokens at -inf
        if (l % a.chunks != 0) return c;
        int token = j;
        if (state[b] == 1 && a.eos >= 0 && a.eos < a.vocab) {
            if (j == 0) c.total = score[b];
            token = j == 0 ? a.eos : j - 1 < a.eos ? j - 1 : j;
        }
        if (token < a.vocab) c.at = b * a.vocab + token;
        return c;
    };
    auto write = [&](int rank, const Cand& c) {
        const int b = c.at / a.vocab, token = c.at % a.vocab;
        const int64_t o = row0 + rank;
        a.next_scores[o] = (float)c.total;
        a.parents[o] = b;
        a.tokens[o] = token;
        if (a.next_done) a.next_done[o] = over[b] || token == a.eos;
    };
    auto shuffle = [](const Cand& c, int d) {
        return Cand{__shfl_xor_sync(0xFFFFFFFFu, c.total, d), __shfl_xor_sync(0xFFFFFFFFu, c.at, d)};
    };
    // the bound as above, from the lists' first candidates
    __shared__ Cand limit[kWarps];
    Cand best = kNone;
    for (int l = tid; l < lists; l += kBeamThreads) {
        const Cand c = candidate(l, 0);
        if (better(c, best)) best = c;
    }
    const Cand sorted = warp_sort(best, lane, better, shuffle);
    if (lane == k - 1) limit[warp] = sorted;
    __syncthreads();
    Cand L = limit[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w)
        if (better(limit[w], L)) L = limit[w];
    Cand* cands = reinterpret_cast<Cand*>(list);
    constexpr int kRoom = (int)(sizeof(list) / sizeof(Cand));
    for (int l = tid; l < lists; l += kBeamThreads)
        for (int j = 0; j < k; ++j) {
            const Cand c = candidate(l, j);
            if (c.at == 0x7FFFFFFF || better(L, c)) break;
            const uint32_t at = atomicAdd(&many, 1u);
            if (at < kRoom) cands[at] = c;
        }
    __syncthreads();
    const int n = (int)many;
    if (n <= kRoom) {
        for (int q = tid; q < n; q += kBeamThreads) {
            const Cand c = cands[q];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += better(cands[j], c);
            if (rank < k) write(rank, c);
        }
    } else {
        // more than the list holds (a bound that a few poor lists pulled down): merged best by best
        Cand prev{INFINITY, -1};
        for (int rank = 0; rank < k; ++rank) {
            best = kNone;
            for (int l = tid; l < lists; l += kBeamThreads)
                for (int j = 0; j < k; ++j) {
                    const Cand c = candidate(l, j);
                    if (!better(c, best)) break;
                    if (better(prev, c)) {
                        best = c;
                        break;
                    }
                }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
                const Cand o = shuffle(best, d);
                if (better(o, best)) best = o;
            }
            __syncthreads();
            if (lane == 0) limit[warp] = best;
            __syncthreads();
            for (int w = 0; w < kWarps; ++w)
                if (better(limit[w], best)) best = limit[w];
            if (tid == 0) write(rank, best);
            prev = best;
        }
    }
    if (tid == 0) a.tickets[g] = 0u;
}

// ---- reordering

// Units of a group's rows are moved position by position: a thread loads its position of every row
// that another beam takes, then stores it to the beams that change.  All of a position is read
// before any of it is written, and no other thread touches it, so the rows are permuted in place,
// with each source read once (a beam that two others take is read twice, the second time from L1).
template <int B, class V, int U>
__global__ void __launch_bounds__(256) reorder_kernel(ReorderArgs a, int64_t per_segment) {
    __shared__ int parent[B];
    __shared__ int64_t limit[B];
    const int g = blockIdx.z, s = a.first_segment + blockIdx.y;
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
        limit[b] = p == b ? 0 : m * per_unit;
    }
    __syncthreads();
    uint8_t* base = a.states + row0 * a.row_stride + (s / a.inner) * a.outer_stride + (s % a.inner) * a.segment_stride;
    const int64_t first = (int64_t)blockIdx.x * 256 * U + threadIdx.x;
    V v[U][B];
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t q = first + u * 256;
            if (q < limit[b]) v[u][b] = *reinterpret_cast<const V*>(base + parent[b] * a.row_stride + q * sizeof(V));
        }
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t q = first + u * 256;
            if (q < limit[b]) *reinterpret_cast<V*>(base + b * a.row_stride + q * sizeof(V)) = v[u][b];
        }
}

template <int B, class V, int U>
cudaError_t reorder_t(const ReorderArgs& a, cudaStream_t st) {
    const int64_t per_segment = a.units * a.unit_bytes / (int64_t)sizeof(V);
    const int64_t x = (per_segment + 256 * U - 1) / (256 * U);
    // grid y and z end at 65535: more segments or groups than that go in several launches
    for (int g0 = 0; g0 < a.groups; g0 += 65535)
        for (int s0 = 0; s0 < a.segments; s0 += 65535) {
            ReorderArgs b = a;
            b.groups = std::min(65535, a.groups - g0);
            b.segments = std::min(65535, a.segments - s0);
            b.states += (int64_t)g0 * a.beams * a.row_stride;
            b.first_segment = s0;
            b.parents += (int64_t)g0 * a.beams;
            if (b.held) b.held += (int64_t)g0 * a.beams;
            reorder_kernel<B, V, U><<<dim3((unsigned)x, b.segments, b.groups), 256, 0, st>>>(b, per_segment);
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
