// Attention over the 8-bit K/V cache.
//
// For query row r (a token and a query head of the K/V head h) at position P:
//   out = sum_p softmax_p(scale * q . k_p) v_p   over   max(start, P + 1 - window, ring) <= p <= P,
// zeros where no position is left.  In base 2, s_p = log2(e) * scale * q . k_p, and V's block exponents
// are folded into the weights:
//   w_p = 2^(s_p + e_v(p) - M),   O = sum w_p * code_p,   l = sum w_p * 2^-e_v(p),   out = O / l,
// with M the running maximum of s_p + e_v(p).  One pass over the codes keeps (M, l, O) per row.  M moves
// only when it falls more than 8 behind, so that O is rescaled a few times per row.
// What this holds: w is two f16 parts, scaled by 2^7, so a key's share of O is lost where s_p + e_v(p) is 2^32
// below the row's largest; l is f32, and a key's share of it is lost where s_p + e_v(p) is 2^133 below: as
// long as V's exponents lie within 110 of one another, only keys with less than 2^-23 of the largest share are.
//
// What bounds it: a decode step reads 2 * dim bytes per position and head and does 4 * dim flops per
// query row with them, so HBM bounds it as long as turning codes into operands costs little.  Hence
//  - the codes go through mma.sync.m16n8k16 f16 with f32 accumulation.  A code is exact in f16: the
//    bytes (code + 128) under the high byte 0x64 are the f16 value 1024 + 128 + code, one subtraction
//    away, 2.5 instructions for 4 codes.  tcgen05 would want the converted tile in shared or tensor
//    memory first, one more trip for an operand that is used by a handful of rows;
//  - q and the weights are split into two f16 parts (x = hi + lo, 22 bits), so scores and outputs keep
//    f32 quality.  Up to 8 query rows: the parts are rows 0-7 and 8-15 of the A operand, the codes the B
//    operand, and the scores' accumulator is the layout of the second product's A operand.  Up to 4 rows
//    (a single token of up to 4 query heads per K/V head): the other way round, the codes are the 16
//    rows of A and the parts are columns 0-3 and 4-7 of B, which takes half the products and half the
//    accumulators (so 4 CTAs fit an SM instead of 3), for one transposition of the weights per block;
//  - any order of dimensions serves as long as both operands agree, so no code is shuffled: a lane's
//    operand for K is 16 consecutive codes of one key, for V 16 consecutive codes of its 4 keys;
//  - every warp streams its own blocks of 16 keys through a private ring in shared memory
//    (cp.async, 16 bytes per lane), without block-wide barriers, and the 4 warps are merged at the end;
//  - where there are fewer (row, head) items than CTAs fit, an item's blocks are cut into runs for the CTAs
//    of a cluster, joined through distributed shared memory, and beyond that into parts joined through
//    global memory, the last part to finish doing it (cut_items chooses).
// Measured (time of a launch): 512 sequences x 16 heads x 751 positions 267 us for 1.61 GB, 6.0 TB/s (281 us from
// cold caches); with a ring of 4,096 the same at 130 positions 119 us, at 4,000 1.22 ms; 4 sequences x 8 heads of up to
// 65,521 positions, 4 query heads each, 105 us for 0.51 GB, 4.9 TB/s; 1 sequence x 16 heads: 130 positions 6.6 us,
// 751 positions 7.5 us; 64 sequences x 751 positions 41 us.  Chunks with f32 on either side come here too, 8 rows
// at a time: the last 1024 of 4096 positions of 4 x 16 heads take 1.65 ms, where 16-bit ones take 149 us on the
// other kernel.
#include <cfloat>
#include <climits>
#include <algorithm>

#include "kv8_attn.cuh"
#include "tcgen05.cuh"

namespace stt {

namespace {

constexpr int kWarps = 4;
constexpr int kMaxParts = 64;
constexpr int kMaxCluster = 8;
constexpr int kMinBlocks = 4;   // of a warp in a part that is joined through memory
// Query rows of a CTA, stages of a warp's ring, CTAs per SM.
template <bool NARROW>
struct Shape {
    static constexpr int kRows = NARROW ? 4 : 8, kStages = NARROW ? 3 : 4, kCtas = NARROW ? 4 : 3;
};
constexpr float kWeightShift = 7.0f;  // weights are scaled by 2^7: at most 2^15 in f16, normal down to 2^-21
constexpr float kLazy = 8.0f;         // how far s + e_v may exceed M

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Transposes the 8 x 8 matrix of 16-bit elements that the warp holds two to a lane, row g columns 2t, 2t + 1.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// x = hi + lo in f16, for two values.
__device__ __forceinline__ void split2(float a, float b, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    *hi = *reinterpret_cast<const uint32_t*>(&h);
    *lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Byte offset of 16-byte piece `c` of key row `r` in a staged block of K or V.  The permutations
// make the reads below conflict-free: a quarter warp reads K rows {2i, 2i+1} x 4 pieces, and V rows
// {0, 2, 4, 6} (or the others of its residue) x 2 pieces (dim 128) or 4 half pieces (dim 64).
template <int D>
__device__ __forceinline__ int k_piece(int r, int c) {
    return D == 128 ? r * 128 + ((c ^ (4 * (r & 1))) << 4) : r * 64 + (c << 4);
}
template <int D>
__device__ __forceinline__ int v_piece(int r, int c) {
    if (D == 128) return r * 128 + ((c ^ (2 * ((r >> 1) & 3))) << 4);
    return (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (2 * ((r >> 1) & 3))) << 4);
}

// One row's softmax state in base 2.
struct RowState {
    float M, l;
};

template <int DT>
__device__ __forceinline__ void load16(const void* base, int64_t at, float (&x)[16]) {
    const typename Elem<DT>::T* p = static_cast<const typename Elem<DT>::T*>(base) + at;
    float a[8], b[8];
    load_elems<DT, 8>(p, a);
    load_elems<DT, 8>(p + 8, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = a[i], x[8 + i] = b[i];
}
__device__ __forceinline__ void load16(const void* base, int dtype, int64_t at, float (&x)[16]) {
    if (dtype == DT_F32) load16<DT_F32>(base, at, x);
    else if (dtype == DT_BF16) load16<DT_BF16>(base, at, x);
    else load16<DT_F16>(base, at, x);
}

// Merges the softmax states of `n` parts and returns the row's output piece O / l times 2^-M.
// State and piece of part j come from the two functions; an empty part has l = 0.
template <class State, class Piece>
__device__ __forceinline__ RowState merge_parts(int n, State state, Piece piece, float4* out) {
    RowState r{-FLT_MAX, 0.0f};
#pragma unroll
    for (int j = 0; j < n; ++j) {
        const RowState s = state(j);
        if (s.l != 0.0f) r.M = fmaxf(r.M, s.M);
    }
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < n; ++j) {
        const RowState s = state(j);
        if (s.l == 0.0f) continue;
        const float f = exp2f(s.M - r.M);
        r.l = fmaf(s.l, f, r.l);
        const float4 p = piece(j);
        o.x = fmaf(p.x, f, o.x), o.y = fmaf(p.y, f, o.y), o.z = fmaf(p.z, f, o.z), o.w = fmaf(p.w, f, o.w);
    }
    *out = o;
    return r;
}
__device__ __forceinline__ float4 row_output(const RowState& r, float4 o) {
    if (r.l == 0.0f) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float f = 1.0f / r.l;
    return make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
}

// CTA (((batch row * groups + row group) * heads + head) * max_parts + part) * cluster + rank.  An
// item's keys are cut into parts x cluster equal runs of blocks; a cluster joins its runs through shared
// memory, the last cluster of an item its parts through global memory.
// SUMS: a block's products are added to O by f32 additions, not by the products' own accumulators (attend_sums).
template <int D, bool NARROW, bool SUMS>
__global__ void __launch_bounds__(kWarps * 32, Shape<NARROW>::kCtas) attend_kernel(Kv8Dev c, Kv8Batch b, Kv8Attention a, int groups,
                                                                int max_parts, int cluster) {
    constexpr int KS = D / 16;          // k steps of the first product
    constexpr int NT = NARROW ? D / 16 : D / 8;  // tiles of 16 (8) dimensions of the second
    constexpr int ROWS = Shape<NARROW>::kRows, kStages = Shape<NARROW>::kStages;
    constexpr int HALF = 16 * D;        // bytes of a staged block of K (and of V)
    constexpr int CH = D / 16;          // 16-byte pieces of a row
    constexpr int VB = D / 8;           // bytes of V that a lane takes of a key
    constexpr int VW = VB / 4;          // in words
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ RowState sm_state[kWarps][ROWS];
    __shared__ RowState own_state[ROWS];
    __shared__ uint32_t last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % cluster, part_of = blockIdx.x / cluster % max_parts, item = blockIdx.x / cluster / max_parts;
    const int h = item % c.heads, rg = item / c.heads % groups, i = item / c.heads / groups;
    Kv8Row row;
    if (!kv8_row(c, b, i, &row)) return;
    // the group's rows: row r is token r / group, query head h * group + r % group
    const int r0 = rg * ROWS;
    const int rows = min(ROWS, row.count * a.group - r0);
    if (rows <= 0) return;
    const int t0 = r0 / a.group, t1 = (r0 + rows - 1) / a.group;
    Sight sight;
    sight.start = a.start ? max(0, __ldg(a.start + i)) : 0;
    sight.window = a.window;
    sight.ring = (row.pos + row.count + kKv8Block - 1) / kKv8Block * kKv8Block - c.cap;
    const int first = sight.lo(row.pos + t0), end = row.pos + t1;  // positions that some row sees
    const int kb0 = first / kKv8Block;
    const int nb = first <= end ? end / kKv8Block - kb0 + 1 : 0;
    // a short context uses fewer parts than were launched
    const int parts = max(1, min(max_parts, nb / (cluster * kWarps * kMinBlocks)));
    if (part_of >= parts) return;
    const int runs = parts * cluster, run = part_of * cluster + rank;
    const int sb0 = kb0 + (int)((int64_t)nb * run / runs), sb1 = kb0 + (int)((int64_t)nb * (run + 1) / runs);
    const int64_t head = (int64_t)row.seq * c.heads + h;
    const int8_t* kbase = c.kc + head * c.cap * D;
    const int8_t* vbase = c.vc + head * c.cap * D;
    const int cap_blocks = c.cap / kKv8Block;
    const int8_t* kexp = c.ke + head * cap_blocks;
    const int8_t* vexp = c.ve + head * cap_blocks;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (kStages * 2 * HALF);
    const int mine = max(0, (sb1 - sb0 - warp + kWarps - 1) / kWarps);  // blocks sb0 + warp + 4 * j

    // Blocks are taken in turn from the ring; a lane copies the same 16-byte pieces of each.
    const int8_t* ksrc = kbase + lane * 16;
    const int8_t* vsrc = vbase + lane * 16;
    uint32_t kdst[HALF / 512], vdst[HALF / 512];
#pragma unroll
    for (int u = 0; u < HALF / 512; ++u) {
        const int p = lane + 32 * u, r = p / CH, ch = p % CH;
        kdst[u] = ring + k_piece<D>(r, ch);
        vdst[u] = ring + HALF + v_piece<D>(r, ch);
    }
    int next = (sb0 + warp) % cap_blocks;           // ring block of the next fetch
    const int stride = kWarps % cap_blocks;
    uint32_t stage = 0;                             // its place in the ring, in bytes
    auto fetch = [&](int j) {
        if (j < mine) {
            const int64_t at = (int64_t)next * HALF;
#pragma unroll
            for (int u = 0; u < HALF / 512; ++u) {
                cp_async16(kdst[u] + stage, ksrc + at + 512 * u);
                cp_async16(vdst[u] + stage, vsrc + at + 512 * u);
            }
            next += stride;
            if (next >= cap_blocks) next -= cap_blocks;
            stage = stage == (kStages - 1) * 2 * HALF ? 0 : stage + 2 * HALF;
        }
        cp_async_commit();
    };
#pragma unroll
    for (int j = 0; j < kStages - 1; ++j) fetch(j);
    // lane j: 2^e_k, e_v and 2^-e_v of this warp's block j of the current 32
    float blk_k = 1.0f, blk_e = 0.0f, blk_l = 1.0f;
    auto fetch_exps = [&](int j) {
        if (j >= mine) return;
        const int blk = (sb0 + warp + kWarps * j) % cap_blocks;
        const int ev = vexp[blk];
        blk_k = pow2i(kexp[blk]);
        blk_e = (float)ev;
        blk_l = pow2i(-ev);
    };
    fetch_exps(lane);

    // q of row qr as hi and lo parts: k step s = 4 * (half) + w holds dimensions 64 * half + 16 * t + 4 * w + 0..3
    const int qr = NARROW ? g & 3 : g;
    const bool live = qr < rows;
    const int tok = live ? (r0 + qr) / a.group : t0;
    uint32_t qa[KS][NARROW ? 2 : 4];
    float q_step;  // scores = accumulator * q_step * 2^e_k
    {
        float x[D / 64][16];
        float amax = 0.0f;
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf) {
            if (live) {
                const int qh = h * a.group + (r0 + qr) % a.group;
                load16(a.q, a.q_dtype, i * a.qs.seq + (int64_t)tok * a.qs.token + qh * a.qs.head + 64 * hf + 16 * t, x[hf]);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                x[hf][e] = live ? x[hf][e] * (a.scale * kLog2e) : 0.0f;
                amax = fmaxf(amax, fabsf(x[hf][e]));
            }
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
        // the row scaled to a maximum in [2^13, 2^14): the parts of its small elements stay normal in f16 (a row
        // below 2^-113 by 2^126, whose inverse is the least normal number)
        const int ex = amax > 0.0f ? max((__float_as_int(amax) >> 23) - 127 - 13, -126) : 0;
        const float up = pow2i(-ex);
        q_step = pow2i(ex);
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t* A = qa[4 * hf + w];
                uint32_t hi[2], lo[2];
                split2(x[hf][4 * w] * up, x[hf][4 * w + 1] * up, &hi[0], &lo[0]);
                split2(x[hf][4 * w + 2] * up, x[hf][4 * w + 3] * up, &hi[1], &lo[1]);
                if constexpr (NARROW) {
                    A[0] = g < 4 ? hi[0] : lo[0], A[1] = g < 4 ? hi[1] : lo[1];
                } else {
                    A[0] = hi[0], A[1] = lo[0], A[2] = hi[1], A[3] = lo[1];
                }
            }
    }
    // the rows whose scores this lane sees: row g at keys 2t, 2t + 1, 2t + 8, 2t + 9, or (narrow) rows
    // sr and sr + 1 at keys g and g + 8
    constexpr int LR = NARROW ? 2 : 1;
    const int sr = NARROW ? 2 * (t & 1) : g;
    int see_lo[LR], see_hi[LR];
    float step[LR];
#pragma unroll
    for (int e = 0; e < LR; ++e) {
        const int P = row.pos + (r0 + sr + e) / a.group;
        see_lo[e] = sr + e < rows ? sight.lo(P) : 0x7FFFFFFF;
        see_hi[e] = sr + e < rows ? P : -1;
        step[e] = NARROW ? __shfl_sync(0xFFFFFFFFu, q_step, 4 * (sr + e)) : q_step;
    }

    float o[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    RowState st[LR];
#pragma unroll
    for (int e = 0; e < LR; ++e) st[e] = RowState{-FLT_MAX, 0.0f};
    // inside every row's sight: no masking needed
    const int all_lo = sight.lo(row.pos + t1), all_hi = row.pos + t0;

    uint32_t read = 0;  // place of block j in the ring, in bytes
    for (int j = 0; j < mine; ++j) {
        if (j > 0 && j % 32 == 0) fetch_exps(j + lane);
        const float k_step = __shfl_sync(0xFFFFFFFFu, blk_k, j % 32);
        const float ev = __shfl_sync(0xFFFFFFFFu, blk_e, j % 32);
        const float to_sum = __shfl_sync(0xFFFFFFFFu, blk_l, j % 32);
        cp_async_wait<kStages - 2>();
        __syncwarp();
        const uint8_t* kst = smem + warp * (kStages * 2 * HALF) + read;
        const uint8_t* vst = kst + HALF;
        read = read == (kStages - 1) * 2 * HALF ? 0 : read + 2 * HALF;
        const int p0 = (sb0 + warp + kWarps * j) * kKv8Block;
        // scores: v[e] of key e's and row e's of this lane
        float v[4];
        auto key_of = [&](int e) { return NARROW ? g + 8 * (e >> 1) : 2 * t + (e & 1) + 8 * (e >> 1); };
        auto row_of = [](int e) { return NARROW ? e & 1 : 0; };
        if constexpr (NARROW) {
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int hf = 0; hf < D / 64; ++hf) {
                const uint4 k0 = *reinterpret_cast<const uint4*>(kst + k_piece<D>(g, 4 * hf + t));
                const uint4 k1 = *reinterpret_cast<const uint4*>(kst + k_piece<D>(8 + g, 4 * hf + t));
                const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint32_t x = w0[u] ^ 0x80808080u, y = w1[u] ^ 0x80808080u;
                    const uint32_t A[4] = {codes_to_f16<0x4140>(x), codes_to_f16<0x4140>(y), codes_to_f16<0x4342>(x),
                                           codes_to_f16<0x4342>(y)};
                    mma16816(s, A, qa[4 * hf + u][0], qa[4 * hf + u][1]);
                }
            }
            // columns 2t, 2t + 1 are one part of rows sr, sr + 1; lane t ^ 2 holds the other
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (s[e] + __shfl_xor_sync(0xFFFFFFFFu, s[e], 2)) * (step[e & 1] * k_step);
        } else {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int hf = 0; hf < D / 64; ++hf) {
                    const uint4 kq = *reinterpret_cast<const uint4*>(kst + k_piece<D>(8 * n + g, 4 * hf + t));
                    const uint32_t w[4] = {kq.x, kq.y, kq.z, kq.w};
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t x = w[u] ^ 0x80808080u;
                        mma16816(s, qa[4 * hf + u], codes_to_f16<0x4140>(x), codes_to_f16<0x4342>(x));
                    }
                }
                v[2 * n] = (s[0] + s[2]) * (step[0] * k_step);
                v[2 * n + 1] = (s[1] + s[3]) * (step[0] * k_step);
            }
        }
        if (p0 < all_lo || p0 + kKv8Block - 1 > all_hi) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int p = p0 + key_of(e);
                if (p < see_lo[row_of(e)] || p > see_hi[row_of(e)]) v[e] = -INFINITY;
            }
        }
        bool grow = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) grow |= v[e] + ev > st[row_of(e)].M + kLazy;
        if (__any_sync(0xFFFFFFFFu, grow)) {
            // (a row of -inf leaves M alone: it starts at -FLT_MAX, never at -inf)
            float f[LR];
#pragma unroll
            for (int e = 0; e < LR; ++e) {
                float mx = NARROW ? fmaxf(v[e], v[2 + e]) : fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
                if constexpr (NARROW) {
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16)) + ev;
                } else {
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2)) + ev;
                }
                f[e] = mx > st[e].M + kLazy ? exp2f(st[e].M - mx) : 1.0f;
                if (mx > st[e].M + kLazy) st[e].M = mx;
                st[e].l *= f[e];
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) o[n][0] *= f[0], o[n][1] *= f[LR - 1], o[n][2] *= f[0], o[n][3] *= f[LR - 1];
        }
        uint32_t pa[NARROW ? 2 : 4];
        {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = exp2_approx(v[e] + (ev + (kWeightShift - st[row_of(e)].M)));
            if constexpr (NARROW) {
                st[0].l = fmaf(w[0] + w[2], to_sum, st[0].l);
                st[LR - 1].l = fmaf(w[1] + w[3], to_sum, st[LR - 1].l);
            } else {
                st[0].l = fmaf((w[0] + w[1]) + (w[2] + w[3]), to_sum, st[0].l);
            }
            uint32_t hi[2], lo[2];
            split2(w[0], w[1], &hi[0], &lo[0]);
            split2(w[2], w[3], &hi[1], &lo[1]);
            if constexpr (NARROW) {
                // lanes t < 2 hand on the leading parts, the others the rest: columns 0-3 and 4-7 of B
                pa[0] = transpose8x8(t < 2 ? hi[0] : lo[0]);
                pa[1] = transpose8x8(t < 2 ? hi[1] : lo[1]);
            } else {
                pa[0] = hi[0], pa[1] = lo[0], pa[2] = hi[1], pa[3] = lo[1];
            }
        }
        // V: keys 2t, 2t + 1, 2t + 8, 2t + 9 of dimensions VB * g + 0 .. VB - 1: n tile n takes dimension n
        // of each lane, or (narrow) the 16 rows of tile n dimensions 2n and 2n + 1 of each
        {
            auto add_product = [](float (&sum)[4], const uint32_t (&A)[4], uint32_t b0, uint32_t b1) {
                if constexpr (SUMS) {
                    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma16816(x, A, b0, b1);
                    const float2 u = add2(make_float2(sum[0], sum[1]), make_float2(x[0], x[1]));
                    const float2 v = add2(make_float2(sum[2], sum[3]), make_float2(x[2], x[3]));
                    sum[0] = u.x, sum[1] = u.y, sum[2] = v.x, sum[3] = v.y;
                } else {
                    mma16816(sum, A, b0, b1);
                }
            };
            uint32_t r[4][VW];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = 2 * t + (e & 1) + 8 * (e >> 1);
                const int byte = VB * g;
                const uint8_t* src = vst + v_piece<D>(key, byte >> 4) + (byte & 15);
                if constexpr (VW == 4) *reinterpret_cast<uint4*>(r[e]) = *reinterpret_cast<const uint4*>(src);
                else *reinterpret_cast<uint2*>(r[e]) = *reinterpret_cast<const uint2*>(src);
            }
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                const uint32_t A = r[0][w] ^ 0x80808080u, B = r[1][w] ^ 0x80808080u;
                const uint32_t C = r[2][w] ^ 0x80808080u, E = r[3][w] ^ 0x80808080u;
                const uint32_t ab0 = __byte_perm(A, B, 0x5140), ab1 = __byte_perm(A, B, 0x7362);
                const uint32_t ce0 = __byte_perm(C, E, 0x5140), ce1 = __byte_perm(C, E, 0x7362);
                const uint32_t x0 = codes_to_f16<0x4140>(ab0), x1 = codes_to_f16<0x4342>(ab0), x2 = codes_to_f16<0x4140>(ab1),
                               x3 = codes_to_f16<0x4342>(ab1), y0 = codes_to_f16<0x4140>(ce0), y1 = codes_to_f16<0x4342>(ce0),
                               y2 = codes_to_f16<0x4140>(ce1), y3 = codes_to_f16<0x4342>(ce1);
                if constexpr (NARROW) {
                    const uint32_t A0[4] = {x0, x1, y0, y1}, A1[4] = {x2, x3, y2, y3};
                    add_product(o[2 * w], A0, pa[0], pa[1]);
                    add_product(o[2 * w + 1], A1, pa[0], pa[1]);
                } else {
                    add_product(o[4 * w], pa, x0, y0);
                    add_product(o[4 * w + 1], pa, x1, y1);
                    add_product(o[4 * w + 2], pa, x2, y2);
                    add_product(o[4 * w + 3], pa, x3, y3);
                }
            }
        }
        __syncwarp();
        fetch(j + kStages - 1);
    }
    // the row's l: its lanes hold different keys
#pragma unroll
    for (int e = 0; e < LR; ++e)
#pragma unroll
        for (int d = NARROW ? 4 : 1; d <= (NARROW ? 16 : 2); d <<= 1) st[e].l += __shfl_xor_sync(0xFFFFFFFFu, st[e].l, d);
    cp_async_wait<0>();
    __syncthreads();
    // warp states to shared memory, the 16-byte pieces of a row permuted so that the lanes of a quarter
    // warp hit different banks
    float4* so = reinterpret_cast<float4*>(smem);
    constexpr int PL = NARROW ? VW : D / 16;  // pieces of a lane
    auto so_at = [&](int w, int r, int piece) {
        const int lt = piece / PL, k = piece % PL;
        const int turn = NARROW ? r : lt + 4 * (r & 1);
        return (w * ROWS + r) * (D / 4) + lt * PL + (k ^ (turn & (PL - 1)));
    };
    if constexpr (NARROW) {
        // the two parts' sums; lanes t and t ^ 2 both have them, and write one row each: dimensions
        // VB * g + 0 .. VB - 1
        const int second = t >> 1, r = sr + second;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] += __shfl_xor_sync(0xFFFFFFFFu, o[n][e], 2);
        if (r < rows) {
#pragma unroll
            for (int k = 0; k < PL; ++k)
                so[so_at(warp, r, PL * g + k)] =
                    second ? make_float4(o[2 * k][1], o[2 * k][3], o[2 * k + 1][1], o[2 * k + 1][3])
                           : make_float4(o[2 * k][0], o[2 * k][2], o[2 * k + 1][0], o[2 * k + 1][2]);
            if (g == 0) sm_state[warp][r] = st[second ? LR - 1 : 0];
        }
    } else if (live) {
        // dimensions 2 * VB * t + 0 .. 2 * VB - 1
#pragma unroll
        for (int k = 0; k < PL; ++k) {
            const int col = 4 * k / VB, n = 4 * k % VB;
            so[so_at(warp, g, PL * t + k)] =
                make_float4(o[n][col] + o[n][col + 2], o[n + 1][col] + o[n + 1][col + 2],
                            o[n + 2][col] + o[n + 2][col + 2], o[n + 3][col] + o[n + 3][col + 2]);
        }
        if (t == 0) sm_state[warp][g] = st[0];
    }
    __syncthreads();
    const int pieces = rows * (D / 4);
    auto write_out = [&](int r, int piece, float4 v) {
        const int token = (r0 + r) / a.group, qh = h * a.group + (r0 + r) % a.group;
        store4(a.out, a.out_dtype, i * a.os.seq + (int64_t)token * a.os.token + qh * a.os.head + 4 * piece, v);
    };
    // the CTA's pieces, then the cluster's: each CTA of it joins and passes on a share of them, from all
    // CTAs' shared memory
    float4* own = so + kWarps * ROWS * (D / 4);
    constexpr int STRIDE = ROWS * (D + 4);
    float* part = a.part + ((int64_t)item * max_parts + part_of) * STRIDE;
    auto pass_on = [&](int p, const RowState& rs, float4 v) {
        const int r = p / (D / 4), piece = p % (D / 4);
        if (parts == 1) {
            write_out(r, piece, row_output(rs, v));
        } else {
            *reinterpret_cast<float4*>(part + r * (D + 4) + 4 + 4 * piece) = v;
            if (piece == 0) *reinterpret_cast<float4*>(part + r * (D + 4)) = make_float4(rs.M, rs.l, 0.0f, 0.0f);
        }
    };
    for (int p = threadIdx.x; p < pieces; p += kWarps * 32) {
        const int r = p / (D / 4), piece = p % (D / 4);
        float4 v;
        const RowState rs = merge_parts(
            kWarps, [&](int w) { return sm_state[w][r]; }, [&](int w) { return so[so_at(w, r, piece)]; }, &v);
        if (cluster == 1) {
            pass_on(p, rs, v);
        } else {
            own[p] = v;
            if (piece == 0) own_state[r] = rs;
        }
    }
    if (cluster > 1) {
        cluster_sync();
        for (int p = threadIdx.x * cluster + rank; p < pieces; p += kWarps * 32 * cluster) {
            float2 st_of[kMaxCluster];
            float4 v_of[kMaxCluster];
#pragma unroll
            for (int j = 0; j < kMaxCluster; ++j) {
                const int from = j < cluster ? j : rank;
                st_of[j] = cluster_load2(smem_u32(&own_state[p / (D / 4)]), from);
                v_of[j] = cluster_load4(smem_u32(&own[p]), from);
                if (j >= cluster) st_of[j].y = 0.0f;
            }
            float4 v;
            const RowState rs = merge_parts(
                kMaxCluster, [&](int j) { return RowState{st_of[j].x, st_of[j].y}; }, [&](int j) { return v_of[j]; }, &v);
            pass_on(p, rs, v);
        }
        cluster_sync();  // no CTA leaves while another reads its shared memory
    }
    if (parts == 1) return;
    // the last of the item's CTAs joins the parts in their order, so the result does not depend on which
    // one that is, and leaves the ticket at zero for the next call
    __syncthreads();
    if (threadIdx.x == 0) last = ticket(a.tickets + item) == (uint32_t)(parts * cluster - 1);
    __syncthreads();
    if (!last) return;
    // each row's factors first, then the pieces, with the parts shared among as many threads as a piece
    // can have: every load is independent of the others
    const float* all = a.part + (int64_t)item * max_parts * STRIDE;
    float2* factor = reinterpret_cast<float2*>(smem);                                      // [rows][parts] (M, l), then 2^(M - max)
    float4* sums = reinterpret_cast<float4*>(smem + kMaxParts * ROWS * sizeof(float2));   // [threads]
    for (int p = threadIdx.x; p < rows * parts; p += kWarps * 32)
        factor[p] = __ldcg(reinterpret_cast<const float2*>(all + (int64_t)(p % parts) * STRIDE + p / parts * (D + 4)));
    __syncthreads();
    for (int r = warp; r < rows; r += kWarps) {
        float M = -FLT_MAX, l = 0.0f;
        for (int j = lane; j < parts; j += 32) {
            const float2 x = factor[r * parts + j];
            if (x.y != 0.0f) M = fmaxf(M, x.x);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, d));
        for (int j = lane; j < parts; j += 32) {
            const float2 x = factor[r * parts + j];
            const float f = x.y != 0.0f ? exp2f(x.x - M) : 0.0f;
            l = fmaf(x.y, f, l);
            factor[r * parts + j].x = f;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, d);
        if (lane == 0) sm_state[0][r] = RowState{M, l};
    }
    __syncthreads();
    constexpr int PIECES = ROWS * (D / 4);
    constexpr int SHARE = PIECES >= kWarps * 32 ? 1 : kWarps * 32 / PIECES;  // threads of a piece
    for (int p0 = 0; p0 < pieces; p0 += kWarps * 32 / SHARE) {
        const int p = p0 + threadIdx.x / SHARE, share_of = threadIdx.x % SHARE;
        const int r = p / (D / 4), piece = p % (D / 4);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (p < pieces) {
            const float* src = all + r * (D + 4) + 4 + 4 * piece;
#pragma unroll 8
            for (int j = share_of; j < parts; j += SHARE) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(src + (int64_t)j * STRIDE));
                const float f = factor[r * parts + j].x;
                v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
            }
        }
        if constexpr (SHARE > 1) {
            sums[threadIdx.x] = v;
            __syncthreads();
            if (share_of == 0)
                for (int e = 1; e < SHARE; ++e) {
                    const float4 x = sums[threadIdx.x + e];
                    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
                }
            __syncthreads();
        }
        if (p < pieces && share_of == 0) write_out(r, piece, row_output(sm_state[0][r], v));
    }
    if (threadIdx.x == 0) a.tickets[item] = 0u;
}

template <int D, bool NARROW>
constexpr size_t attend_smem() {
    // the warps' rings; at the end of a split context the factors and shared sums of its merge
    return std::max((size_t)kWarps * Shape<NARROW>::kStages * 2 * 16 * D,
                    kMaxParts * Shape<NARROW>::kRows * sizeof(float2) + kWarps * 32 * sizeof(float4));
}

// How an item's keys are cut: the runs that a model of the time finds best.  It was fitted to calls of
// 16 heads over 16 .. 751 positions at 1 .. 64 streams and of 8 heads over 4,000 .. 65,000: a CTA takes
// 3 us besides its blocks, a block of 16 keys takes a warp 0.6 us on an idle SM and 1.5 us on a full
// one, joining a cluster takes 1 us and joining parts through memory 3 us and a little for each.  (Parts
// alone, without clusters: 751 positions of 16 heads 11.0 us, with them 7.2 us.)
struct Cut {
    int parts, cluster;
    double us;
};
Cut cut_items(int64_t items, int64_t blocks, int slots) {
    Cut best{1, 1, 1e30};
    for (int cluster = 1; cluster <= kMaxCluster; cluster *= 2)
        for (int parts = 1; parts <= kMaxParts; parts = parts < 8 ? parts + 1 : parts + parts / 4) {
            const int64_t runs = (int64_t)parts * cluster;
            if ((runs > 1 && (runs * kWarps > blocks + kWarps || items * runs > INT_MAX)) || (parts > 1 && (cluster < kMaxCluster / 2 || items * parts > kKv8MaxPartials ||
                                                                         runs * kWarps * kMinBlocks > blocks)))
                break;
            const double fill = std::min(1.0, (double)(items * runs) / slots);
            const double waves = (double)((items * runs + slots - 1) / slots);
            const double block_us = std::max(0.6, 1.5 * fill);
            const double cta_us = 3.0 + block_us * (double)((blocks + runs * kWarps - 1) / (runs * kWarps));
            // (a tenth of a CTA's time for contexts that differ in length)
            const double us = (waves + 0.1) * cta_us + (cluster > 1 ? 1.0 : 0.0) + (parts > 1 ? 3.0 + 0.1 * parts : 0.0);
            if (us < best.us) best = Cut{parts, cluster, us};
        }
    return best;
}

template <bool NARROW>
int64_t row_groups(int64_t rows) {
    return (rows + Shape<NARROW>::kRows - 1) / Shape<NARROW>::kRows;
}

template <int D, bool NARROW, bool SUMS>
cudaError_t attend_t(const Kv8Dev& c, const Kv8Batch& b, const Kv8Attention& a, const Cut& cut, cudaStream_t st) {
    const int groups = (int)row_groups<NARROW>((int64_t)b.tokens * a.group);
    const int64_t items = (int64_t)b.n * c.heads * groups;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * cut.parts * cut.cluster));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = attend_smem<D, NARROW>();
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cut.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cut.cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, attend_kernel<D, NARROW, SUMS>, c, b, a, groups, cut.parts, cut.cluster);
}

// A product's f32 accumulator is truncated, not rounded, at every block: a warp's sums drift by about 1.3e-8
// of themselves a block.  f32 outputs of runs that are longer than 32 blocks for a warp therefore get their own
// additions (80 x 8 heads over 60,000 positions 3.2e-7 off, without them 2e-6 and more, whose growth has no end),
// at 3% of the time where HBM does not hide them; shorter runs (512 x 16 heads over 751 positions: 267 us, with
// the additions 275 us) and 16-bit outputs do without.
constexpr int kMaxRun = 32;
template <int D, bool NARROW>
cudaError_t attend_sums(const Kv8Dev& c, const Kv8Batch& b, const Kv8Attention& a, const Cut& cut, int64_t blocks, cudaStream_t st) {
    const bool sums = a.out_dtype == DT_F32 && blocks > (int64_t)cut.parts * cut.cluster * kWarps * kMaxRun;
    return sums ? attend_t<D, NARROW, true>(c, b, a, cut, st) : attend_t<D, NARROW, false>(c, b, a, cut, st);
}

template <int D, bool NARROW>
cudaError_t configure_t() {
    for (const auto kernel : {attend_kernel<D, NARROW, true>, attend_kernel<D, NARROW, false>}) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)attend_smem<D, NARROW>());
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace

size_t kv8_partial_bytes(int dim) { return (size_t)kKv8MaxPartials * kKv8Rows * (dim + 4) * sizeof(float); }

cudaError_t kv8_configure(int num_sms, Kv8Machine* m) {
    m->num_sms = num_sms;
    for (const cudaError_t e : {configure_t<128, true>(), configure_t<128, false>(), configure_t<64, true>(), configure_t<64, false>(),
                                kv8_configure_prompt(m)})
        if (e != cudaSuccess) return e;
    return cudaSuccess;
}

cudaError_t launch_kv8_attention(const Kv8Dev& c, const Kv8Batch& b, const Kv8Attention& a, const Kv8Machine& m,
                                 cudaStream_t st) {
    const int64_t rows = (int64_t)b.tokens * a.group, items = (int64_t)b.n * c.heads;  // rows of a K/V head
    const int64_t blocks = (a.window > 0 ? std::min<int64_t>((int64_t)a.window + b.tokens, c.cap) : c.cap) / kKv8Block + 1;
    // The narrow form: 512 sequences x 751 positions 276 us (the other form 311), 4 x 65,521 positions of 4
    // query heads each 107 us (117); calls of a few microseconds are within 0.3 us, or up to 1 us slower with
    // head_dim 64.
    const bool narrow = rows <= Shape<true>::kRows;
    const Cut cut = narrow ? cut_items(items, blocks, Shape<true>::kCtas * m.num_sms)
                           : cut_items(items * row_groups<false>(rows), blocks, Shape<false>::kCtas * m.num_sms);
    if (rows > kKv8Rows && a.q_dtype != DT_F32 && a.out_dtype != DT_F32) {
        const PromptPlan plan = kv8_prompt_plan(rows, items, blocks, a.out_dtype, m);
        if (plan.us < cut.us) return launch_kv8_prompt(c, b, a, plan.cluster, st);
    }
    if (narrow) return c.dim == 128 ? attend_sums<128, true>(c, b, a, cut, blocks, st) : attend_sums<64, true>(c, b, a, cut, blocks, st);
    return c.dim == 128 ? attend_sums<128, false>(c, b, a, cut, blocks, st) : attend_sums<64, false>(c, b, a, cut, blocks, st);
}

}  // namespace stt
