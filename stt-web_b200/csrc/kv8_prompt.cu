// Attention over the 8-bit K/V cache for chunks of many query rows, on the 5th-generation tensor cores.
//
// The formula is kv8_attn.cu's.  A CTA takes up to 256 query rows of a K/V head (rows are tokens x the
// head's group of query heads) as two tiles of 128, and walks over the keys 128 at a time:
//   S = Q K^T   (tcgen05, f16 x f16 -> f32 in TMEM),  weights in registers,  O += P V  (P from TMEM).
// What bounds it: per tile of 128 x 128 scores and 128 dimensions the two products take 1024 cycles of
// the tensor cores, the 16384 exponentials 1024 cycles of the 16-per-cycle special function units; the
// codes of K and V are turned into f16 once for both tiles.  Hence
//  - roles per warpgroup: one of softmax for each tile (a thread owns a row and holds its 128 scores in
//    registers: no shuffles, one trip to TMEM), one that turns codes into f16 operands, one whose first
//    warp issues products, with mbarriers between them: while one tile is in its softmax the other is
//    on the tensor cores.  The registers go where they are needed (setmaxnreg);
//  - the codes come straight into the registers of the threads that convert them, the next step's
//    while this one's are written (staged through shared memory first, a step waited for its copies:
//    3.4 us a step against 1.3);
//  - K's and V's codes go to shared memory as whole numbers, exact in f16; the blocks' exponents enter
//    in the softmax, where they are free: a score is the accumulator times (row step * 2^e_k * scale), the
//    argument of the exponential takes + e_v, and so the weight is 2^(s + e_v - M) with the running
//    maximum M of s + e_v.  The sum of the softmax takes the weight times 2^(E - e_v), one fused
//    multiply-add in the place of the addition.  What that holds: in f16 a weight keeps its bits down to
//    2^-20 of the row's largest and is lost below 2^-31, so a key whose s + e_v is that far below the
//    others adds nothing to the output, in whichever dimension; and the f32 sum keeps every key whose
//    share is above 2^-22 of the largest while V's exponents lie within 110 of one another (a weight is
//    flushed to zero below 2^-126, 2^132 below the row's largest);
//  - q is exact in f16 once its row is scaled by a power of two.  Weights, scaled by 2^6, are rounded to f16
//    for bf16 outputs: at most 2^-11 of each against the output's own 2^-8 (its error grows by 1%).  For f16
//    outputs that would be as much as their own rounding (errors up to 25% above its alone), so there P
//    has two f16 parts, the rest behind the first in what the scores leave free of their 128 columns, and
//    O += P V two products: 22 bits, for 20% more time;
//  - M moves only when a score exceeds it by 8 (weights then reach 2^14, inside f16), so that O, which
//    lives in TMEM, is rescaled a few times per row instead of at every tile.
// Both operands of a product lie in core matrices of 8 rows x 16 bytes: a key's 8 dimensions are one
// row of K's K-major matrix and of V's MN-major one, so both are written alike.
// Where there are fewer row blocks than SMs, a cluster of CTAs takes the steps of a row block in equal
// runs; at the end each sends O, M and l of every row to the shared memory of the CTA that joins that row
// in its share.
// Measured: the last 1024 of 4096 positions, 4 sequences x 16 heads of 128, 149 us with bf16 outputs, 0.81
// PFLOP/s, and 179 us with f16 ones; a step of two tiles takes 2.1 us (its products 1.1 us, its exponentials as
// long on the other units; a tile's softmax waits 0.7 us a step for its products), with weights in two parts
// 2.6 us, a CTA 6 to 11 us besides (its rows in and out, the first step's latency).  Halves of 64 keys with scores and weights in alternating buffers hide that wait, but products of
// 64 columns are less than half as fast: 165 us.
// Every wait is bounded: one that gives up sets the CTA's abort word, all roles leave, the copies and
// products in flight are waited for, and the cache's error word records it.
#include <cfloat>
#include <algorithm>

#include "kv8_attn.cuh"
#include "tcgen05.cuh"

namespace stt {

namespace {

constexpr int kTile = 128;                // rows of a query tile and keys of a step
constexpr int kStepBlocks = kTile / kKv8Block;
constexpr int kSoftmaxWarps = 8, kDequantWarps = 4;
constexpr int kMmaWarp = kSoftmaxWarps + kDequantWarps;
constexpr int kThreads = 512;
// registers of a thread: 128 at the launch, then by role (256 * 184 + 128 * 104 + 128 * 40 = 512 * 128)
constexpr int kSoftmaxRegs = 184, kDequantRegs = 104, kMmaRegs = 40;
static_assert(256 * kSoftmaxRegs + 128 * kDequantRegs + 128 * kMmaRegs == kThreads * 128, "the split is what the block has");
constexpr uint32_t kTmemCols = 512;       // S of both tiles, O of both tiles
constexpr uint32_t kOCol = 256;
constexpr int kExpSlots = 4;              // steps whose exponents are kept
constexpr float kWeightShift = 6.0f;
constexpr float kLazy = 8.0f;             // how far a score may exceed M

template <int D>
struct PromptSmem {
    uint8_t q[2][kTile * D * 2];          // f16, core matrices of 8 rows x 16 bytes, D / 8 of them per 8 rows
    uint8_t k[2][kTile * D * 2], v[2][kTile * D * 2];
    __align__(16) float k_step[kExpSlots][kStepBlocks], v_exp[kExpSlots][kStepBlocks], to_sum[kExpSlots][kStepBlocks];
    uint64_t q_full[2], s_full[2], p_half[2], p_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], e_full[kExpSlots];
    uint64_t q_raw[kSoftmaxWarps];
    uint64_t done;
    float2 state[2 * kTile];              // M and l of the CTA's share of the rows, by rank of the cluster
    uint32_t tmem;
    int abort;
};

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A row of 128 rows of codes, its 16-code pieces in an order of its own, so that the 8 threads of a
// quarter warp write to different banks; and the pieces as f16 in core matrices.
template <int D>
__device__ __forceinline__ void load_row(const int8_t* src, bool there, int r, uint4 (&w)[D / 16]) {
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
        w[s] = there ? __ldg(reinterpret_cast<const uint4*>(src) + (s + r) % (D / 16)) : make_uint4(0, 0, 0, 0);
}
template <int D>
__device__ __forceinline__ void store_row(const uint4 (&w)[D / 16], uint8_t* dst, int r) {
    uint8_t* out = dst + (r >> 3) * (D / 8) * 128 + (r & 7) * 16;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        const int c = (s + r) % (D / 16);
        const uint32_t x[4] = {w[s].x ^ 0x80808080u, w[s].y ^ 0x80808080u, w[s].z ^ 0x80808080u, w[s].w ^ 0x80808080u};
#pragma unroll
        for (int half = 0; half < 2; ++half)
            *reinterpret_cast<uint4*>(out + (2 * c + half) * 128) =
                make_uint4(codes_to_f16<0x4140>(x[2 * half]), codes_to_f16<0x4342>(x[2 * half]),
                           codes_to_f16<0x4140>(x[2 * half + 1]), codes_to_f16<0x4342>(x[2 * half + 1]));
    }
}
// (All warps of a warpgroup execute the same one of these, once.)
template <int N>
__device__ __forceinline__ void registers_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 8 outputs: sums times the row's factor, in the output's type.
__device__ __forceinline__ uint4 pack8(const float* o, float f, int dtype) {
    uint32_t w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
        w[u] = dtype == DT_BF16 ? pack2(o[2 * u] * f, o[2 * u + 1] * f, Elem<DT_BF16>())
                                : pack2(o[2 * u] * f, o[2 * u + 1] * f, Elem<DT_F16>());
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// CTA (row block from the last to the first, batch row, head, rank in the cluster).  FINE: weights in two f16 parts.
template <int D, int DT, bool FINE>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(Kv8Dev c, Kv8Batch b, Kv8Attention a, int row_blocks, int cluster) {
    extern __shared__ __align__(128) uint8_t prompt_smem[];
    PromptSmem<D>& sm = *reinterpret_cast<PromptSmem<D>*>(prompt_smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % cluster, item = blockIdx.x / cluster;
    const int h = item % c.heads, i = item / c.heads % b.n;
    const int rb = row_blocks - 1 - item / c.heads / b.n;  // the later rows see more keys: they start first
    Kv8Row row;
    if (!kv8_row(c, b, i, &row)) return;
    const int r0 = rb * 2 * kTile;
    const int rows = min(2 * kTile, row.count * a.group - r0);
    if (rows <= 0) return;
    const int tiles = rows > kTile ? 2 : 1;
    const int t0 = r0 / a.group, t1 = (r0 + rows - 1) / a.group;
    Sight sight;
    sight.start = a.start ? max(0, __ldg(a.start + i)) : 0;
    sight.window = a.window;
    sight.ring = (row.pos + row.count + kKv8Block - 1) / kKv8Block * kKv8Block - c.cap;
    const int first = sight.lo(row.pos + t0), end = row.pos + t1;
    const int kb_all = first / kKv8Block;
    const int nb_all = first <= end ? end / kKv8Block - kb_all + 1 : 0;
    // this CTA's run of steps, and its blocks
    const int steps_all = (nb_all + kStepBlocks - 1) / kStepBlocks;
    const int step0 = steps_all * rank / cluster, steps = steps_all * (rank + 1) / cluster - step0;
    const int kb0 = kb_all + step0 * kStepBlocks, nb = min(nb_all - step0 * kStepBlocks, steps * kStepBlocks);
    const int64_t head = (int64_t)row.seq * c.heads + h;
    const int cap_blocks = c.cap / kKv8Block;
    volatile int* abort = &sm.abort;
    // the softmax's sum is held over 2^E; any E near the exponents of V serves
    auto base_exp = [&] {
        return nb_all > 0 ? fminf(fmaxf((float)c.ve[head * cap_blocks + kb_all % cap_blocks], -60.0f), 60.0f) : 0.0f;
    };

    if (threadIdx.x == 0) {
        for (int j = 0; j < 2; ++j) {
            mbar_init(&sm.q_full[j], 4);
            mbar_init(&sm.s_full[j], 1);
            mbar_init(&sm.p_half[j], 4);
            mbar_init(&sm.p_full[j], 4);
            mbar_init(&sm.k_full[j], kDequantWarps);
            mbar_init(&sm.k_empty[j], 1);
            mbar_init(&sm.v_full[j], kDequantWarps);
            mbar_init(&sm.v_empty[j], 1);
        }
        for (int j = 0; j < kExpSlots; ++j) mbar_init(&sm.e_full[j], 1);
        mbar_init(&sm.done, 1);
        for (int j = 0; j < kSoftmaxWarps; ++j) mbar_init(&sm.q_raw[j], 1);
        sm.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = sm.tmem;

    auto out_row = [&](int r) {
        const int tok = (r0 + r) / a.group, qh = h * a.group + (r0 + r) % a.group;
        return static_cast<uint16_t*>(a.out) + i * a.os.seq + (int64_t)tok * a.os.token + qh * a.os.head;
    };
    // the cluster's two barriers, which every thread passes
    auto meet = [&] {
        __syncwarp();
        if (cluster > 1) {
            cluster_sync();
            cluster_sync();
        }
    };
    if (warp >= kSoftmaxWarps && warp < kMmaWarp) {
        registers_down<kDequantRegs>();
        const int r = threadIdx.x - kSoftmaxWarps * 32;
        const int8_t* ke = c.ke + head * cap_blocks;
        const int8_t* ve = c.ve + head * cap_blocks;
        // row r of step j is slot r % 16 of block kb0 + 8 j + r / 16
        const int8_t* kc = c.kc + (head * c.cap + r % kKv8Block) * D;
        const int8_t* vc = c.vc + (head * c.cap + r % kKv8Block) * D;
        int at = (kb0 + r / kKv8Block) % cap_blocks;
        const int stride = kStepBlocks % cap_blocks;
        auto there = [&](int j) { return j * kStepBlocks + r / kKv8Block < nb; };
        uint4 kq[D / 16], vq[D / 16];
        load_row<D>(kc + (int64_t)at * (kKv8Block * D), there(0), r, kq);
        load_row<D>(vc + (int64_t)at * (kKv8Block * D), there(0), r, vq);
        // the next step's exponents, lane by lane
        int ek = 0, ev = 0;
        auto fetch_exps = [&](int j) {
            const int blk = j * kStepBlocks + lane;
            if (lane < kStepBlocks && blk < nb) {
                const int where = (kb0 + blk) % cap_blocks;
                ek = __ldg(ke + where);
                ev = __ldg(ve + where);
            }
        };
        if (warp == kSoftmaxWarps) fetch_exps(0);
        const int E = (int)base_exp();
        for (int j = 0; j < steps; ++j) {
            const int st = j & 1;
            if (warp == kSoftmaxWarps) {
                // the slot is free: V of step j - 1 was written, so the products of step j - 3 are done,
                // and with them the softmax of step j - 4
                if (lane < kStepBlocks) {
                    sm.k_step[j % kExpSlots][lane] = pow2i(ek);
                    sm.v_exp[j % kExpSlots][lane] = (float)ev;
                    sm.to_sum[j % kExpSlots][lane] = pow2i(E - ev);
                }
                fetch_exps(j + 1);
            }
            at += stride;
            if (at >= cap_blocks) at -= cap_blocks;
            if (!__all_sync(0xFFFFFFFFu, j < 2 || mbar_wait(&sm.k_empty[st], ((j >> 1) - 1) & 1, abort))) break;
            store_row<D>(kq, sm.k[st], r);
            load_row<D>(kc + (int64_t)at * (kKv8Block * D), j + 1 < steps && there(j + 1), r, kq);
            proxy_fence();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sm.k_full[st]);
                if (warp == kSoftmaxWarps) mbar_arrive(&sm.e_full[j % kExpSlots]);
            }
            if (!__all_sync(0xFFFFFFFFu, j < 2 || mbar_wait(&sm.v_empty[st], ((j >> 1) - 1) & 1, abort))) break;
            store_row<D>(vq, sm.v[st], r);
            load_row<D>(vc + (int64_t)at * (kKv8Block * D), j + 1 < steps && there(j + 1), r, vq);
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.v_full[st]);
        }
        meet();
    } else if (warp >= kMmaWarp) {
        registers_down<kMmaRegs>();  // (one instruction for the four warps, as the ISA asks of a warpgroup)
        if (warp == kMmaWarp) {
            constexpr uint32_t GROUP = D * 16;  // bytes of 8 rows: D / 8 core matrices
            const uint32_t qk_desc = instr_desc_f16(kTile, kTile);
            const uint32_t pv_desc = instr_desc_f16(kTile, D) | (1u << 16);  // V is MN-major
            auto qk = [&](int q, int st) {
                const uint32_t qa = smem_u32(sm.q[q]), ka = smem_u32(sm.k[st]);
    #pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    mma_f16_ss(tmem + q * kTile, smem_desc(qa + k * 256, 128, GROUP), smem_desc(ka + k * 256, 128, GROUP), qk_desc,
                               k > 0);
                mma_commit(&sm.s_full[q]);
            };
            auto pv = [&](int q, int st, int half, bool add) {
                const uint32_t va = smem_u32(sm.v[st]);
#pragma unroll
                for (int part = 0; part < (FINE ? 2 : 1); ++part)
#pragma unroll
                    for (int k = half * (kTile / 32); k < (half + 1) * (kTile / 32); ++k)
                        mma_f16_ts(tmem + kOCol + q * kTile, tmem + q * kTile + part * (kTile / 2) + k * 8,
                                   smem_desc(va + k * 2 * GROUP, GROUP, 128), pv_desc, add || part > 0 || k > 0);
            };
            bool ok = true;  // (without a step too, `done` says that nothing writes the operands any more)
            for (int q = 0; ok && q < tiles; ++q) ok = mbar_wait(&sm.q_full[q], 0, abort);
            ok = ok && steps > 0;
            if (ok) ok = mbar_wait(&sm.k_full[0], 0, abort);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (ok) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) {
                    for (int q = 0; q < tiles; ++q) qk(q, 0);
                    mma_commit(&sm.k_empty[0]);
                }
                __syncwarp();
            }
            for (int j = 0; ok && j < steps; ++j) {
                const int st = j & 1, nx = (j + 1) & 1;
                const bool more = j + 1 < steps;
                ok = mbar_wait(&sm.v_full[st], (j >> 1) & 1, abort);
                if (ok && more) ok = mbar_wait(&sm.k_full[nx], ((j + 1) >> 1) & 1, abort);
                for (int q = 0; ok && q < tiles; ++q) {
                    // the weights of the first 64 keys, then the others'
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sm.p_half[q], j & 1, abort));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) pv(q, st, 0, j > 0);
                    __syncwarp();
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sm.p_full[q], j & 1, abort));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) {
                        pv(q, st, 1, true);
                        if (more) qk(q, nx);
                    }
                    __syncwarp();
                }
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                if (elect_one()) {
                    mma_commit(&sm.v_empty[st]);
                    if (more) mma_commit(&sm.k_empty[nx]);
                }
                __syncwarp();
            }
            if (elect_one()) mma_commit(&sm.done);  // also on abort: arrives once the products issued so far are done
            __syncwarp();
        }
        meet();
    } else {
        registers_up<kSoftmaxRegs>();
        if (warp / 4 < tiles) {
        const int q = warp / 4, quarter = warp & 3, r = q * kTile + quarter * 32 + lane;
        const bool live = r < rows;
        const int tok = live ? (r0 + r) / a.group : t0;
        const int P = row.pos + tok;
        const int see_lo = live ? sight.lo(P) : 0x7FFFFFFF, see_hi = live ? P : -1;
        // the warp's 32 rows of the operand, and the thread's own row
        uint8_t* mine = sm.q[q] + quarter * 4 * (D / 8) * 128;
        uint8_t* own = mine + (lane >> 3) * (D / 8) * 128 + (lane & 7) * 16;
        float q_step, q_scale;  // scores = accumulator * (q_step * 2^e_k) * q_scale
        {
            // the row of q: scaled to a maximum in [2^13, 2^14), which is exact, and with scale's sign (a row below
            // 2^-113 by 2^126, whose inverse is the least normal number)
            const uint32_t there = __ballot_sync(0xFFFFFFFFu, live);
            if (lane == 0) mbar_expect_tx(&sm.q_raw[warp], __popc(there) * 2 * D);
            __syncwarp();
            if (live)
                bulk_g2s(mine + lane * 2 * D, static_cast<const uint16_t*>(a.q) + i * a.qs.seq + (int64_t)tok * a.qs.token +
                                                  (h * a.group + (r0 + r) % a.group) * a.qs.head,
                         2 * D, &sm.q_raw[warp]);
            __all_sync(0xFFFFFFFFu, mbar_wait(&sm.q_raw[warp], 0, abort));  // (one that gave up is seen below)
            uint4 raw[D / 8];  // pieces in an order of the lane's own, as in load_row
#pragma unroll
            for (int e = 0; e < D / 8; ++e)
                raw[e] = live ? *reinterpret_cast<const uint4*>(mine + lane * 2 * D + (e + lane) % (D / 8) * 16)
                              : make_uint4(0, 0, 0, 0);
            __syncwarp();
            float amax = 0.0f;
#pragma unroll
            for (int e = 0; e < D / 8; ++e) {
                const uint32_t w[4] = {raw[e].x, raw[e].y, raw[e].z, raw[e].w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float2 f = unpack2(w[u], Elem<DT>());
                    amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
            }
            const int ex = amax > 0.0f ? max((__float_as_int(amax) >> 23) - 127 - 13, -126) : 0;
            const float up = a.scale == 0.0f ? 0.0f : copysignf(pow2i(-ex), a.scale);
            q_step = pow2i(ex);
            q_scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;
#pragma unroll
            for (int e = 0; e < D / 8; ++e) {
                const uint32_t w[4] = {raw[e].x, raw[e].y, raw[e].z, raw[e].w};
                uint32_t o[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float2 f = unpack2(w[u], Elem<DT>());
                    o[u] = pack_f16(f.x * up, f.y * up);
                }
                *reinterpret_cast<uint4*>(own + (e + lane) % (D / 8) * 128) = make_uint4(o[0], o[1], o[2], o[3]);
            }
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.q_full[q]);
        }
        const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t s_col = lane_base + q * kTile, o_col = lane_base + kOCol + q * kTile;
        // the tile's rows see all of [all_lo, all_hi]
        const int tt0 = (r0 + q * kTile) / a.group, tt1 = (r0 + min(rows, (q + 1) * kTile) - 1) / a.group;
        const int all_lo = sight.lo(row.pos + tt1), all_hi = row.pos + tt0;
        const float E = base_exp();
        float M = -FLT_MAX, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < steps; ++j) {
            // the scores (half of the lanes poll for them) and the exponents (the other half)
            ok = __all_sync(0xFFFFFFFFu, lane < 16 ? mbar_wait(&sm.s_full[q], j & 1, abort)
                                                   : mbar_wait(&sm.e_full[j % kExpSlots], (j / kExpSlots) & 1, abort));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float k_step[kStepBlocks], v_exp[kStepBlocks];  // what turns block u's accumulators into scores, e_v
#pragma unroll
            for (int u = 0; u < kStepBlocks; u += 4) {
                const float4 ks = *reinterpret_cast<const float4*>(&sm.k_step[j % kExpSlots][u]);
                const float4 vs = *reinterpret_cast<const float4*>(&sm.v_exp[j % kExpSlots][u]);
                const float s[4] = {ks.x, ks.y, ks.z, ks.w}, e[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
                for (int v = 0; v < 4; ++v) k_step[u + v] = fmaxf(q_step * s[v] * q_scale, 1e-37f), v_exp[u + v] = e[v];
            }
            const int p0 = (kb0 + j * kStepBlocks) * kKv8Block;
            const bool masked = p0 < all_lo || p0 > all_hi - (kTile - 1);  // (p0 + kTile can pass 2^31)
            const int lo = see_lo - p0, hi = see_hi - p0;  // (no overflow: see_lo <= 2^31 - 1, p0 >= 0)
            float x[kTile];
            tmem_ld128(s_col, x);
            if (masked) {
#pragma unroll
                for (int e = 0; e < kTile; ++e)
                    if (e < lo || e > hi) x[e] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < kStepBlocks; ++u) {
                const float* y = x + 16 * u;
                const float m0 = max3(y[0], y[1], y[2]), m1 = max3(y[3], y[4], y[5]), m2 = max3(y[6], y[7], y[8]);
                const float m3 = max3(y[9], y[10], y[11]), m4 = max3(y[12], y[13], y[14]);
                const float bm = max3(max3(m0, m1, m2), max3(m3, m4, y[15]), -INFINITY);
                mx = fmaxf(mx, fmaf(bm, k_step[u], v_exp[u]));
            }
            const bool grow = mx > M + kLazy;
            if (__any_sync(0xFFFFFFFFu, grow)) {
                const float f = grow ? exp2f(M - mx) : 1.0f;
                if (grow) M = mx;
                l *= f;
                if (j > 0) {
#pragma unroll 1
                    for (int ch = 0; ch < D / 16; ++ch) {
                        float o[16];
                        tmem_ld16f(o_col + 16 * ch, o);
                        uint32_t w[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(o[e] * f);
                        tmem_st(o_col + 16 * ch, w);
                    }
                }
            }
            float part[2] = {0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < kStepBlocks; u += 2) {
                uint32_t w[16], rest[16];
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const float step = k_step[u + v];
                    const float ev = v_exp[u + v];
                    const float add = ev + (kWeightShift - M);
                    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const float2 y = fma2(make_float2(x[16 * (u + v) + e], x[16 * (u + v) + e + 1]), make_float2(step, step),
                                              make_float2(add, add));
                        const float2 z = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                        s = add2(s, z);
                        w[8 * v + e / 2] = pack_f16(z.x, z.y);
                        if constexpr (FINE) {
                            const float2 first = unpack2(w[8 * v + e / 2], Elem<DT_F16>());
                            rest[8 * v + e / 2] = pack_f16(z.x - first.x, z.y - first.y);
                        }
                    }
                    part[v] = fmaf(s.x + s.y, sm.to_sum[j % kExpSlots][u + v], part[v]);
                }
                tmem_st(s_col + 8 * u, w);  // over scores, all of which this thread has read
                if constexpr (FINE) tmem_st(s_col + kTile / 2 + 8 * u, rest);
                if (u == kStepBlocks / 2 - 2) {
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.p_half[q]);
                }
            }
            l += part[0] + part[1];
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.p_full[q]);
        }
        mbar_drain(&sm.done, 0);
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const bool whole = __all_sync(0xFFFFFFFFu, ok && *abort == 0);
        const int share = (rows + cluster - 1) / cluster;
        if (cluster > 1) {
            __syncwarp();
            cluster_sync();  // every CTA's products are done: the sums may lie over the operands
            if (live)
                cluster_store2(smem_u32(&sm.state[r % share * cluster + rank]), r / share, M, l);
        }
        uint8_t* staged = reinterpret_cast<uint8_t*>(&sm) + r * (2 * D + 16);  // over the operands: no bank twice
        float4* sums = reinterpret_cast<float4*>(&sm);  // [row of the share][rank][D / 4], pieces permuted by row
#pragma unroll
        for (int ch = 0; ch < D / 32; ++ch) {
            float o[32];
            if (whole && steps > 0) {  // (a run without a step has nothing in TMEM)
                tmem_ld32(o_col + 32 * ch, o);
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0.0f;
            }
            if (cluster > 1) {
                if (live) {
                    const uint32_t at = smem_u32(sums + (r % share * cluster + rank) * (D / 4));
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        cluster_store4(at + 16 * ((8 * ch + e) ^ (r % share & 7)), r / share, o[4 * e], o[4 * e + 1],
                                       o[4 * e + 2], o[4 * e + 3]);
                }
            } else {
                const float f = l == 0.0f ? 0.0f : pow2i((int)E) / l;
                if (l == 0.0f) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 32; e += 8)
                    *reinterpret_cast<uint4*>(staged + (32 * ch + e) * 2) = pack8(o + e, f, a.out_dtype);
            }
        }
        if (cluster == 1) {
            proxy_fence();
            if (live && whole) bulk_s2g(out_row(r), staged, 2 * D);
            bulk_s2g_wait();
        } else {
            __syncwarp();
            cluster_sync();
        }
        } else {
            meet();
        }
        if (cluster > 1 && *abort == 0) {
            // each CTA joins its share of the rows; a thread 8 dimensions of one at a time
            const int share = (rows + cluster - 1) / cluster;
            const int mine = min(rows - rank * share, share);
            const float E = base_exp();
            for (int p = threadIdx.x; p < mine * (D / 8); p += kSoftmaxWarps * 32) {
                const int at = p / (D / 8), d8 = p % (D / 8);
                float M = -FLT_MAX, l = 0.0f, o[8] = {};
                for (int k = 0; k < cluster; ++k) {
                    const float2 st = sm.state[at * cluster + k];
                    if (st.y != 0.0f) M = fmaxf(M, st.x);
                }
                for (int k = 0; k < cluster; ++k) {
                    const float2 st = sm.state[at * cluster + k];
                    if (st.y == 0.0f) continue;
                    const float4* from = reinterpret_cast<const float4*>(&sm) + (at * cluster + k) * (D / 4);
                    const float4 x = from[(2 * d8) ^ (at & 7)], y = from[(2 * d8 + 1) ^ (at & 7)];
                    const float f = exp2f(st.x - M);
                    l = fmaf(st.y, f, l);
                    const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] = fmaf(v[e], f, o[e]);
                }
                const float f = l == 0.0f ? 0.0f : pow2i((int)E) / l;
                *reinterpret_cast<uint4*>(out_row(rank * share + at) + 8 * d8) = pack8(o, f, a.out_dtype);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0 && *abort) atomicCAS(c.err, 0, -5);  // STT_E_DEVICE_FLAG
    if (warp == kMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// at least 120 KB, so that one CTA holds an SM and all of its tensor memory
template <int D>
constexpr size_t prompt_smem_bytes() {
    return sizeof(PromptSmem<D>) > 120 * 1024 ? sizeof(PromptSmem<D>) : 120 * 1024;
}
static_assert(prompt_smem_bytes<128>() <= 227 * 1024, "the stages fit one SM's shared memory");

cudaLaunchConfig_t prompt_config(int64_t ctas, int cluster, size_t smem, cudaStream_t st, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = cluster;
    attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    return cfg;
}

template <int D, int DT, bool FINE>
cudaError_t prompt_t(const Kv8Dev& c, const Kv8Batch& b, const Kv8Attention& a, int cluster, cudaStream_t st) {
    const int row_blocks = (int)(((int64_t)b.tokens * a.group + 2 * kTile - 1) / (2 * kTile));
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg =
        prompt_config((int64_t)b.n * c.heads * row_blocks * cluster, cluster, prompt_smem_bytes<D>(), st, attr);
    return cudaLaunchKernelEx(&cfg, prompt_kernel<D, DT, FINE>, c, b, a, row_blocks, cluster);
}

template <int D>
cudaError_t configure_t() {
    for (const auto kernel : {prompt_kernel<D, DT_BF16, false>, prompt_kernel<D, DT_F16, false>, prompt_kernel<D, DT_BF16, true>,
                              prompt_kernel<D, DT_F16, true>}) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)prompt_smem_bytes<D>());
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t kv8_configure_prompt(Kv8Machine* m) {
    for (const cudaError_t e : {configure_t<128>(), configure_t<64>()})
        if (e != cudaSuccess) return e;
    m->prompt_ctas[0] = m->num_sms;
    for (int j = 1; j < 4; ++j) {
        cudaLaunchAttribute attr[1];
        const cudaLaunchConfig_t cfg = prompt_config(m->num_sms << j, 1 << j, prompt_smem_bytes<128>(), 0, attr);
        int clusters = 0;
        const cudaError_t e = cudaOccupancyMaxActiveClusters(&clusters, prompt_kernel<128, DT_BF16, false>, &cfg);
        if (e != cudaSuccess) return e;
        m->prompt_ctas[j] = std::min(clusters << j, m->num_sms);
    }
    return cudaSuccess;
}

PromptPlan kv8_prompt_plan(int64_t rows, int64_t items, int64_t blocks, int out_dtype, const Kv8Machine& m) {
    // fitted to 16 .. 1024 tokens over 256 .. 30,000 positions: a CTA takes 6 us besides its steps, a step
    // 2.1 us with two tiles and 1.9 us with one (2.6 and 2.35 with weights in two parts), a cluster 2 us more.  The other kernel's time comes from a
    // model of the same calls: 64 tokens over 256 positions of 4 heads take 7.2 us there and 11 us here, 256
    // over 4096 of 16 heads 117 us there and 34 us here
    const int64_t ctas = items * ((rows + 2 * kTile - 1) / (2 * kTile)), steps = (blocks + kStepBlocks - 1) / kStepBlocks;
    const double step = rows > kTile ? (out_dtype == DT_F16 ? 2.6 : 2.1) : (out_dtype == DT_F16 ? 2.35 : 1.9);
    PromptPlan best{1, 1e30};
    for (int j = 0; j < 4 && (1 << j) <= steps; ++j) {
        const int cluster = 1 << j;
        if (m.prompt_ctas[j] < cluster) break;
        const double waves = (double)((ctas * cluster + m.prompt_ctas[j] - 1) / m.prompt_ctas[j]);
        const double us = waves * (6.0 + step * (double)((steps + cluster - 1) / cluster)) +
                          (cluster > 1 ? 2.0 : 0.0);
        if (us < best.us) best = PromptPlan{cluster, us};
    }
    return best;
}

template <int D, int DT>
cudaError_t prompt_fine(const Kv8Dev& c, const Kv8Batch& b, const Kv8Attention& a, int cluster, cudaStream_t st) {
    return a.out_dtype == DT_F16 ? prompt_t<D, DT, true>(c, b, a, cluster, st) : prompt_t<D, DT, false>(c, b, a, cluster, st);
}

cudaError_t launch_kv8_prompt(const Kv8Dev& c, const Kv8Batch& b, const Kv8Attention& a, int cluster, cudaStream_t st) {
    if (c.dim == 128)
        return a.q_dtype == DT_BF16 ? prompt_fine<128, DT_BF16>(c, b, a, cluster, st) : prompt_fine<128, DT_F16>(c, b, a, cluster, st);
    return a.q_dtype == DT_BF16 ? prompt_fine<64, DT_BF16>(c, b, a, cluster, st) : prompt_fine<64, DT_F16>(c, b, a, cluster, st);
}

}  // namespace stt
