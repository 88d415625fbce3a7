// Writing the 8-bit K/V cache and reading it back.
//
// Append.  The tokens of a call that fall into one block of 16 get one exponent per head,
//   e = max(e_old, smallest e with max|x| <= 127 * 2^e),
// where e_old counts only if the block holds older tokens (tokens before the call's first one).  New
// codes are rint(x * 2^-e), and where e > e_old the older codes move to rint(q * 2^(e_old - e)): all of
// it exact f32 arithmetic with one rounding to a whole number, so the result does not depend on the
// machine.  A block can grow while it fills, each move rounding once more: a code ends up within
// 1/2 + 1/4 + 1/8 + ... < 1 step of its value.
#include "kv8.cuh"

namespace stt {

namespace {

constexpr int kThreads = 256;

// N (2 or 4) codes of a row as one word.
template <int N>
__device__ __forceinline__ uint32_t load_codes(const int8_t* p) {
    if constexpr (N == 4) return *reinterpret_cast<const uint32_t*>(p);
    else return *reinterpret_cast<const uint16_t*>(p);
}
template <int N>
__device__ __forceinline__ void store_codes(int8_t* p, uint32_t w) {
    if constexpr (N == 4) *reinterpret_cast<uint32_t*>(p) = w;
    else *reinterpret_cast<uint16_t*>(p) = (uint16_t)w;
}

// Raises the error word where a sequence comes twice in one append: its two rows would write the
// same blocks.  One warp per batch row looks at the rows before it.
__device__ __forceinline__ void check_repeated(const Kv8Dev& c, const Kv8Batch& b, int i, int seq, int lane) {
    if (!b.seqs) return;
    bool twice = false;
    for (int j = lane; j < i; j += 32) twice |= __ldg(b.seqs + j) == seq;
    if (__any_sync(0xFFFFFFFFu, twice) && lane == 0) atomicCAS(c.err, 0, -1);
}

// One warp per (block, K or V, head) of a batch row: every new token of the block is loaded once
// (32 lanes x dim / 32 elements, all rows in flight together), the maximum goes through shuffles,
// and a token's codes leave as one row of `dim` bytes.  Heads are the innermost index, so that
// neighbouring warps read neighbouring pieces of a token.
template <int D, int DT>
__global__ void __launch_bounds__(kThreads) append_kernel(Kv8Dev c, Kv8Batch b, const typename Elem<DT>::T* __restrict__ k,
                                                          const typename Elem<DT>::T* __restrict__ v, Kv8Strides s, int nb) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31;
    int64_t task = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const int h = (int)(task % c.heads);
    task /= c.heads;
    const int kv = (int)(task & 1);
    task >>= 1;
    const int blk = (int)(task % nb);
    task /= nb;
    if (task >= b.n) return;
    const int i = (int)task;
    Kv8Row r;
    if (!kv8_row(c, b, i, &r)) return;
    if (h == 0 && kv == 0 && blk == 0) check_repeated(c, b, i, r.seq, lane);
    if (r.count > 0 && (r.pos + r.count - 1) / kKv8Block - r.pos / kKv8Block >= c.cap / kKv8Block) {
        if (lane == 0) atomicCAS(c.err, 0, -1);  // the call's tokens would overwrite one another in the ring
        return;
    }
    const int p0 = (r.pos / kKv8Block + blk) * kKv8Block;  // the block's first position
    const int lo = max(p0, r.pos), hi = min(p0 + kKv8Block, r.pos + r.count);  // new positions lo .. hi-1
    if (lo >= hi) return;
    const int slot = p0 % c.cap;
    const int64_t head = (int64_t)r.seq * c.heads + h;
    int8_t* codes = (kv ? c.vc : c.kc) + (head * c.cap + slot) * D + lane * N;
    int8_t* exps = (kv ? c.ve : c.ke) + head * (c.cap / kKv8Block) + slot / kKv8Block;
    const typename Elem<DT>::T* src = (kv ? v : k) + i * s.seq + (int64_t)(lo - r.pos) * s.token + h * s.head + lane * N;
    const int old = lo - p0, many = hi - lo;
    const int was = old ? *exps : kKv8MinExp;
    float x[kKv8Block][N];
#pragma unroll
    for (int t = 0; t < kKv8Block; ++t)
        if (t < many) load_elems<DT, N>(src + t * s.token, x[t]);
    float amax = 0.0f;
    bool finite = true;
#pragma unroll
    for (int t = 0; t < kKv8Block; ++t)
        if (t < many) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float a = fabsf(x[t][e]);
                if (a < __int_as_float(0x7F800000)) amax = fmaxf(amax, a);
                else finite = false;
            }
        }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    if (!__all_sync(0xFFFFFFFFu, finite) && lane == 0) atomicCAS(c.err, 0, -5);  // STT_E_DEVICE_FLAG
    const int e = max(was, kv8_exponent(amax));
    const float inv = pow2i(-e);
    if (old && e > was) {
        const float shift = pow2i(was - e);
        for (int t = 0; t < old; ++t) {
            int8_t* row = codes + t * D;
            const uint32_t q = load_codes<N>(row);
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < N; ++j)
                w |= (uint32_t)(__float2int_rn((float)(int8_t)(q >> (8 * j)) * shift) & 0xFF) << (8 * j);
            store_codes<N>(row, w);
        }
    }
#pragma unroll
    for (int t = 0; t < kKv8Block; ++t)
        if (t < many) {
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) w |= (uint32_t)(kv8_code(x[t][j], inv) & 0xFF) << (8 * j);
            store_codes<N>(codes + (old + t) * D, w);
        }
    if (lane == 0 && (e != was || !old)) *exps = (int8_t)e;
}

// Values of a range of tokens.  A thread turns 8 codes into 8 values.
template <int D, int DT>
__global__ void __launch_bounds__(kThreads) read_kernel(Kv8Dev c, Kv8Batch b, void* __restrict__ k, void* __restrict__ v,
                                                        Kv8Strides s) {
    int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int piece = (int)(item % (D / 8));
    item /= D / 8;
    const int h = (int)(item % c.heads);
    item /= c.heads;
    const int t = (int)(item % b.tokens);
    item /= b.tokens;
    if (item >= b.n) return;
    const int i = (int)item;
    Kv8Row r;
    if (!kv8_row(c, b, i, &r) || t >= r.count) return;
    const int slot = (r.pos + t) % c.cap;
    const int64_t head = (int64_t)r.seq * c.heads + h;
    const int64_t at = i * s.seq + t * s.token + h * s.head + piece * 8;
    const int64_t ce = head * (c.cap / kKv8Block) + slot / kKv8Block, cc = (head * c.cap + slot) * D + piece * 8;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const float step = pow2i((half ? c.ve : c.ke)[ce]);
        const char4* q = reinterpret_cast<const char4*>((half ? c.vc : c.kc) + cc);
        void* out = half ? v : k;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const char4 w = q[j];
            store4<DT>(out, at + 4 * j, make_float4(w.x * step, w.y * step, w.z * step, w.w * step));
        }
    }
}

template <int D, int DT>
cudaError_t append_t(const Kv8Dev& c, const Kv8Batch& b, const void* k, const void* v, const Kv8Strides& s,
                     cudaStream_t st) {
    using T = typename Elem<DT>::T;
    const int nb = (b.tokens + 2 * kKv8Block - 2) / kKv8Block;  // blocks that `tokens` tokens can touch
    const int64_t tasks = (int64_t)b.n * nb * 2 * c.heads;
    const int64_t ctas = (tasks + kThreads / 32 - 1) / (kThreads / 32);
    append_kernel<D, DT><<<(unsigned)ctas, kThreads, 0, st>>>(c, b, static_cast<const T*>(k), static_cast<const T*>(v), s, nb);
    return cudaGetLastError();
}

template <int D, int DT>
cudaError_t read_t(const Kv8Dev& c, const Kv8Batch& b, void* k, void* v, const Kv8Strides& s, cudaStream_t st) {
    const int64_t items = (int64_t)b.n * b.tokens * c.heads * (D / 8);
    read_kernel<D, DT><<<(unsigned)((items + kThreads - 1) / kThreads), kThreads, 0, st>>>(c, b, k, v, s);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8Dev& c, const Kv8Batch& b, const void* k, const void* v, int dtype,
                              const Kv8Strides& s, cudaStream_t st) {
    if (c.dim == 128) {
        if (dtype == DT_F32) return append_t<128, DT_F32>(c, b, k, v, s, st);
        if (dtype == DT_BF16) return append_t<128, DT_BF16>(c, b, k, v, s, st);
        return append_t<128, DT_F16>(c, b, k, v, s, st);
    }
    if (dtype == DT_F32) return append_t<64, DT_F32>(c, b, k, v, s, st);
    if (dtype == DT_BF16) return append_t<64, DT_BF16>(c, b, k, v, s, st);
    return append_t<64, DT_F16>(c, b, k, v, s, st);
}

cudaError_t launch_kv8_read(const Kv8Dev& c, const Kv8Batch& b, void* k, void* v, int dtype, const Kv8Strides& s,
                            cudaStream_t st) {
    if (c.dim == 128) {
        if (dtype == DT_F32) return read_t<128, DT_F32>(c, b, k, v, s, st);
        if (dtype == DT_BF16) return read_t<128, DT_BF16>(c, b, k, v, s, st);
        return read_t<128, DT_F16>(c, b, k, v, s, st);
    }
    if (dtype == DT_F32) return read_t<64, DT_F32>(c, b, k, v, s, st);
    if (dtype == DT_BF16) return read_t<64, DT_BF16>(c, b, k, v, s, st);
    return read_t<64, DT_F16>(c, b, k, v, s, st);
}

}  // namespace stt
