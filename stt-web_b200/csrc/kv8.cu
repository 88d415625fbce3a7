// Writing the 8-bit K/V cache and reading it back.
//
// Append.  The tokens of a call that fall into one block of 16 get one exponent per head,
//   e = max(e_old, smallest e with max|x| <= 127 * 2^e),
// where e_old counts only if the block holds older tokens (tokens before the call's first one).  New
// codes are rint(x * 2^-e), and where e > e_old the older codes move to rint(q * 2^(e_old - e)): all of
// it exact f32 arithmetic with one rounding to a whole number, so the result does not depend on the
// machine.  A block can grow while it fills, each move rounding once more: a code ends up within
// 1/2 + 1/4 + 1/8 + ... < 1 step of its value.
//
// Both are bound by memory, so what counts is loads in flight.  Measured from cold caches: append of 2048 tokens of
// 8 sequences x 16 heads of 128 in bf16 34 us for 201 MB, 5.9 TB/s (with the rows held as f32, half the warps on an
// SM, 52 us), in f32, whose rows take twice the registers, 60 us for 336 MB, 5.6 TB/s; of one token of 512
// sequences (f32) 10 us for 10.5 MB, a launch and three dependent loads (8.4 us in L2; a warp for K and another
// for V took 10.5 us there); read of 2055 tokens of the 8 sequences (bf16) 35 us for 202 MB, 5.9 TB/s.
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

// rint(x * f) of N values, as bytes: f is a power of two and |x * f| <= 127.5.
template <int N>
__device__ __forceinline__ uint32_t pack_codes(const float (&x)[N], float f) {
    uint32_t u[N];
#pragma unroll
    for (int j = 0; j < N; ++j) u[j] = __float_as_uint(__fmaf_rn(x[j], f, 12582912.0f));
    if constexpr (N == 4) return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
    else return __byte_perm(u[0], u[1], 0x0040);
}

// Raises the error word where a sequence comes twice in one append: its two rows would write the
// same blocks.  One warp per batch row looks at the rows before it; rows without tokens, a padded batch's,
// write nothing and do not count.
__device__ __forceinline__ void check_repeated(const Kv8Dev& c, const Kv8Batch& b, int i, int seq, int lane) {
    if (!b.seqs) return;
    bool twice = false;
    for (int j = lane; j < i; j += 32) twice |= __ldg(b.seqs + j) == seq && (!b.count || __ldg(b.count + j) > 0);
    if (__any_sync(0xFFFFFFFFu, twice) && lane == 0) atomicCAS(c.err, 0, -1);
}

// N elements of a row as they lie in memory, in words.
template <int DT, int N>
struct Raw {
    static constexpr bool kShort = DT != DT_F32;
    static constexpr int kWords = kShort ? N / 2 : N;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const typename Elem<DT>::T* p) {
        if constexpr (kWords == 4) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
            w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
        } else if constexpr (kWords == 2) {
            const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
            w[0] = u.x, w[1] = u.y;
        } else {
            w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
        }
    }
    __device__ __forceinline__ void values(float (&x)[N]) const {
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
            if constexpr (kShort) {
                const float2 f = unpack2(w[j], Elem<DT>());
                x[2 * j] = f.x, x[2 * j + 1] = f.y;
            } else {
                x[j] = __uint_as_float(w[j]);
            }
        }
    }
    // Greatest magnitude so far, as bits; 16-bit types two at a time (they order like the values too).
    __device__ __forceinline__ uint32_t take_max(uint32_t m) const {
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
            if constexpr (kShort) m = __vmaxu2(m, w[j] & 0x7FFF7FFFu);
            else m = max(m, w[j] & 0x7FFFFFFFu);
        }
        return m;
    }
    // The f32 bits of such a maximum; 0x7F800000 and more are not finite.
    static __device__ __forceinline__ uint32_t bits(uint32_t m) {
        if constexpr (kShort) {
            const float2 f = unpack2(max(m >> 16, m & 0xFFFFu), Elem<DT>());
            return __float_as_uint(f.x);
        } else {
            return m;
        }
    }
};

// One warp per (block, K or V, head) of a batch row: every new token of the block is loaded once
// (32 lanes x dim / 32 elements, all rows in flight together), the maximum goes through shuffles,
// and a token's codes leave as one row of `dim` bytes.  A CTA's warps take neighbouring heads, so that
// they read neighbouring pieces of a token.  MAX is the most new tokens of a block: 1 for calls of one
// token, whose warps need a third of the registers and take K and V of a head together.
//
// The maximum is taken over the bit patterns of |x| (they order like the values; anything from
// 0x7F800000 on is not finite, and sends the warp through the checks below), and a code is
// the low byte of x * 2^-e + 1.5 * 2^23, whose unit is 1: the addition rounds to nearest, ties to even.
template <int D, int DT, int MAX>
__global__ void __launch_bounds__(kThreads, MAX == 1 ? 6 : DT == DT_F32 ? 2 : 4) append_kernel(Kv8Dev c, Kv8Batch b, const typename Elem<DT>::T* __restrict__ k,
                                                          const typename Elem<DT>::T* __restrict__ v, Kv8Strides ks, Kv8Strides vs,
                                                          int nb, int ctas_per_block) {
    constexpr int N = D / 32;
    constexpr int KV = MAX == 1 ? 2 : 1;  // of K and V, how many a warp takes
    const int lane = threadIdx.x & 31;
    const int rest = blockIdx.x / ctas_per_block;
    const int task = (blockIdx.x - rest * ctas_per_block) * (kThreads / 32) + (threadIdx.x >> 5);
    if (task >= 2 / KV * c.heads) return;
    const int kv0 = task >= c.heads, h = task - kv0 * c.heads;
    const int i = rest / nb, blk = rest - i * nb;
    Kv8Row r;
    if (!kv8_row(c, b, i, &r)) return;
    if (task == 0 && blk == 0 && r.count > 0) check_repeated(c, b, i, r.seq, lane);
    if (r.count > 0 && (r.pos + r.count - 1) / kKv8Block - r.pos / kKv8Block >= c.cap / kKv8Block) {
        if (lane == 0) atomicCAS(c.err, 0, -1);  // the call's tokens would overwrite one another in the ring
        return;
    }
    const int p0 = (r.pos / kKv8Block + blk) * kKv8Block;  // the block's first position
    const int lo = max(p0, r.pos), hi = min(p0 + kKv8Block, r.pos + r.count);  // new positions lo .. hi-1
    if (lo >= hi) return;
    const int slot = p0 % c.cap;
    const int64_t head = (int64_t)r.seq * c.heads + h;
    const int64_t code_at = (head * c.cap + slot) * D + lane * N, exp_at = head * (c.cap / kKv8Block) + slot / kKv8Block;
    const int old = lo - p0, many = hi - lo;
    Raw<DT, N> x[KV][MAX];
    int was[KV];
    // (a block with fewer tokens loads its last one again: no branch keeps the loads apart)
#pragma unroll
    for (int u = 0; u < KV; ++u) {
        const Kv8Strides& s = kv0 + u ? vs : ks;
        const typename Elem<DT>::T* src = (kv0 + u ? v : k) + i * s.seq + (int64_t)(lo - r.pos) * s.token + h * s.head + lane * N;
#pragma unroll
        for (int t = 0; t < MAX; ++t) x[u][t].load(src + min(t, many - 1) * s.token);
        was[u] = (kv0 + u ? c.ve : c.ke)[exp_at];
    }
#pragma unroll
    for (int u = 0; u < KV; ++u) {
        int8_t* codes = (kv0 + u ? c.vc : c.kc) + code_at;
        if (old == 0) was[u] = kKv8MinExp;
        uint32_t amax = 0;
#pragma unroll
        for (int t = 0; t < MAX; ++t) amax = x[u][t].take_max(amax);
        amax = __reduce_max_sync(0xFFFFFFFFu, Raw<DT, N>::bits(amax));
        const bool finite = amax < 0x7F800000u;
        if (!finite) {
            // infinities or NaN: the exponent of the finite values; infinities become +-127 steps, NaN 0
            if (lane == 0) atomicCAS(c.err, 0, -5);  // STT_E_DEVICE_FLAG
            amax = 0;
#pragma unroll
            for (int t = 0; t < MAX; ++t) {
                float y[N];
                x[u][t].values(y);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const uint32_t w = __float_as_uint(y[j]) & 0x7FFFFFFFu;
                    if (w < 0x7F800000u) amax = max(amax, w);
                }
            }
            amax = __reduce_max_sync(0xFFFFFFFFu, amax);
        }
        const int e = max(was[u], kv8_exponent(__uint_as_float(amax)));
        const float f = pow2i(-e);
        if (old && e > was[u]) {
            const float shift = pow2i(was[u] - e);
#pragma unroll 4
            for (int t = 0; t < old; ++t) {
                const uint32_t q = load_codes<N>(codes + t * D);
                float y[N];
#pragma unroll
                for (int j = 0; j < N; ++j) y[j] = (float)(int8_t)(q >> (8 * j));
                store_codes<N>(codes + t * D, pack_codes<N>(y, shift));
            }
        }
#pragma unroll
        for (int t = 0; t < MAX; ++t)
            if (t < many) {
                float y[N];
                x[u][t].values(y);
                if (!finite)  // clamped as steps: 127 * 2^122 is more than an f32 holds
#pragma unroll
                    for (int j = 0; j < N; ++j) y[j] = y[j] != y[j] ? 0.0f : fminf(fmaxf(y[j] * f, -127.0f), 127.0f);
                store_codes<N>(codes + (old + t) * D, pack_codes<N>(y, finite ? f : 1.0f));
            }
        if (lane == 0 && (e != was[u] || !old)) (kv0 + u ? c.ve : c.ke)[exp_at] = (int8_t)e;
    }
}

// Tokens of a CTA.  16 leave a last wave nearly empty where rows hold about 16 (8.5 tokens of 512 sequences,
// f32: 20.7 us, 8 take 18.1 us for 106 MB); 4 do no better, and 2 take 22 us.
constexpr int kReadTokens = 8;

// Values of a range of tokens.  A thread keeps its place in a token (as many codes as fill 16 bytes of
// values, in K and in V) and walks over the tokens, several in flight.  A code becomes a value in three
// instructions: the byte code + 128 under 0x4B0000 is the f32 value 2^23 + 128 + code; the difference to
// 2^23 + 128 is exact, and so is its product with a power of two.  (The difference after the product, in one
// fused multiply-add, leaves f32's range from the exponent 105 on.)
template <int D, int DT>
__global__ void __launch_bounds__(kThreads) read_kernel(Kv8Dev c, Kv8Batch b, void* __restrict__ k, void* __restrict__ v,
                                                        Kv8Strides ks, Kv8Strides vs, int token_ctas, int head_ctas) {
    constexpr int N = 16 / (int)sizeof(typename Elem<DT>::T);
    const int part = blockIdx.x / head_ctas, item = (blockIdx.x - part * head_ctas) * kThreads + threadIdx.x;
    const int i = part / token_ctas, t0 = (part - i * token_ctas) * kReadTokens;
    const int piece = item % (D / N), h = item / (D / N);
    Kv8Row r;
    if (!kv8_row(c, b, i, &r) || h >= c.heads) return;
    const int t1 = min(t0 + kReadTokens, r.count);
    const int64_t head = (int64_t)r.seq * c.heads + h;
    const int8_t *kc = c.kc + head * c.cap * D + piece * N, *vc = c.vc + head * c.cap * D + piece * N;
    const int8_t *ke = c.ke + head * (c.cap / kKv8Block), *ve = c.ve + head * (c.cap / kKv8Block);
    int slot = t0 < t1 ? (r.pos + t0) % c.cap : 0;
#pragma unroll 4
    for (int t = t0; t < t1; ++t) {
        uint32_t q[2][N / 4];
        float step[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int j = 0; j < N / 4; ++j)
                q[half][j] = __ldg(reinterpret_cast<const uint32_t*>((half ? vc : kc) + (int64_t)slot * D) + j);
            step[half] = pow2i(__ldg((half ? ve : ke) + slot / kKv8Block));
        }
        if (++slot == c.cap) slot = 0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float y[N];
#pragma unroll
            for (int j = 0; j < N; ++j)
                y[j] = (__uint_as_float(__byte_perm(q[half][j / 4] ^ 0x80808080u, 0x4B000000u, 0x7650 | (j % 4))) - 8388736.0f) * step[half];
            void* out = half ? v : k;
            const Kv8Strides& s = half ? vs : ks;
            const int64_t at = i * s.seq + t * s.token + h * s.head + piece * N;
            if constexpr (DT == DT_F32) {
                *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = make_float4(y[0], y[1], y[2], y[3]);
            } else {
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) =
                    make_uint4(pack2(y[0], y[1], Elem<DT>()), pack2(y[2], y[3], Elem<DT>()), pack2(y[4], y[5], Elem<DT>()),
                               pack2(y[6], y[7], Elem<DT>()));
            }
        }
    }
}

template <int D, int DT>
cudaError_t append_t(const Kv8Dev& c, const Kv8Batch& b, const void* k, const void* v, const Kv8Strides& ks,
                     const Kv8Strides& vs, cudaStream_t st) {
    using T = typename Elem<DT>::T;
    const T *kt = static_cast<const T*>(k), *vt = static_cast<const T*>(v);
    const int nb = (b.tokens + 2 * kKv8Block - 2) / kKv8Block;  // blocks that `tokens` tokens can touch
    const int per_block = ((b.tokens == 1 ? 1 : 2) * c.heads + kThreads / 32 - 1) / (kThreads / 32);
    const unsigned grid = (unsigned)((int64_t)b.n * nb * per_block);
    if (b.tokens == 1) append_kernel<D, DT, 1><<<grid, kThreads, 0, st>>>(c, b, kt, vt, ks, vs, nb, per_block);
    else append_kernel<D, DT, kKv8Block><<<grid, kThreads, 0, st>>>(c, b, kt, vt, ks, vs, nb, per_block);
    return cudaGetLastError();
}

template <int D, int DT>
cudaError_t read_t(const Kv8Dev& c, const Kv8Batch& b, void* k, void* v, const Kv8Strides& ks, const Kv8Strides& vs,
                   cudaStream_t st) {
    const int token_ctas = (b.tokens + kReadTokens - 1) / kReadTokens;
    const int head_ctas = (c.heads * (D * (int)sizeof(typename Elem<DT>::T) / 16) + kThreads - 1) / kThreads;
    read_kernel<D, DT><<<(unsigned)((int64_t)b.n * token_ctas * head_ctas), kThreads, 0, st>>>(c, b, k, v, ks, vs, token_ctas,
                                                                                              head_ctas);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8Dev& c, const Kv8Batch& b, const void* k, const void* v, int dtype,
                              const Kv8Strides& ks, const Kv8Strides& vs, cudaStream_t st) {
    if (c.dim == 128) {
        if (dtype == DT_F32) return append_t<128, DT_F32>(c, b, k, v, ks, vs, st);
        if (dtype == DT_BF16) return append_t<128, DT_BF16>(c, b, k, v, ks, vs, st);
        return append_t<128, DT_F16>(c, b, k, v, ks, vs, st);
    }
    if (dtype == DT_F32) return append_t<64, DT_F32>(c, b, k, v, ks, vs, st);
    if (dtype == DT_BF16) return append_t<64, DT_BF16>(c, b, k, v, ks, vs, st);
    return append_t<64, DT_F16>(c, b, k, v, ks, vs, st);
}

cudaError_t launch_kv8_read(const Kv8Dev& c, const Kv8Batch& b, void* k, void* v, int dtype, const Kv8Strides& ks,
                            const Kv8Strides& vs, cudaStream_t st) {
    if (c.dim == 128) {
        if (dtype == DT_F32) return read_t<128, DT_F32>(c, b, k, v, ks, vs, st);
        if (dtype == DT_BF16) return read_t<128, DT_BF16>(c, b, k, v, ks, vs, st);
        return read_t<128, DT_F16>(c, b, k, v, ks, vs, st);
    }
    if (dtype == DT_F32) return read_t<64, DT_F32>(c, b, k, v, ks, vs, st);
    if (dtype == DT_BF16) return read_t<64, DT_BF16>(c, b, k, v, ks, vs, st);
    return read_t<64, DT_F16>(c, b, k, v, ks, vs, st);
}

}  // namespace stt
