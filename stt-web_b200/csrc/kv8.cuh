// Device helpers of the 8-bit K/V cache's kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv8.h"

namespace stt {

// 2^e for whole e, clamped to the normal range (e = -126 .. 127): the bits of the exponent field.
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((max(-126, min(127, e)) + 127) << 23); }

// 2^x to 2^-22 of it, and 0 below 2^-126.
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Two f32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
          "l"(reinterpret_cast<const uint64_t&>(c)));
    return r;
}

// Smallest e >= kKv8MinExp with amax <= 127 * 2^e, for finite amax >= 0: amax = 1.m * 2^E and
// 127 * 2^(E-6) = 1.984375 * 2^E, so E - 6 serves while the mantissa field is at most 0x7E0000.
__device__ __forceinline__ int kv8_exponent(float amax) {
    const int bits = __float_as_int(amax);
    const int e = (bits >> 23) - 127 - 6 + ((bits & 0x7FFFFF) > 0x7E0000 ? 1 : 0);
    return max(kKv8MinExp, e);
}

// Takes a ticket after the CTA's writes: called by one thread behind a barrier, it releases what the
// CTA wrote and, for the thread that comes last, acquires what the others did.
__device__ __forceinline__ uint32_t ticket(uint32_t* counter) {
    uint32_t before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
    return before;
}

// Row i of the batch.  false (and the error word raised) where its entries are out of range.
struct Kv8Row {
    int seq, pos, count;
};
__device__ __forceinline__ bool kv8_row(const Kv8Dev& c, const Kv8Batch& b, int i, Kv8Row* r) {
    r->seq = b.seqs ? __ldg(b.seqs + i) : i;
    r->pos = __ldg(b.pos + i);
    r->count = b.count ? __ldg(b.count + i) : b.tokens;
    const bool ok = r->seq >= 0 && r->seq < c.n_seqs && r->count >= 0 && r->count <= b.tokens && r->pos >= 0 &&
                    r->pos <= 0x7FFFFFFF - b.tokens - 2 * kKv8Block;
    if (!ok) atomicCAS(c.err, 0, -1);  // STT_E_INVALID_ARG
    return ok;
}

template <int DT>
struct Elem;
template <>
struct Elem<DT_F32> {
    using T = float;
};
template <>
struct Elem<DT_BF16> {
    using T = __nv_bfloat16;
};
template <>
struct Elem<DT_F16> {
    using T = __half;
};

__device__ __forceinline__ float2 unpack2(uint32_t w, Elem<DT_BF16>) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, Elem<DT_F16>) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, Elem<DT_BF16>) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, Elem<DT_F16>) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// N (2, 4 or 8) consecutive elements as f32; p aligned to N elements.
template <int DT, int N>
__device__ __forceinline__ void load_elems(const typename Elem<DT>::T* p, float (&x)[N]) {
    if constexpr (DT == DT_F32) {
        if constexpr (N >= 4) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
                x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
            }
        } else {
            const float2 v = __ldg(reinterpret_cast<const float2*>(p));
            x[0] = v.x, x[1] = v.y;
        }
    } else {
        uint32_t w[N / 2];
        if constexpr (N == 8) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (N == 4) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
            w[0] = v.x, w[1] = v.y;
        } else {
            w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
        }
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float2 f = unpack2(w[i], Elem<DT>());
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
}

// 4 consecutive elements from f32; p aligned to 4 elements.
template <int DT>
__device__ __forceinline__ void store4(void* base, int64_t at, float4 v) {
    if constexpr (DT == DT_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(base) + at) = v;
    } else {
        const uint2 w = make_uint2(pack2(v.x, v.y, Elem<DT>()), pack2(v.z, v.w, Elem<DT>()));
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + at) = w;
    }
}
__device__ __forceinline__ void store4(void* base, int dtype, int64_t at, float4 v) {
    if (dtype == DT_F32) store4<DT_F32>(base, at, v);
    else if (dtype == DT_BF16) store4<DT_BF16>(base, at, v);
    else store4<DT_F16>(base, at, v);
}

}  // namespace stt
