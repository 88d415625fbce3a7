// What the two attention kernels over the 8-bit K/V cache share.
#pragma once

#include "kv8.cuh"

namespace stt {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Bytes `sel` of biased codes (code + 128) as a pair of f16 codes.
template <int SEL>
__device__ __forceinline__ uint32_t codes_to_f16(uint32_t biased) {
    uint32_t r = __byte_perm(biased, 0x64646464u, SEL);
    const __half2 v = __hsub2(*reinterpret_cast<__half2*>(&r), __float2half2_rn(1152.0f));
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Positions [lo, hi] that the query at position P sees.
struct Sight {
    int start, window, ring;
    __device__ __forceinline__ int lo(int P) const {
        int a = max(start, ring);
        return window > 0 && P + 1 - window > a ? P + 1 - window : a;
    }
};

}  // namespace stt
