// What the two attention kernels over the 8-bit K/V cache share.
#pragma once

#include "kv8.cuh"

namespace stt {

constexpr float kLog2e = 1.4426950408889634f;

// Cluster barrier; loads from and stores to the same place of CTA `rank`'s shared memory.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_at(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t addr, int rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_at(addr, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t addr, int rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(cluster_at(addr, rank))
                 : "memory");
    return v;
}
__device__ __forceinline__ void cluster_store2(uint32_t addr, int rank, float x, float y) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(cluster_at(addr, rank)), "f"(x), "f"(y) : "memory");
}
__device__ __forceinline__ void cluster_store4(uint32_t addr, int rank, float x, float y, float z, float w) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_at(addr, rank)), "f"(x), "f"(y), "f"(z),
                 "f"(w)
                 : "memory");
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
