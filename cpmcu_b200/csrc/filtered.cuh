// What drawing under filters and the check of drafted tokens share: a token's weight, its whole units, and looks into a cluster's shared memory.
#pragma once
#include "common.cuh"

namespace {

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_blocks() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// Reads, writes and additions in the shared memory of the cluster's block ``rank``, at the place that ``own`` is in this block's.
__device__ __forceinline__ uint32_t peer32(const void* own, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_address(own, rank)) : "memory");
    return v;
}
__device__ __forceinline__ uint64_t peer64(const void* own, uint32_t rank) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(cluster_address(own, rank)) : "memory");
    return v;
}
__device__ __forceinline__ void put32(const void* own, uint32_t rank, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" :: "r"(cluster_address(own, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void put64(const void* own, uint32_t rank, uint64_t v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" :: "r"(cluster_address(own, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ void add64(const void* own, uint32_t rank, uint64_t v) {
    asm volatile("red.shared::cluster.add.u64 [%0], %1;" :: "r"(cluster_address(own, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ void red32(const void* own, uint32_t rank, uint32_t v) {
    asm volatile("red.shared::cluster.add.u32 [%0], %1;" :: "r"(cluster_address(own, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t add32(const void* own, uint32_t rank, uint32_t v) {
    uint32_t old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(cluster_address(own, rank)), "r"(v) : "memory");
    return old;
}

// floor(w 2^40) of a weight (0 to 1) by its bits: 24 bits of significand, shifted.
__device__ __forceinline__ uint64_t units_of(uint32_t bits) {
    return ((uint64_t)((bits & 0x7fffffu) | 0x800000u) << 17) >> min(63u, 127u - (bits >> 23));
}

// A token's weight exp((z - top) / t) from its logit.
struct Weigher {
    float top, t;
    float inverse;                                     // 1 / t where the quotient by it is exact, else 0
    __device__ __forceinline__ void set(float top_, float t_) {
        top = top_;
        t = t_;
        inverse = t > 0x1p-60f && t < 0x1p60f ? __frcp_rn(t) : 0.f;
    }
    // (x - top) / t correctly rounded.  For t within 2^60 of 1 by Markstein's method (IBM J. Res. Dev. 34, 1990): with r = 1 / t rounded, q = x r, and
    // the remainder x - q t, which a fused multiply-add gives exactly, q + r (x - q t) rounds to the quotient.  Where it overflows the weight is 0.
    __device__ __forceinline__ float over_t(float x) const {
        if (inverse == 0.f) return __fdiv_rn(x, t);
        const float q = __fmul_rn(x, inverse);
        return __fmaf_rn(__fmaf_rn(-q, t, x), inverse, q);
    }
    // Whether ``form_quick`` gives the same: the usual case, in which a token's weight is formed without a branch.
    __device__ __forceinline__ bool quick() const { return inverse != 0.f && top < INFINITY; }
    __device__ __forceinline__ float form_quick(float x) const {
        x = __fsub_rn(x, top);
        const float q = __fmul_rn(x, inverse), v = expf(__fmaf_rn(__fmaf_rn(-q, t, x), inverse, q));
        return v >= 0.f ? v : 0.f;
    }
    __device__ __forceinline__ float form(float x) const {
        if (top == INFINITY) return x == INFINITY ? 1.f : 0.f;
        const float v = expf(over_t(__fsub_rn(x, top)));
        return v >= 0.f ? v : 0.f;                     // a logit that is no number is never drawn
    }
};

// What a row's filters keep: the tokens whose weight's bits are above ``border``, and those at it up to the index ``cut``; ``total``: their mass.  With border
// kOneToken: the token ``cut`` alone, with all of the mass.
constexpr uint32_t kOneToken = 0xffffffffu;
struct KeptRow {
    float top;
    uint32_t border;
    int cut, unused;
    uint64_t total, unused2;
};

}  // namespace
