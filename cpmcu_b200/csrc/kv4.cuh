// The page of a cache held in 4 bits.  64 tokens of one key-value head are one record:
//
//     [key codes 32 d][value codes 32 d][key parameters 512][value parameters 512]        64 d + 1024 bytes
//
// A row of d channels is quantised in two halves.  Every half has a scale s and a middle m (bf16 both), and a code c of
// 0..15 stands for m + s * (c - 8).  Two halves, not groups of 32, because their scales then meet the scores (keys) and the
// softmax weights (values) instead of every channel, and 16 lanes share one in the kernel that stores.
//
// The codes lie in the order in which a warp's lanes take them as fragments of mma.m16n8k16, so that a lane reads its 16 tokens
// by 16-byte (d a multiple of 64) or 8-byte loads and unpacks them with one mask each.  A slice of 16 tokens takes 8 d bytes; in it words of
// 32 bits go by (pair of blocks of 16 channels, lane, upper eight tokens or lower):
//     keys    lane = (token % 8) * 4 + (channel % 16) / 4         word: eight channels of one token
//     values  lane = ((channel % 16) / 2) * 4 + (token % 8) / 2   word: four channels of two neighbouring tokens, one in each half
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

template <int D>
struct Kv4 {
    static_assert(D == 32 || D == 64 || D == 96 || D == 128, "head sizes of the 4-bit cache");
    static constexpr int kRun = D % 64 == 0 ? 2 : 1;        // pairs of blocks whose words lie together for a lane
    static constexpr int kLaneBytes = 8 * kRun;
    static constexpr int kSlice = 8 * D;                    // bytes of 16 tokens' codes
    static constexpr int kValues = 32 * D;                  // where the value codes begin
    static constexpr int kKeyParams = 64 * D;
    static constexpr int kValueParams = 64 * D + 512;
    static constexpr int kBytes = 64 * D + 1024;
    // Byte of the word of (16-token slice, pair of blocks, lane, upper eight tokens).
    __host__ __device__ static constexpr int word(int slice, int pair, int lane, int upper) {
        return slice * kSlice + (pair / kRun) * (32 * kLaneBytes) + lane * kLaneBytes + (pair % kRun) * 8 + upper * 4;
    }
};

// A half row's parameters as they are stored: the scale in the lower 16 bits, the middle in the upper ones.
__device__ __forceinline__ float kv4_scale(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float kv4_middle(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// The parameters of a half row whose smallest and largest channel are lo and hi.  Every rounding is written out (no contraction), so
// that a row has the same codes wherever it is stored.
__device__ __forceinline__ uint32_t kv4_parameters(float lo, float hi) {
    const bf16 s = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
    const bf16 m = __float2bfloat16_rn(__fadd_rn(lo, __fmul_rn(8.0f, __bfloat162float(s))));
    return (uint32_t)__bfloat16_as_ushort(s) | ((uint32_t)__bfloat16_as_ushort(m) << 16);
}
// 1 / s, or 0 where all channels are (nearly) equal: every code is then 8.
__device__ __forceinline__ float kv4_inverse(float s) { return s > 0.f ? __fdiv_rn(1.0f, s) : 0.f; }
__device__ __forceinline__ uint32_t kv4_code(float x, float m, float inverse) {
    const float c = __fadd_rn(rintf(__fmul_rn(__fsub_rn(x, m), inverse)), 8.0f);
    return (uint32_t)fminf(fmaxf(c, 0.0f), 15.0f);          // a channel that is not a number takes code 0
}
__device__ __forceinline__ float kv4_value(uint32_t code, uint32_t p) {
    return __fadd_rn(kv4_middle(p), __fmul_rn(kv4_scale(p), (float)(int)code - 8.0f));
}
