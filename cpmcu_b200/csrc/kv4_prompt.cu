// Attention of prompt tokens over the 4-bit cache on the fifth-generation tensor cores, head sizes 64 and 128.
//
// A block takes 256 rows of queries, the query heads of one key-value head for some consecutive tokens (16 tokens at 16 heads), so that all of them share
// every key and value.  Four warps unpack the codes, 128 keys a step, into fp16 tiles in shared memory: K [keys][d] and V
// [d][keys], 128-byte swizzle, the K-major operands of S = Q K^T and O += P V (tcgen05.mma, accumulators in tensor memory).  The two halves of 128
// rows take turns: while one half's products run, the other half's rows are in the softmax, a thread to a row, which writes P as fp16 over the S it read.
//
// fp16 and not bf16: its 11 bits hold s (c - 8) exactly, 8 bits times 3, so that scores are as exact as their fp32 sums.  The rest of a
// key's product, m times the sum of the query's half row, is 16 more columns of the operands: m three times and the sum as three fp16 numbers,
// for both halves.  A value is rounded to 11 bits (2^-12 of it, where the output has 8).
// What fp16 lacks in range is taken care of by powers of two: a query row, a page's keys and a page's values are divided by the power of two below
// their largest magnitude, scores are multiplied by the first two again, and the accumulator stands for O / 2^E with E the largest power of the
// values so far.
//
// Unpacking a key and a value costs about two instructions a number, 256 rows of softmax four times as many; a block of 128 rows would pay it twice.
// Bound by the exponentials and the issue slots of the softmax; see the launcher for where the other kernel is faster.
//
// Every wait is bounded: a block that gives up records an error, stops, frees its tensor memory and returns (nothing is in flight then: tiles are
// written by ordinary stores).
#include "kv4.cuh"
#include "tcgen05.cuh"

CPM_BOUNDS_TU(kv4_prompt)

namespace kv4p {
using namespace tc5;

constexpr int kRows = 256;
constexpr int kStepKeys = 128;                          // two pages
constexpr int kStages = 2;
constexpr int kSoftmaxWarps = 8, kUnpackWarps = 4;
constexpr int kThreads = (kSoftmaxWarps + 1 + kUnpackWarps) * 32;
constexpr float kBehind = 8.0f;                         // the running maximum may lie 2^8 behind
constexpr int kHalfBytes = 128 * 128;                   // 128 rows of 128 bytes

constexpr int kExtra = 128 * 32;                        // 16 more columns of 128 rows, two runs of 16 bytes a row
// Matrix descriptor of such a tile: K-major, no swizzle; groups of 8 rows 128 bytes apart, the two runs 2,048.
__device__ __forceinline__ uint64_t smem_desc_plain(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)(2048 >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}

template <int D>
struct Sizes {
    static constexpr int kHalves = D / 64;
    static constexpr int kTile = 128 * D * 2;           // 128 rows of Q, 128 keys of K or of V
    static constexpr int kVPage = D * 128;              // [d][64 keys]
    static constexpr int kSmem = 2 * kTile + 2 * kStages * kTile + (2 + kStages) * kExtra + 1024;
    static constexpr uint32_t idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }     // fp16 in, fp32 sums
    static constexpr int kO = 256;
};

struct Args {
    const bf16* q;
    bf16* out;
    const uint8_t* records;
    const int *kv_len, *slots, *page_table, *cu_q, *tile_seq, *tile_row;
    int max_pages, n_heads, n_kv, group, window, tile_tokens;
    float scale;
};

// What a step's unpacking tells the softmax: per page, and per token for steps that some row sees in part.
struct StepInfo { alignas(16) float k_token[kStepKeys]; int v_token[kStepKeys]; float k_scale[2]; int v_power[2]; uint32_t bad[2][2]; };

enum : int { ERR_Q = 1, ERR_K_FULL, ERR_V_FULL, ERR_K_EMPTY, ERR_V_EMPTY, ERR_S_FULL, ERR_P_FULL, ERR_O_FULL };
__device__ int g_error;

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long ra, rb, rc, rd;
    float2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(rb) : "f"(b.x), "f"(b.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(rc) : "f"(c.x), "f"(c.y));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(rd) : "l"(ra), "l"(rb), "l"(rc));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(rd));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long ra, rb, rd;
    float2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(rb) : "f"(b.x), "f"(b.y));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(rd));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long ra, rb, rd;
    float2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(rb) : "f"(b.x), "f"(b.y));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(rd));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float power2(int e) { return __uint_as_float((uint32_t)(max(-126, min(127, e)) + 127) << 23); }
// The power of two below a finite number (0 and what is no number: 0).
__device__ __forceinline__ int power_below(float x) { return x > 0.f && x < INFINITY ? max(-110, min(110, (int)(__float_as_uint(x) >> 23) - 127)) : 0; }
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// A word's codes less 8, as pairs: nibbles 0 and 4, 1 and 5, 2 and 6, 3 and 7.
__device__ __forceinline__ void unpack8(uint32_t w, __half2 (&r)[4]) {
    const __half2 low = __floats2half2_rn(-1032.f, -1032.f), sixteenth = __floats2half2_rn(0.0625f, 0.0625f), high = __floats2half2_rn(-72.f, -72.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t v = w >> (8 * i);
        uint32_t a, b;
        asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(a) : "r"(v));
        asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(b) : "r"(v));
        r[2 * i] = __hadd2(*reinterpret_cast<__half2*>(&a), low);
        r[2 * i + 1] = __hfma2(*reinterpret_cast<__half2*>(&b), sixteenth, high);
    }
}

// A lane's share of 16 tokens of one page: code words and parameters.
template <int D>
struct Slice {
    uint32_t k[D / 32][2], v[D / 32][2];                // [pair of 16-channel blocks][upper eight tokens]
    uint2 kp[2];                                        // rows g and g + 8
    uint4 vp[2];                                        // rows 2 j and 2 j + 1, and eight further
    __device__ __forceinline__ void load(const uint8_t* rec, int slice, int lane, int tokens) {
        using L = Kv4<D>;
        const int g = lane >> 2, j = lane & 3;
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
            const uint4 a = *reinterpret_cast<const uint4*>(rec + L::word(slice, 2 * x, lane, 0));
            k[2 * x][0] = a.x; k[2 * x][1] = a.y; k[2 * x + 1][0] = a.z; k[2 * x + 1][1] = a.w;
            const uint4 b = *reinterpret_cast<const uint4*>(rec + L::kValues + L::word(slice, 2 * x, lane, 0));
            v[2 * x][0] = b.x; v[2 * x][1] = b.y; v[2 * x + 1][0] = b.z; v[2 * x + 1][1] = b.w;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int rk = 16 * slice + g + 8 * u, rv = 16 * slice + 2 * j + 8 * u;
            kp[u] = *reinterpret_cast<const uint2*>(rec + L::kKeyParams + rk * 8);
            vp[u] = *reinterpret_cast<const uint4*>(rec + L::kValueParams + rv * 8);
            // behind the sequence's end: what lies there may be no number
            if (rk >= tokens) kp[u] = make_uint2(0u, 0u);
            if (rv >= tokens) vp[u].x = vp[u].y = 0u;
            if (rv + 1 >= tokens) vp[u].z = vp[u].w = 0u;
        }
    }
};
__device__ __forceinline__ float bound_of(uint32_t p) { return fabsf(kv4_middle(p)) + 8.f * kv4_scale(p); }

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
kv4_prompt_kernel(const __grid_constant__ Args a) {
    using Z = Sizes<D>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t q_full, k_full[kStages], v_full[kStages], k_empty[kStages], v_empty[kStages], s_full[2], p_full[2], o_full[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ StepInfo info[4];
    __shared__ float bounds[2][2][2][kUnpackWarps];      // [step parity][keys, values][page][warp]
    __shared__ uint32_t bads[2][2][kUnpackWarps];        // [step parity][page][warp]: 16 tokens each
    pdl_launch_dependents();
    pdl_wait();

    const int tile = gridDim.y - 1 - blockIdx.y;          // later tiles of a sequence have more keys: they go first
    const int row0 = a.tile_row[tile], seq = a.tile_seq[tile];
    if (row0 % a.tile_tokens) return;                     // (the list is of 64-token tiles)
    const int head_kv = blockIdx.x % a.n_kv, part = blockIdx.x / a.n_kv;
    const int q_begin = a.cu_q[seq], q_len = a.cu_q[seq + 1] - q_begin, kv_len = a.kv_len[seq], history = kv_len - q_len;
    const int tokens = min(a.tile_tokens, q_len - row0);
    const int first = part * kRows, n_rows = min(kRows, tokens * a.group - first);       // rows of the tile: token by token, head by head
    if (n_rows <= 0) return;
    const int pos_low = history + row0 + first / a.group, pos_high = history + row0 + (first + n_rows - 1) / a.group;
    const int n_keys = min(kv_len, pos_high + 1);
    const int step0 = a.window ? max(0, pos_low - a.window + 1) / kStepKeys : 0;
    const int n_steps = max(0, (n_keys + kStepKeys - 1) / kStepKeys - step0);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_smem = base, k_smem = base + 2 * Z::kTile, v_smem = k_smem + kStages * Z::kTile;
    const uint32_t qx_smem = v_smem + kStages * Z::kTile, kx_smem = qx_smem + 2 * kExtra;
    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&q_full), kSoftmaxWarps);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&k_full[s]), kUnpackWarps);
            mbar_init(smem_u32(&v_full[s]), kUnpackWarps);
            mbar_init(smem_u32(&k_empty[s]), 1);
            mbar_init(smem_u32(&v_empty[s]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&p_full[i]), 4);
            mbar_init(smem_u32(&o_full[i]), 1);
        }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    for (int i = threadIdx.x; i < (2 + kStages) * 128; i += kThreads)        // the second runs are zeros throughout
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" :: "r"(qx_smem + (i / 128) * kExtra + 2048 + (i % 128) * 16), "r"(0u) : "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (warp == kSoftmaxWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = tmem_slot;
    auto fail = [&](int code) {
        atomicCAS(&g_error, 0, code);
        atomicExch(&abort_flag, 1);
    };
    auto aborted = [&]() { return *(volatile int*)&abort_flag != 0; };

    if (warp > kSoftmaxWarps) {
        // ---- unpacking ----
        const int uw = warp - kSoftmaxWarps - 1, g = lane >> 2, j4 = lane & 3;
        const int* table = a.page_table + (int64_t)a.slots[seq] * a.max_pages;
        const uint8_t* records = a.records + (int64_t)head_kv * Kv4<D>::kBytes;
        const int64_t page_stride = (int64_t)a.n_kv * Kv4<D>::kBytes;
        const int last_page = (n_keys - 1) / kPageTokens;
        Slice<D> now[2];
        auto load = [&](int step) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int page = 2 * (step0 + step) + p;      // a page behind the keys: its scores are masked, any page will do
                now[p].load(records + (int64_t)CPM_PAGE(table, min(page, last_page), a.max_pages) * page_stride, uw, lane, kv_len - page * kPageTokens);
            }
        };
        if (n_steps > 0) load(0);
        bool alive = true;                                   // after an abort the loop goes on without waiting: the warps meet at a barrier in every step
        for (int st = 0; st < n_steps; ++st) {
            if (__any_sync(0xffffffffu, aborted())) alive = false;
            const int s = st & 1, ph = (st >> 1) & 1, par = st & 1;
            // the largest magnitudes of the pages' keys and values; tokens whose values are no numbers
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                float bk = 0.f, bv = 0.f;
                uint32_t bad = 0;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float k0 = bound_of(now[p].kp[u].x), k1 = bound_of(now[p].kp[u].y);
                    bk = fmaxf(bk, fmaxf(k0 < INFINITY ? k0 : 0.f, k1 < INFINITY ? k1 : 0.f));
                    const float v0 = fmaxf(bound_of(now[p].vp[u].x), bound_of(now[p].vp[u].y)), v1 = fmaxf(bound_of(now[p].vp[u].z), bound_of(now[p].vp[u].w));
                    const bool ok0 = bound_of(now[p].vp[u].x) + bound_of(now[p].vp[u].y) < INFINITY, ok1 = bound_of(now[p].vp[u].z) + bound_of(now[p].vp[u].w) < INFINITY;
                    if (!ok0) { now[p].vp[u].x = now[p].vp[u].y = 0u; bad |= 1u << (2 * j4 + 8 * u); }
                    if (!ok1) { now[p].vp[u].z = now[p].vp[u].w = 0u; bad |= 2u << (2 * j4 + 8 * u); }
                    bv = fmaxf(bv, fmaxf(ok0 ? v0 : 0.f, ok1 ? v1 : 0.f));
                }
                const uint32_t mk = __reduce_max_sync(0xffffffffu, __float_as_uint(bk)), mv = __reduce_max_sync(0xffffffffu, __float_as_uint(bv));
                bad = __reduce_or_sync(0xffffffffu, bad);
                if (lane == 0) {
                    bounds[par][0][p][uw] = __uint_as_float(mk);
                    bounds[par][1][p][uw] = __uint_as_float(mv);
                    bads[par][p][uw] = bad;
                }
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            int ek[2], ev[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const float4 k = *reinterpret_cast<const float4*>(bounds[par][0][p]), v = *reinterpret_cast<const float4*>(bounds[par][1][p]);
                ek[p] = power_below(fmaxf(fmaxf(k.x, k.y), fmaxf(k.z, k.w)));
                const float most = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
                ev[p] = most > 0.f ? power_below(most) : -110;
            }
            if (uw == 0 && lane < 2) {
                StepInfo& i = info[st & 3];
                i.k_scale[lane] = power2(ek[lane]);
                i.v_power[lane] = ev[lane];
                i.bad[lane][0] = bads[par][lane][0] | bads[par][lane][1] << 16;
                i.bad[lane][1] = bads[par][lane][2] | bads[par][lane][3] << 16;
            }
            const auto v_of = [](uint32_t x, uint32_t y) {
                const float most = fmaxf(bound_of(x), bound_of(y));
                return most > 0.f ? power_below(most) : -110;
            };
            const int key0 = (step0 + st) * kStepKeys;
            const bool masked = key0 + kStepKeys - 1 > pos_low || (a.window && key0 <= pos_high - a.window);
            if (masked && g == 0)
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int row = 64 * p + 16 * uw + 2 * j4 + 8 * u;
                        info[st & 3].v_token[row] = v_of(now[p].vp[u].x, now[p].vp[u].y);
                        info[st & 3].v_token[row + 1] = v_of(now[p].vp[u].z, now[p].vp[u].w);
                    }
            // ---- keys ----
            if (alive && !__all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&k_empty[s]), ph ^ 1))) {
                if (lane == 0) fail(ERR_K_EMPTY);
                alive = false;
            }
#pragma unroll
            for (int p = 0; p < 2; ++p) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int row = 64 * p + 16 * uw + g + 8 * u;
                    const int e = masked ? power_below(fmaxf(bound_of(now[p].kp[u].x), bound_of(now[p].kp[u].y))) : ek[p];
                    const float down = power2(-e);
                    if (masked && j4 == 0) info[st & 3].k_token[row] = power2(e);
                    const __half2 sc[2] = {__float2half2_rn(kv4_scale(now[p].kp[u].x) * down), __float2half2_rn(kv4_scale(now[p].kp[u].y) * down)};
                    if (j4 == 0) {
                        const __half m0 = __float2half_rn(kv4_middle(now[p].kp[u].x) * down), m1 = __float2half_rn(kv4_middle(now[p].kp[u].y) * down);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(kx_smem + s * kExtra + row * 16), "r"(half2_bits(__halves2half2(m0, m0))),
                                     "r"(half2_bits(__halves2half2(m0, m1))), "r"(half2_bits(__halves2half2(m1, m1))), "r"(0u) : "memory");
                    }
                    const uint32_t at = k_smem + s * Z::kTile + row * 128;
#pragma unroll
                    for (int b = 0; b < D / 32; ++b) {
                        __half2 r[4];
                        unpack8(now[p].k[b][u], r);
                        const int h = 2 * b / (D / 32);
#pragma unroll
                        for (int odd = 0; odd < 2; ++odd) {
                            const int byte = ((32 * b + 16 * odd) % 64 + 4 * j4) * 2;
                            const uint32_t dst = at + (32 * b / 64) * kHalfBytes + ((uint32_t)(((byte >> 4) ^ (row & 7)) << 4) | (byte & 15));
                            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" :: "r"(dst), "r"(half2_bits(__hmul2(r[2 * odd], sc[h]))),
                                         "r"(half2_bits(__hmul2(r[2 * odd + 1], sc[h]))) : "memory");
                        }
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&k_full[s]));
            // ---- values ----
            if (alive && !__all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&v_empty[s]), ph ^ 1))) {
                if (lane == 0) fail(ERR_V_EMPTY);
                alive = false;
            }
#pragma unroll
            for (int p = 0; p < 2; ++p) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint4 par4 = now[p].vp[u];
                    const float d0 = power2(-(masked ? v_of(par4.x, par4.y) : ev[p])), d1 = power2(-(masked ? v_of(par4.z, par4.w) : ev[p]));
                    __half2 sc[2], md[2];                // of two neighbouring tokens
                    sc[0] = __floats2half2_rn(kv4_scale(par4.x) * d0, kv4_scale(par4.z) * d1);
                    sc[1] = __floats2half2_rn(kv4_scale(par4.y) * d0, kv4_scale(par4.w) * d1);
                    md[0] = __floats2half2_rn(kv4_middle(par4.x) * d0, kv4_middle(par4.z) * d1);
                    md[1] = __floats2half2_rn(kv4_middle(par4.y) * d0, kv4_middle(par4.w) * d1);
                    const int byte = (16 * uw + 2 * j4 + 8 * u) * 2;
#pragma unroll
                    for (int b = 0; b < D / 32; ++b) {
                        __half2 r[4];
                        unpack8(now[p].v[b][u], r);
                        const int h = 2 * b / (D / 32);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int row = 32 * b + 16 * (i >> 1) + 2 * g + (i & 1);
                            const uint32_t dst = v_smem + s * Z::kTile + p * Z::kVPage + row * 128 + ((uint32_t)(((byte >> 4) ^ (row & 7)) << 4) | (byte & 15));
                            asm volatile("st.shared.b32 [%0], %1;" :: "r"(dst), "r"(half2_bits(__hfma2(r[i], sc[h], md[h]))) : "memory");
                        }
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&v_full[s]));
            if (st + 1 < n_steps) load(st + 1);
        }
    } else if (warp == kSoftmaxWarps) {
        // ---- the products, issued by one thread ----
        if (lane == 0) {
            auto issue_qk = [&](int i, int s) {
#pragma unroll
                for (int half = 0; half < Z::kHalves; ++half) {
                    const uint64_t da = smem_desc_sw128(q_smem + i * Z::kTile + half * kHalfBytes), db = smem_desc_sw128(k_smem + s * Z::kTile + half * kHalfBytes);
#pragma unroll
                    for (int k = 0; k < 4; ++k) tcgen05_mma_f16(tmem + i * 128, da + 2 * k, db + 2 * k, Z::idesc(128), (half | k) != 0);
                }
                tcgen05_mma_f16(tmem + i * 128, smem_desc_plain(qx_smem + i * kExtra), smem_desc_plain(kx_smem + s * kExtra), Z::idesc(128), 1);
            };
            auto issue_pv = [&](int i, int s, bool accumulate) {
#pragma unroll
                for (int page = 0; page < 2; ++page) {
                    const uint64_t db = smem_desc_sw128(v_smem + s * Z::kTile + page * Z::kVPage);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tcgen05_mma_f16_ts(tmem + Z::kO + i * D, tmem + i * 128 + page * 32 + k * 8, db + 2 * k, Z::idesc(D), accumulate || (page | k) != 0);
                }
            };
            bool ok = n_steps > 0;
            if (ok && !mbar_wait_bounded(smem_u32(&q_full), 0)) { fail(ERR_Q); ok = false; }
            if (ok && !mbar_wait_bounded(smem_u32(&k_full[0]), 0)) { fail(ERR_K_FULL); ok = false; }
            if (ok) {
                tcgen05_fence_after();
                issue_qk(0, 0);
                tcgen05_commit(smem_u32(&s_full[0]));
                issue_qk(1, 0);
                tcgen05_commit(smem_u32(&s_full[1]));
                tcgen05_commit(smem_u32(&k_empty[0]));
            }
            for (int st = 0; ok && st < n_steps && !aborted(); ++st) {
                const int s = st & 1, ph = (st >> 1) & 1, s1 = (st + 1) & 1, ph1 = ((st + 1) >> 1) & 1;
                if (!mbar_wait_bounded(smem_u32(&v_full[s]), ph)) { fail(ERR_V_FULL); break; }
                for (int i = 0; i < 2; ++i) {
                    if (!mbar_wait_bounded(smem_u32(&p_full[i]), st & 1)) { fail(ERR_P_FULL); ok = false; break; }
                    tcgen05_fence_after();
                    issue_pv(i, s, st > 0);
                    if (i == 1) tcgen05_commit(smem_u32(&v_empty[s]));
                    if (st + 1 < n_steps) {
                        if (i == 0 && !mbar_wait_bounded(smem_u32(&k_full[s1]), ph1)) { fail(ERR_K_FULL); ok = false; break; }
                        tcgen05_fence_after();
                        issue_qk(i, s1);
                        tcgen05_commit(smem_u32(&s_full[i]));
                        if (i == 1) tcgen05_commit(smem_u32(&k_empty[s1]));
                    } else {
                        tcgen05_commit(smem_u32(&o_full[i]));
                    }
                }
            }
        }
    } else {
        // ---- queries, softmax and output: a thread to a row ----
        const int i = warp >> 2, r = threadIdx.x & 127, row = first + 128 * i + r;
        const bool valid = 128 * i + r < n_rows;
        const int64_t at = ((int64_t)(q_begin + row0 + row / a.group) * a.n_heads + head_kv * a.group + row % a.group) * D;
        const int limit = valid ? history + row0 + row / a.group : -1;      // the last key that the row sees
        const int from = a.window ? max(0, limit - a.window + 1) : 0;       // and the first
        float sl2;
        {
            // divided by a power of two so that the largest channel lies between 256 and 512, and a half row's sum below 65,504
            uint4 raw[D / 8];
            float most = 0.f;
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                raw[c] = valid ? *reinterpret_cast<const uint4*>(a.q + at + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
                const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) most = fmaxf(most, fmaxf(fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xffff0000u))));
            }
            const int e2 = most > 0.f && most < INFINITY ? power_below(most) - 8 : 0;
            const float down = power2(-e2);
            sl2 = power2(e2) * a.scale * 1.4426950408889634f;
            float total[2] = {0.f, 0.f};
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
                uint32_t h[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y0 = __uint_as_float(w[e] << 16) * down, y1 = __uint_as_float(w[e] & 0xffff0000u) * down;
                    total[c / (D / 16)] += y0 + y1;
                    h[e] = half2_bits(__floats2half2_rn(y0, y1));
                }
                const uint32_t dst = q_smem + i * Z::kTile + (c / 8) * kHalfBytes + r * 128 + (uint32_t)(((c & 7) ^ (r & 7)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(dst), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
            }
            __half term[2][3];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float left = total[h];
#pragma unroll
                for (int e = 0; e < 3; ++e) {
                    term[h][e] = __float2half_rn(left);
                    left -= __half2float(term[h][e]);
                }
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(qx_smem + i * kExtra + r * 16), "r"(half2_bits(__halves2half2(term[0][0], term[0][1]))),
                         "r"(half2_bits(__halves2half2(term[0][2], term[1][0]))), "r"(half2_bits(__halves2half2(term[1][1], term[1][2]))), "r"(0u) : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&q_full));
        }
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t s_addr = lanes + i * 128, o_addr = lanes + Z::kO + i * D;
        float m = -INFINITY, l = 0.f;
        int power = -1000;                                   // the accumulator stands for O / 2^power
        bool ok = true;
        for (int st = 0; st < n_steps; ++st) {
            if (__any_sync(0xffffffffu, aborted())) { ok = false; break; }
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&s_full[i]), st & 1))) {
                if (lane == 0) fail(ERR_S_FULL);
                ok = false;
                break;
            }
            tcgen05_fence_after();
            const StepInfo& inf = info[st & 3];
            const int key0 = (step0 + st) * kStepKeys;
            const bool masked = key0 + kStepKeys - 1 > pos_low || (a.window && key0 <= pos_high - a.window);
            uint32_t v[2][32];
            auto get = [&](int p) {                           // a page's 64 scores
                tmem_load_32cols(s_addr + 64 * p, v[0]);
                tmem_load_32cols(s_addr + 64 * p + 32, v[1]);
                tmem_load_wait();
                if (masked) {
                    const int key = key0 + 64 * p;
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            v[c][e] = key + c * 32 + e > limit || key + c * 32 + e < from ? 0xff800000u : __float_as_uint(__uint_as_float(v[c][e]) * inf.k_token[64 * p + 32 * c + e]);
                }
            };
            auto top = [&]() {
                float mx = -INFINITY;
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int e = 0; e < 32; e += 2) mx = max3(mx, __uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1]));
                return mx;
            };
            const float sl[2] = {masked ? sl2 : sl2 * inf.k_scale[0], masked ? sl2 : sl2 * inf.k_scale[1]};
            int highest = max(inf.v_power[0], inf.v_power[1]);
            if (masked) {
                highest = -110;
#pragma unroll 4
                for (int e = 0; e < kStepKeys; ++e)
                    if (key0 + e <= limit && key0 + e >= from) highest = max(highest, inf.v_token[e]);
            }
            get(1);
            float m_new = top() * sl[1];
            get(0);
            m_new = fmaxf(m_new, top() * sl[0]);
            const bool grow = m_new > m + kBehind || (m == -INFINITY && m_new > -INFINITY);
            const int power_new = max(power, highest);
            if (__any_sync(0xffffffffu, grow || power_new > power)) {
                const float alpha = grow ? ex2(m - m_new) : 1.f;        // 0 the first time
                l *= alpha;
                if (st > 0) {
                    const float by = alpha * power2(power - power_new);
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[32];
                        tmem_load_32cols(o_addr + c * 32, o);
                        tmem_load_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * by);
                        tmem_store_32cols(o_addr + c * 32, o);
                    }
                }
                if (grow) m = m_new;
                power = power_new;
            }
            const float use = m == -INFINITY ? 0.f : m;
            auto weigh = [&](int p) {
                float2 sum = make_float2(0.f, 0.f);
                const float factor = power2(inf.v_power[p] - power);
                const float2 by = make_float2(sl[p], sl[p]), less = make_float2(-use, -use);
                float2 f2 = make_float2(factor, factor);
                uint32_t packed[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const float2 x = fma2(make_float2(__uint_as_float(v[e >> 4][(2 * e) & 31]), __uint_as_float(v[e >> 4][(2 * e + 1) & 31])), by, less);
                    const float2 w = make_float2(ex2(x.x), ex2(x.y));
                    sum = add2(sum, w);
                    if (masked) f2 = make_float2(power2(inf.v_token[64 * p + 2 * e] - power), power2(inf.v_token[64 * p + 2 * e + 1] - power));
                    float2 y = mul2(w, f2);
                    if (masked) y = make_float2(w.x > 0.f ? y.x : 0.f, w.y > 0.f ? y.y : 0.f);
                    packed[e] = half2_bits(__floats2half2_rn(y.x, y.y));
                }
                l += sum.x + sum.y;
                tmem_store_32cols(s_addr + p * 32, packed);
            };
            // (the second page's P lies over the first page's scores, which are in registers by then)
            weigh(0);
            get(1);
            weigh(1);
            if (inf.bad[0][0] | inf.bad[0][1] | inf.bad[1][0] | inf.bad[1][1]) {
                // values that are no numbers are not in the tile: the rows that see them are no numbers
#pragma unroll 1
                for (int e = 0; e < kStepKeys; ++e)
                    if ((inf.bad[e >> 6][(e >> 5) & 1] >> (e & 31) & 1) && key0 + e <= limit && key0 + e >= from) l = NAN;
            }
            tmem_store_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&p_full[i]));
        }
        if (ok && n_steps > 0) {
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(smem_u32(&o_full[i]), 0))) {
                if (lane == 0) fail(ERR_O_FULL);
                ok = false;
            }
            tcgen05_fence_after();
        }
        if (ok) {
            const float inv = l == 0.f ? 0.f : power2(power) / l;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                if (n_steps > 0) {
                    tmem_load_32cols(o_addr + c * 32, o);
                    tmem_load_wait();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;
                }
                if (valid)
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        store4(a.out + at + c * 32 + e, make_float4(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv,
                                                                    __uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv));
            }
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == kSoftmaxWarps) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
    }
}

template <int D>
int prompt(const Args& a, int n_tiles, cudaStream_t stream) {
    static bool done[kMaxDevices];
    const int status = ensure_dynamic_smem(kv4_prompt_kernel<D>, Sizes<D>::kSmem, done);
    if (status != CPM_OK) return status;
    const int64_t parts = (int64_t)((a.tile_tokens * a.group + kRows - 1) / kRows) * a.n_kv;
    if (n_tiles > 65535 || parts > 0x7fffffff) return CPM_BAD_ARGUMENT;
    cpm_launch(kLaunchAttention, kv4_prompt_kernel<D>, dim3((unsigned)parts, n_tiles), kThreads, Sizes<D>::kSmem, stream, a);
    return launch_status();
}

}  // namespace kv4p

// Reads and clears the error that a kernel recorded (0: none).
CPM_API int cpm_kv4_prompt_error() {
    int code = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&code, kv4p::g_error, sizeof(int)) != cudaSuccess) return -1;
    if (code) cudaMemcpyToSymbol(kv4p::g_error, &zero, sizeof(int));
    return code;
}

// q, out bf16 [tokens, heads, d]; the tiles are of 64 tokens, taken together up to 256 rows of a key-value head.
CPM_API int cpm_kv4_prompt(const void* q, const void* records, void* out, const int* kv_len, const int* slots, const int* page_table, int max_pages,
                           const int* cu_q, const int* tile_seq, const int* tile_row, int n_tiles, int n_heads, int n_kv, int d, int window, float scale,
                           cudaStream_t stream) {
    if (n_tiles <= 0) return CPM_OK;
    if (n_heads < 1 || n_kv < 1 || n_heads % n_kv || window < 0 || !(scale > 0.f)) return CPM_BAD_ARGUMENT;
    if (((uintptr_t)records | (uintptr_t)q | (uintptr_t)out) & 15) return CPM_BAD_ARGUMENT;
    const int group = n_heads / n_kv;
    const int tile_tokens = group == 1 ? 256 : group == 2 ? 128 : 64;
    const kv4p::Args a{(const bf16*)q, (bf16*)out, (const uint8_t*)records, kv_len, slots, page_table, cu_q, tile_seq, tile_row, max_pages, n_heads, n_kv,
                       group, window, tile_tokens, scale};
    switch (d) {
        case 64: return kv4p::prompt<64>(a, n_tiles, stream);
        case 128: return kv4p::prompt<128>(a, n_tiles, stream);
        default: return CPM_BAD_ARGUMENT;
    }
}
