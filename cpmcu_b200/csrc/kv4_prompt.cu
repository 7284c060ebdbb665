// Attention of prompt tokens over the 4-bit cache on the fifth-generation tensor cores, head sizes 64 and 128.
//
// A block takes 256 rows of queries, the query heads of one key-value head for some consecutive tokens (16 tokens at 16 heads), so that all of them share
// every key and value.  Four warps unpack the codes, a page of 64 keys a step, into fp16 tiles in shared memory: K [keys][d] and V
// [d][keys], 128-byte swizzle, the K-major operands of S = Q K^T and O += P V (tcgen05.mma, accumulators in tensor memory); four tiles of each.  Eight
// warps are the softmax, a thread to a row, which writes P as fp16 over the S it read; four more issue the products, one each for the scores and the
// values of a half of 128 rows.  A half has two S: the next page's scores are formed while this one's are in the softmax, so that only the softmax
// itself is in a row's way.  (2,048 tokens of 32 heads on 2 behind 4,101 keys, 172 GFLOP: one S of 128 keys, whose softmax waits for its products, 347
// us; two S and one issuing warp 333, two issuing warps 269, powers of two by 16 tokens instead of by page 262, four issuing warps and one barrier for a
// page's keys and values 247, products issued by an elected thread of a converged warp instead of by lane 0 in a branch 231, no look at the abort flag
// before a wait has failed 226, 760 TFLOP/s.)
//
// fp16 and not bf16: its 11 bits hold s (c - 8) exactly, 8 bits times 3, so that scores are as exact as their fp32 sums.  The rest of a
// key's product, m times the sum of the query's half row, is 16 more columns of the operands: m three times and the sum as three fp16 numbers,
// for both halves.  A value is rounded to 11 bits (2^-12 of it, where the output has 8), a weight times its value's power of two to 11 as well; what is
// below 2^-14 of the largest of its 16 tokens' values, or of the row's largest weight and power, keeps fewer, an error of 2^-25 of these.
// What fp16 lacks in range is taken care of by powers of two: a query row, 16 tokens' keys and 16 tokens' values are divided by the power of two below
// their largest magnitude, scores are multiplied by the first two again, and the accumulator stands for O / 2^E with E the largest power of the
// values so far.
//
// Unpacking a key and a value costs about two instructions a number, 256 rows of softmax four to five; a block of 128 rows would pay it twice.
// Bound by two chains of about 2,400 cycles a page, the four unpacking warps' (one to a scheduler, which waits for each instruction before the next) and
// the softmax's (two to a scheduler; exponentials alone are 1,024), where the products take 1,400.  (Eight unpacking warps with registers that the issuing
// warps give up, 228 us: the softmax is as long.  Scores taken 32 at a time to need fewer registers, 250.)
//
// Every wait is bounded: a block that gives up records an error, stops, lets the products in flight end (tiles are written by ordinary stores, so
// nothing else is), frees its tensor memory and returns.
#include "kv4.cuh"
#include "tcgen05.cuh"
#include <type_traits>

CPM_BOUNDS_TU(kv4_prompt)

namespace kv4p {
using namespace tc5;

constexpr int kRows = 256;
constexpr int kStages = 4;                              // tiles of keys, and of values
constexpr int kInfos = 8;                               // steps that unpacking may be ahead of the softmax, and one
constexpr int kSoftmaxWarps = 8, kUnpackWarps = 4;
constexpr int kIssueWarps = 4;                          // scores and weighted values of both halves
constexpr int kThreads = (kSoftmaxWarps + kIssueWarps + kUnpackWarps) * 32;      // 128 registers each
constexpr float kBehind = 8.0f;                         // the running maximum may lie 2^8 behind
constexpr int kQHalf = 128 * 128, kKHalf = 64 * 128;    // 128 rows of Q, 64 keys: runs of 128 bytes
constexpr int kQExtra = 128 * 32, kKExtra = 64 * 32;    // 16 more columns, two runs of 16 bytes a row
// Matrix descriptor of such a tile of ``rows`` rows: K-major, no swizzle; groups of 8 rows 128 bytes apart, the two runs 16 * rows.
__device__ __forceinline__ uint64_t smem_desc_plain(uint32_t addr, int rows) {
    return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)rows << 16) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}

template <int D>
struct Sizes {
    static constexpr int kHalves = D / 64;
    static constexpr int kQ = 128 * D * 2, kKv = kPageTokens * D * 2;       // 128 rows of Q; a page's keys, or values
    static constexpr int kSmem = 2 * kQ + 2 * kStages * kKv + 2 * kQExtra + kStages * kKExtra + 1024;
    static constexpr uint32_t idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }     // fp16 in, fp32 sums
    static constexpr int kO = 256;                      // tensor memory: half i's S at 128 i and 128 i + 64, its O at 256 + i d
};

struct Args {
    const bf16* q;
    bf16* out;
    const uint8_t* records;
    const int *kv_len, *slots, *page_table, *cu_q, *tile_seq, *tile_row;
    float* parts;                                       // with shares of the keys: [share][row of q][d + 2]: values, maximum, sum
    int max_pages, n_heads, n_kv, group, window, tile_tokens, n_tokens;
    float scale;
};

// What unpacking a page tells the softmax: for each 16 tokens, and per token where some row sees the page in part.
struct StepInfo {
    alignas(16) float k_token[kPageTokens];
    int v_token[kPageTokens];
    alignas(16) float k_scale[4];
    alignas(16) int v_power[4];
    alignas(16) uint32_t bad[4];                        // value half rows that are no numbers: bit 2 t + h of token t
};

enum : int { ERR_Q = 1, ERR_FULL, ERR_EMPTY, ERR_S_FULL, ERR_P_FULL, ERR_O_FULL };
__device__ int g_error;

// True in one thread of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
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
    uint32_t k1, v1;                                    // one of the 32 parameters of the 16 rows: row lane / 2, half lane % 2
    __device__ __forceinline__ void load(const uint8_t* rec, int slice, int lane) {
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
        }
        k1 = *reinterpret_cast<const uint32_t*>(rec + L::kKeyParams + slice * 128 + lane * 4);
        v1 = *reinterpret_cast<const uint32_t*>(rec + L::kValueParams + slice * 128 + lane * 4);
    }
    // Behind the sequence's end, after ``tokens`` of the page: what lies there may be no number.
    __device__ __forceinline__ void trim(int slice, int lane, int tokens) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int rk = 16 * slice + (lane >> 2) + 8 * u, rv = 16 * slice + 2 * (lane & 3) + 8 * u;
            if (rk >= tokens) kp[u] = make_uint2(0u, 0u);
            if (rv >= tokens) vp[u].x = vp[u].y = 0u;
            if (rv + 1 >= tokens) vp[u].z = vp[u].w = 0u;
        }
        if (16 * slice + (lane >> 1) >= tokens) k1 = v1 = 0u;
    }
};
__device__ __forceinline__ float bound_of(uint32_t p) { return fabsf(kv4_middle(p)) + 8.f * kv4_scale(p); }

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
kv4_prompt_kernel(const __grid_constant__ Args a) {
    using Z = Sizes<D>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t q_full[2], full[kStages], empty[kStages], s_full[2][2], p_full[2][2], o_done[2][2];      // (of two S the softmax may be two steps ahead of the products: each has its own barriers)
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ StepInfo info[kInfos];
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
    // few rows and many keys: a tile's pages are shared out over gridDim.z blocks
    const int first_page = a.window ? max(0, pos_low - a.window + 1) / kPageTokens : 0;
    const int all_steps = max(0, (n_keys + kPageTokens - 1) / kPageTokens - first_page), share = (all_steps + gridDim.z - 1) / gridDim.z;
    const int page0 = first_page + blockIdx.z * share, n_steps = max(0, min(share, all_steps - (int)blockIdx.z * share));
    // whether some row sees some key of a step and not another
    const auto in_part = [&](int st) {
        const int key0 = (page0 + st) * kPageTokens;
        return key0 + kPageTokens - 1 > pos_low || (a.window && key0 <= pos_high - a.window);
    };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_smem = base, k_smem = base + 2 * Z::kQ, v_smem = k_smem + kStages * Z::kKv, qx_smem = v_smem + kStages * Z::kKv, kx_smem = qx_smem + 2 * kQExtra;
    if (threadIdx.x == 0) {
#pragma unroll 1
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&full[s]), kUnpackWarps);
            mbar_init(smem_u32(&empty[s]), 2);
        }
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&q_full[i]), 4);
            mbar_init(smem_u32(&s_full[i][0]), 1);
            mbar_init(smem_u32(&s_full[i][1]), 1);
            mbar_init(smem_u32(&p_full[i][0]), 4);
            mbar_init(smem_u32(&p_full[i][1]), 4);
            mbar_init(smem_u32(&o_done[i][0]), 1);
            mbar_init(smem_u32(&o_done[i][1]), 1);
        }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // the second runs of the further columns are zeros throughout
#pragma unroll 1
    for (int i = threadIdx.x; i < 2 * 128; i += kThreads)
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" :: "r"(qx_smem + (i / 128) * kQExtra + 2048 + (i % 128) * 16), "r"(0u) : "memory");
#pragma unroll 1
    for (int i = threadIdx.x; i < kStages * 64; i += kThreads)
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" :: "r"(kx_smem + (i / 64) * kKExtra + 1024 + (i % 64) * 16), "r"(0u) : "memory");
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
    // A wait that another role's failure ends too (looked at only when the barrier is not ready: it would lengthen every step).
    auto wait = [&](const uint64_t& bar, uint32_t parity) {
        const uint32_t at = smem_u32(&bar);
        if (mbar_try_wait(at, parity)) return true;
#pragma unroll 1
        for (uint32_t i = 1; i < kSpinLimit; ++i) {
            if (mbar_try_wait(at, parity)) return true;
            if (*(volatile int*)&abort_flag != 0) break;
        }
        return false;
    };

    if (warp >= kSoftmaxWarps + kIssueWarps) {
        // ---- unpacking: a warp takes 16 tokens of every page, whose codes were asked for a page ahead ----
        const int slice = warp - kSoftmaxWarps - kIssueWarps, g = lane >> 2, j4 = lane & 3;
        const int* table = a.page_table + (int64_t)a.slots[seq] * a.max_pages;
        const uint8_t* records = a.records + (int64_t)head_kv * Kv4<D>::kBytes;
        const int64_t page_stride = (int64_t)a.n_kv * Kv4<D>::kBytes;
        int ids = 0;                                          // 32 page numbers, one a lane
        auto load = [&](Slice<D>& to, int st) {
            if ((st & 31) == 0) ids = st + lane < n_steps ? CPM_PAGE(table, page0 + st + lane, a.max_pages) : 0;
            const int number = __shfl_sync(0xffffffffu, ids, st & 31);
            to.load(records + (int64_t)number * page_stride, slice, lane);
        };
        // where a lane's numbers go in a swizzled tile, by what of the place depends on the lane
        uint32_t k_off[4], v_off[2][2];
#pragma unroll
        for (int x = 0; x < 4; ++x) k_off[x] = k_smem + (16 * slice + g) * 128 + (((2 * x) ^ (j4 >> 1) ^ g) << 4) + (j4 & 1) * 8;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) v_off[u][e] = v_smem + (2 * g + e) * 128 + (((2 * slice + u) ^ ((2 * g + e) & 7)) << 4) + 4 * j4;
        Slice<D> even, odd;
        if (n_steps > 0) load(even, 0);
        bool alive = true;                                   // after an abort the loop goes on without waiting
        const auto unpack = [&](Slice<D>& now, int st) {
            const int left = kv_len - (page0 + st) * kPageTokens;
            if (left < kPageTokens) now.trim(slice, lane, left);
            const int s = st % kStages, ph = (st / kStages) & 1;
            // the largest magnitudes of the 16 tokens' keys and values; value half rows that are no numbers
            const float k_bound = bound_of(now.k1), v_bound = bound_of(now.v1);
            const bool v_finite = v_bound < INFINITY;
            const float most_k = __uint_as_float(__reduce_max_sync(0xffffffffu, k_bound < INFINITY ? __float_as_uint(k_bound) : 0u));
            const uint32_t bad = __ballot_sync(0xffffffffu, !v_finite);
            if (bad) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t mine = bad >> (4 * j4 + 16 * u);
                    if (mine & 1) now.vp[u].x = 0u;
                    if (mine & 2) now.vp[u].y = 0u;
                    if (mine & 4) now.vp[u].z = 0u;
                    if (mine & 8) now.vp[u].w = 0u;
                }
            }
            const float most_v = __uint_as_float(__reduce_max_sync(0xffffffffu, v_finite ? __float_as_uint(v_bound) : 0u));
            const int ek = power_below(most_k), ev = most_v > 0.f ? power_below(most_v) : -110;
            StepInfo& inf = info[st % kInfos];
            if (lane == 0) {
                inf.k_scale[slice] = power2(ek);
                inf.v_power[slice] = ev;
                inf.bad[slice] = bad;
            }
            float down_k[2] = {power2(-ek), power2(-ek)}, down_v[2][2] = {{power2(-ev), power2(-ev)}, {power2(-ev), power2(-ev)}};
            if (in_part(st)) {                                // every token by itself
                const auto v_of = [](uint32_t x, uint32_t y) {
                    const float most = fmaxf(bound_of(x), bound_of(y));
                    return most > 0.f ? power_below(most) : -110;
                };
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int k_row = 16 * slice + g + 8 * u, v_row = 16 * slice + 2 * j4 + 8 * u;
                    const int e = power_below(fmaxf(bound_of(now.kp[u].x), bound_of(now.kp[u].y))), e0 = v_of(now.vp[u].x, now.vp[u].y), e1 = v_of(now.vp[u].z, now.vp[u].w);
                    down_k[u] = power2(-e);
                    down_v[u][0] = power2(-e0);
                    down_v[u][1] = power2(-e1);
                    if (j4 == 0) inf.k_token[k_row] = power2(e);
                    if (g == 0) {
                        inf.v_token[v_row] = e0;
                        inf.v_token[v_row + 1] = e1;
                    }
                }
            }
            if (alive && !__all_sync(0xffffffffu, wait(empty[s], ph ^ 1))) {
                if (lane == 0) fail(ERR_EMPTY);
                alive = false;
            }
            // ---- keys ----
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float down = down_k[u];
                const __half2 sc[2] = {__float2half2_rn(kv4_scale(now.kp[u].x) * down), __float2half2_rn(kv4_scale(now.kp[u].y) * down)};
                if (j4 == 0) {
                    const __half m0 = __float2half_rn(kv4_middle(now.kp[u].x) * down), m1 = __float2half_rn(kv4_middle(now.kp[u].y) * down);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(kx_smem + s * kKExtra + (16 * slice + g + 8 * u) * 16),
                                 "r"(half2_bits(__halves2half2(m0, m0))), "r"(half2_bits(__halves2half2(m0, m1))), "r"(half2_bits(__halves2half2(m1, m1))), "r"(0u) : "memory");
                }
#pragma unroll
                for (int b = 0; b < D / 32; ++b) {
                    __half2 r[4];
                    unpack8(now.k[b][u], r);
                    const int h = 2 * b / (D / 32);
#pragma unroll
                    for (int odd = 0; odd < 2; ++odd)
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" :: "r"(k_off[2 * (b & 1) + odd] + s * Z::kKv + (b >> 1) * kKHalf + u * 1024),
                                     "r"(half2_bits(__hmul2(r[2 * odd], sc[h]))), "r"(half2_bits(__hmul2(r[2 * odd + 1], sc[h]))) : "memory");
                }
            }
            // ---- values ----
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint4 p4 = now.vp[u];
                const float d0 = down_v[u][0], d1 = down_v[u][1];       // of two neighbouring tokens
                const __half2 sc[2] = {__floats2half2_rn(kv4_scale(p4.x) * d0, kv4_scale(p4.z) * d1), __floats2half2_rn(kv4_scale(p4.y) * d0, kv4_scale(p4.w) * d1)};
                const __half2 md[2] = {__floats2half2_rn(kv4_middle(p4.x) * d0, kv4_middle(p4.z) * d1), __floats2half2_rn(kv4_middle(p4.y) * d0, kv4_middle(p4.w) * d1)};
#pragma unroll
                for (int b = 0; b < D / 32; ++b) {
                    __half2 r[4];
                    unpack8(now.v[b][u], r);
                    const int h = 2 * b / (D / 32);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        asm volatile("st.shared.b32 [%0], %1;" :: "r"(v_off[u][i & 1] + s * Z::kKv + (32 * b + 16 * (i >> 1)) * 128),
                                     "r"(half2_bits(__hfma2(r[i], sc[h], md[h]))) : "memory");
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&full[s]));
        };
#pragma unroll 1
        for (int st = 0; st < n_steps; st += 2) {
            if (st + 1 < n_steps) load(odd, st + 1);
            unpack(even, st);
            if (st + 1 >= n_steps) break;
            if (st + 2 < n_steps) load(even, st + 2);
            unpack(odd, st + 1);
        }
    } else if (warp >= kSoftmaxWarps && warp < kSoftmaxWarps + 2) {
        // ---- a half's scores, issued by one thread as soon as a page's keys are there and an S is free ----
        const int i = warp - kSoftmaxWarps;
        if (n_steps > 0) {
            if (!wait(q_full[i], 0)) fail(ERR_Q);
#pragma unroll 1
            for (int st = 0; st < n_steps; ++st) {
                const int s = st % kStages;
                if (!__all_sync(0xffffffffu, wait(full[s], (st / kStages) & 1))) { fail(ERR_FULL); break; }
                if (st >= 2 && !__all_sync(0xffffffffu, wait(o_done[i][st & 1], ((st - 2) >> 1) & 1))) { fail(ERR_O_FULL); break; }
                tcgen05_fence_after();
                if (elect_one()) {
                    const uint32_t to = tmem + i * 128 + (st & 1) * 64;
#pragma unroll
                    for (int half = 0; half < Z::kHalves; ++half) {
                        const uint64_t da = smem_desc_sw128(q_smem + i * Z::kQ + half * kQHalf), db = smem_desc_sw128(k_smem + s * Z::kKv + half * kKHalf);
#pragma unroll
                        for (int k = 0; k < 4; ++k) tcgen05_mma_f16(to, da + 2 * k, db + 2 * k, Z::idesc(64), (half | k) != 0);
                    }
                    tcgen05_mma_f16(to, smem_desc_plain(qx_smem + i * kQExtra, 128), smem_desc_plain(kx_smem + s * kKExtra, 64), Z::idesc(64), 1);
                    tcgen05_commit(smem_u32(&s_full[i][st & 1]));
                }
                __syncwarp();
            }
        }
        __syncwarp();
    } else if (warp >= kSoftmaxWarps + 2) {
        // ---- a half's weighted values, issued by one thread ----
        const int i = warp - kSoftmaxWarps - 2;
#pragma unroll 1
        for (int st = 0; st < n_steps; ++st) {
            const int s = st % kStages;
            if (!__all_sync(0xffffffffu, wait(full[s], (st / kStages) & 1))) { fail(ERR_FULL); break; }
            if (!__all_sync(0xffffffffu, wait(p_full[i][st & 1], (st >> 1) & 1))) { fail(ERR_P_FULL); break; }
            tcgen05_fence_after();
            if (elect_one()) {
                const uint64_t db = smem_desc_sw128(v_smem + s * Z::kKv);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    tcgen05_mma_f16_ts(tmem + Z::kO + i * D, tmem + i * 128 + (st & 1) * 64 + k * 8, db + 2 * k, Z::idesc(D), st > 0 || k != 0);
                tcgen05_commit(smem_u32(&o_done[i][st & 1]));
                tcgen05_commit(smem_u32(&empty[s]));             // (the page's scores were formed before)
            }
            __syncwarp();
        }
        __syncwarp();
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
            float most = 0.f;
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
                const uint4 raw = valid ? *reinterpret_cast<const uint4*>(a.q + at + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
                const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) most = fmaxf(most, fmaxf(fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xffff0000u))));
            }
            const int e2 = most > 0.f && most < INFINITY ? power_below(most) - 8 : 0;
            const float down = power2(-e2);
            sl2 = power2(e2) * a.scale * 1.4426950408889634f;
            __half term[2][3];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float total = 0.f;
#pragma unroll 2
                for (int c = h * (D / 16); c < (h + 1) * (D / 16); ++c) {
                    const uint4 raw = valid ? *reinterpret_cast<const uint4*>(a.q + at + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
                    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
                    uint32_t x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float y0 = __uint_as_float(w[e] << 16) * down, y1 = __uint_as_float(w[e] & 0xffff0000u) * down;
                        total += y0 + y1;
                        x[e] = half2_bits(__floats2half2_rn(y0, y1));
                    }
                    const uint32_t dst = q_smem + i * Z::kQ + (c / 8) * kQHalf + r * 128 + (uint32_t)(((c & 7) ^ (r & 7)) << 4);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(dst), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
                }
#pragma unroll
                for (int e = 0; e < 3; ++e) {
                    term[h][e] = __float2half_rn(total);
                    total -= __half2float(term[h][e]);
                }
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(qx_smem + i * kQExtra + r * 16), "r"(half2_bits(__halves2half2(term[0][0], term[0][1]))),
                         "r"(half2_bits(__halves2half2(term[0][2], term[1][0]))), "r"(half2_bits(__halves2half2(term[1][1], term[1][2]))), "r"(0u) : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&q_full[i]));
        }
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t o_addr = lanes + Z::kO + i * D;
        float m = -INFINITY, l = 0.f;
        uint32_t lost = 0;                                   // bit h: the row sees a value whose half h is no number
        int power = -1000;                                   // the accumulator stands for O / 2^power
        bool ok = true;
#pragma unroll 1
        for (int st = 0; st < n_steps; ++st) {
            if (!__all_sync(0xffffffffu, wait(s_full[i][st & 1], (st >> 1) & 1))) {
                if (lane == 0) fail(ERR_S_FULL);
                ok = false;
                break;
            }
            tcgen05_fence_after();
            const StepInfo& inf = info[st % kInfos];
            const int key0 = (page0 + st) * kPageTokens;
            const uint32_t s_addr = lanes + i * 128 + (st & 1) * 64;
            const auto soften = [&](auto masked_tag) {
                constexpr bool MASKED = decltype(masked_tag)::value;
                uint32_t v[2][32];
                tmem_load_32cols(s_addr, v[0]);
                tmem_load_32cols(s_addr + 32, v[1]);
                tmem_load_wait();
                const int4 v_power = *reinterpret_cast<const int4*>(inf.v_power);
                const float4 k_scale = *reinterpret_cast<const float4*>(inf.k_scale);
                const float by_slice[4] = {MASKED ? sl2 : sl2 * k_scale.x, MASKED ? sl2 : sl2 * k_scale.y, MASKED ? sl2 : sl2 * k_scale.z, MASKED ? sl2 : sl2 * k_scale.w};
                int highest = max(max(v_power.x, v_power.y), max(v_power.z, v_power.w));
                if constexpr (MASKED) {
                    highest = -110;
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const int key = key0 + 32 * c + e;
                            const bool seen = key <= limit && key >= from;
                            v[c][e] = seen ? __float_as_uint(__uint_as_float(v[c][e]) * inf.k_token[32 * c + e]) : 0xff800000u;
                            if (seen) highest = max(highest, inf.v_token[32 * c + e]);
                        }
                }
                float m_new = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float most = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 16; e += 2) most = max3(most, __uint_as_float(v[c / 2][16 * (c & 1) + e]), __uint_as_float(v[c / 2][16 * (c & 1) + e + 1]));
                    m_new = fmaxf(m_new, most * by_slice[c]);
                }
                const bool grow = m_new > m + kBehind || (m == -INFINITY && m_new > -INFINITY);
                const int power_new = max(power, highest);
                if (__any_sync(0xffffffffu, grow || power_new > power)) {
                    const float alpha = grow ? ex2(m - m_new) : 1.f;        // 0 the first time
                    l *= alpha;
                    if (st > 0) {
                        // the products of the page before have to be in O
                        if (!__all_sync(0xffffffffu, wait(o_done[i][(st - 1) & 1], ((st - 1) >> 1) & 1)) && lane == 0) fail(ERR_O_FULL);
                        tcgen05_fence_after();
                        const float by = alpha * power2(power - power_new);
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tmem_load_16cols(o_addr + c * 16, o);
                            tmem_load_wait();
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * by);
                            tmem_store_16cols(o_addr + c * 16, o);
                        }
                    }
                    if (grow) m = m_new;
                    power = power_new;
                }
                const float use = m == -INFINITY ? 0.f : m;
                const float factor[4] = {power2(v_power.x - power), power2(v_power.y - power), power2(v_power.z - power), power2(v_power.w - power)};
                const float2 less = make_float2(-use, -use);
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                for (int run = 0; run < 2; ++run) {
                    uint32_t packed[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int c = 2 * run + e / 8;
                        const float2 by = make_float2(by_slice[c], by_slice[c]);
                        float2 f2 = make_float2(factor[c], factor[c]);
                        const float2 x = fma2(make_float2(__uint_as_float(v[run][2 * e]), __uint_as_float(v[run][2 * e + 1])), by, less);
                        const float2 w = make_float2(ex2(x.x), ex2(x.y));
                        sum = add2(sum, w);
                        if constexpr (MASKED) f2 = make_float2(power2(inf.v_token[32 * run + 2 * e] - power), power2(inf.v_token[32 * run + 2 * e + 1] - power));
                        float2 y = mul2(w, f2);
                        if constexpr (MASKED) y = make_float2(w.x > 0.f ? y.x : 0.f, w.y > 0.f ? y.y : 0.f);
                        packed[e] = half2_bits(__floats2half2_rn(y.x, y.y));
                    }
                    tmem_store_16cols(s_addr + 16 * run, packed);
                }
                l += sum.x + sum.y;
            };
            // (two copies of the code: the one for pages that every row sees whole has nothing of the other's)
            if (in_part(st)) soften(std::true_type{});
            else soften(std::false_type{});
            if (inf.bad[0] | inf.bad[1] | inf.bad[2] | inf.bad[3]) {
                // values that are no numbers are not in the tile: the halves of the rows that see them are no numbers
#pragma unroll 1
                for (int e = 0; e < kPageTokens; ++e)
                    if (key0 + e <= limit && key0 + e >= from) lost |= inf.bad[e >> 4] >> (2 * (e & 15)) & 3u;
            }
            tmem_store_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&p_full[i][st & 1]));
        }
        if (ok && n_steps > 0) {
            if (!__all_sync(0xffffffffu, wait(o_done[i][(n_steps - 1) & 1], ((n_steps - 1) >> 1) & 1))) {
                if (lane == 0) fail(ERR_O_FULL);
                ok = false;
            }
            tcgen05_fence_after();
        }
        if (ok) {
            const bool shared = gridDim.z > 1;
            float* mine = a.parts + ((int64_t)blockIdx.z * a.n_tokens * a.n_heads + at / D) * (D + 4);
            const float by = shared ? (n_steps > 0 ? power2(power) : 0.f) : l == 0.f ? 0.f : power2(power) / l;
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
                const float by_half = lost >> (c >= D / 32) & 1 ? NAN : by;
                uint32_t o[16];
                if (n_steps > 0) {
                    tmem_load_16cols(o_addr + c * 16, o);
                    tmem_load_wait();
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = 0u;
                }
                if (valid)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const float4 y = make_float4(__uint_as_float(o[e]) * by_half, __uint_as_float(o[e + 1]) * by_half, __uint_as_float(o[e + 2]) * by_half,
                                                     __uint_as_float(o[e + 3]) * by_half);
                        if (shared) store4(mine + c * 16 + e, y);
                        else store4(a.out + at + c * 16 + e, y);
                    }
            }
            if (valid && shared) *reinterpret_cast<float2*>(mine + D) = make_float2(m, l);
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == kSoftmaxWarps) {
        if (*(volatile int*)&abort_flag != 0)                 // a product takes less than a microsecond
            for (int x = 0; x < 16; ++x) __nanosleep(20000);
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
    }
}

// Adds up the shares of a row of q: a warp a row.
template <int D>
__global__ void __launch_bounds__(256)
kv4_prompt_join_kernel(const float* __restrict__ parts, bf16* __restrict__ out, int64_t rows, int shares) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= rows) return;
    const auto place = [&](int z) { return parts + ((int64_t)z * rows + row) * (D + 4); };
    float top = -INFINITY, l = 0.f, o[D / 32];
    for (int z = 0; z < shares; ++z) top = fmaxf(top, place(z)[D]);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
#pragma unroll 4
    for (int z = 0; z < shares; ++z) {
        const float* p = place(z);
        const float2 ml = *reinterpret_cast<const float2*>(p + D);
        const float by = ml.x > -INFINITY ? ex2(ml.x - top) : 0.f;
        l += ml.y * by;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] += p[lane + 32 * i] * by;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) out[row * D + lane + 32 * i] = from_f32<bf16>(o[i] * inv);
}

template <int D>
int prompt(const Args& a, int n_tiles, int shares, cudaStream_t stream) {
    static bool done[kMaxDevices];
    const int status = ensure_dynamic_smem(kv4_prompt_kernel<D>, Sizes<D>::kSmem, done);
    if (status != CPM_OK) return status;
    const int64_t blocks = (int64_t)((a.tile_tokens * a.group + kRows - 1) / kRows) * a.n_kv, rows = (int64_t)a.n_tokens * a.n_heads;
    if (n_tiles > 65535 || blocks > 0x7fffffff || rows / 8 >= 0x7fffffff) return CPM_BAD_ARGUMENT;
    cpm_launch(kLaunchAttention, kv4_prompt_kernel<D>, dim3((unsigned)blocks, n_tiles, shares), kThreads, Sizes<D>::kSmem, stream, a);
    if (shares > 1)
        cpm_launch(kLaunchAttention, kv4_prompt_join_kernel<D>, dim3((unsigned)((rows + 7) / 8)), 256, 0, stream, (const float*)a.parts, a.out, rows, shares);
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

// q, out bf16 [tokens, heads, d]; the tiles are of 64 tokens, taken together up to 256 rows of a key-value head.  ``shares`` > 1: a tile's keys are shared out
// over so many blocks, whose parts (shares x tokens x heads x (d + 4) floats in ``parts``) a second kernel adds up; every token has to be in a tile then.
CPM_API int cpm_kv4_prompt(const void* q, const void* records, void* out, const int* kv_len, const int* slots, const int* page_table, int max_pages,
                           const int* cu_q, const int* tile_seq, const int* tile_row, int n_tiles, float* parts, int shares, int n_tokens, int n_heads, int n_kv,
                           int d, int window, float scale, cudaStream_t stream) {
    if (n_tiles <= 0) return CPM_OK;
    if (n_heads < 1 || n_kv < 1 || n_heads % n_kv || window < 0 || !(scale > 0.f) || shares < 1 || shares > 64 || (shares > 1 && !parts)) return CPM_BAD_ARGUMENT;
    if (((uintptr_t)records | (uintptr_t)q | (uintptr_t)out) & 15) return CPM_BAD_ARGUMENT;
    const int group = n_heads / n_kv;
    const int tile_tokens = group == 1 ? 256 : group == 2 ? 128 : 64;
    const kv4p::Args a{(const bf16*)q, (bf16*)out, (const uint8_t*)records, kv_len, slots, page_table, cu_q, tile_seq, tile_row, parts, max_pages,
                       n_heads, n_kv, group, window, tile_tokens, n_tokens, scale};
    switch (d) {
        case 64: return kv4p::prompt<64>(a, n_tiles, shares, stream);
        case 128: return kv4p::prompt<128>(a, n_tiles, shares, stream);
        default: return CPM_BAD_ARGUMENT;
    }
}
