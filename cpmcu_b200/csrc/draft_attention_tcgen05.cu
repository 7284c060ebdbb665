// Attention of a few tokens a sequence over the paged cache on the fifth-generation tensor cores (bf16; head sizes 32, 64, 96 and 128): what
// draft_attention.cu computes, with weights rounded to bf16 for their product (operands of one tcgen05.mma have one type, and values are bf16).  The difference that makes is a
// relative norm of 0.0004 to 0.0018, as in the same sums with weights rounded on the host; against 64 bits the output's rounding alone is 0.0016 to 0.0018, with it 0.0017 to 0.0019.
//
// All query heads of a key-value head and all of a sequence's tokens are rows of one matrix (row = token * group + head), cut into tiles of one or two halves of 128 rows,
// so that few tokens read every key once: 5 tokens at 16 heads are 80 rows.  S = Q K^T and O += P V are tcgen05.mma with the accumulators in tensor memory; Q, and
// a page of 64 keys and values a step, come by TMA.  A half has two S, so that the next page's scores are formed during this one's softmax, which writes P as bf16
// over the S it read.
//
// The work is a line: every (sequence, tile, key-value head) is a unit of its pages and a few more for its beginning and end, and every block takes a piece of
// equal cost of that line, so that unequal sequences leave no SM idle.  A unit that several blocks have is put together by a second kernel.
//
// What bounds it: with 256 rows a block the softmax's chains (a row a thread: 64 scores scaled, raised, added and packed a page; 64 drafted tokens of 32 heads on 2 of 128
// behind 131,071 keys take 127 to 148 us by the card's clock, 930 to 1,080 TFLOP/s; tensor pipe 61 % of the active time, issue slots 52 %, exponentials' unit 46 %).
// With few rows what surrounds the pages: 64 sequences of 6 to 8,192 keys, 5 tokens, 16 heads on 2 of 64 take 44 us, of which the keys' way from memory is 21, the line and
// the first page 5, blocks that end at 27 to 38 us, and the parts' addition the rest; 16 trees of 16 tokens behind 500 to 6,000 keys 37 us, 12 pages of 1.08 us a block
// and 8 us for the parts; one sequence of 1,000 keys 12.5 us, all of it launch, first page and parts.
//
// Of the pages that hold the step's own tokens a warp looks at the values before they are multiplied: what lies behind the keys becomes 0, and so does what is no
// finite number, which is added at the end to the rows that see it (0 times such a value would reach the others).
//
// Every wait is bounded: a block that gives up records an error, stops, waits (bounded) for its copies and products in flight, frees its tensor memory and returns.
#include "tcgen05.cuh"
#include <type_traits>

CPM_BOUNDS_TU(draft_attention_tcgen05)

namespace da5 {
using namespace tc5;

constexpr int kMostSeqs = 512;                          // of one launch
constexpr int kStages = 4;                              // pages under way
constexpr int kOdd = 8;                                 // places for marks of segments with pages: the cleaning warp is at most kStages pages, and so segments, ahead
static_assert(kOdd > kStages + 1, "a mark is read before its place is taken again");
constexpr float kBehind = 8.0f;                         // the running maximum may lie 2^8 behind
// (kExtra of 1 to 4 and kLeast of 1 to 8 differ by less than two boxes do.)
constexpr int kExtra = 2;                               // pages that a unit's beginning and end are worth
constexpr int kLeast = 4;                               // cost that a block is worth its part's addition
// Of four pairs of a row's weights one is formed by ex2_poly (2,048 pages of 256 rows a key-value head, 64 tokens at 131,071 keys: none 140 us, one 127, two 152)
constexpr int kPoly = 8;                                // a bit for each of the four

template <int D, int H>
struct Sizes {
    static constexpr int kChunks = (D + 63) / 64;       // runs of 64 channels
    static constexpr int kQHalf = 128 * 128;            // 128 rows x 128 bytes
    static constexpr int kQ = kChunks * kQHalf, kK = kChunks * 64 * 128, kV = D * 128;
    static constexpr int kQBufs = H == 1 ? 2 : 1;
    static constexpr int kSmem = H * kQBufs * kQ + kStages * (kK + kV) + 1024;
    static constexpr int kTmem = 128 * H + D * H <= 256 ? 256 : 512, kO = 128 * H;       // half i's S at 128 i and 128 i + 64, its O at 128 H + i D
    static constexpr int kThreads = 32 * (4 * H + 2 * H + 2);
    static constexpr int kBlocks = kSmem <= 100 * 1024 && H == 1 ? 2 : 1;                // an SM
    static constexpr uint32_t kIdescQK = instr_desc_bf16(128, 64), kIdescPV = instr_desc_bf16(128, D);
};

struct Args {
    bf16* out;
    const int *kv_len, *cu, *slots, *page_table;
    const int64_t* ancestors;
    const bf16* v;
    float* scratch;                                     // Cuts, then per block two places of (D + 2) x rows floats: channels, maximum, sum
    int n_slots, max_pages, n_pages, n_tokens, n_seqs, n_heads, n_kv, group, most, per_half, rows;       // per_half: tokens of a half; rows: of a place
    int parts;                                          // tiles that a sequence has at most
    float scale_log2;
};

// A unit that several blocks have: the one it begins in and the last.  Few units have a Cut each, (sequence, tile, head) by number; of many, a block has one of the
// unit that goes on behind it.
struct __align__(8) Cut { int first_block, last_block, token, rows, head, unused; };      // last_block -1: none; its first token, and rows
constexpr int kCutFloats = sizeof(Cut) / 4;
__host__ __device__ __forceinline__ bool by_unit(const Args& a, int grid) { return (int64_t)a.n_seqs * a.parts * a.n_kv <= grid; }

enum : int { ERR_Q = 1, ERR_K_FULL, ERR_V_FULL, ERR_K_EMPTY, ERR_V_EMPTY, ERR_S_FULL, ERR_P_FULL, ERR_O_DONE, ERR_V_READY };
__device__ int g_error;

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
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long ra, rb, rd;
    float2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(rb) : "f"(b.x), "f"(b.y));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(rd));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// 2^x of two numbers up to 100 without the unit that ex2 runs on, which gives 16 results a cycle and multiprocessor and which a page's weights would wait for: x = n + f with
// f in [-1/2, 1/2]; 2^f by a polynomial of degree 4 whose coefficients minimise the largest relative error, 2.6e-6 (2^-18.5; the weights enter their product with 8
// bits); 2^n by its exponent bits, which the sum with 1.5 * 2^23 + 127 leaves in its lowest ones.  From 2^-127 down the result is 0; what is no number stays none.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
    const float magic = 12582912.f + 127.f;
    x = make_float2(max_nan(x.x, -127.f), max_nan(x.y, -127.f));
    const float2 t = add2(x, make_float2(magic, magic)), n = add2(t, make_float2(-magic, -magic)), f = fma2(n, make_float2(-1.f, -1.f), x);
    float2 p = fma2(f, make_float2(0.009570101276040077f, 0.009570101276040077f), make_float2(0.05591785907745361f, 0.05591785907745361f));
    p = fma2(p, f, make_float2(0.240247443318367f, 0.240247443318367f));
    p = fma2(p, f, make_float2(0.6931217908859253f, 0.6931217908859253f));
    p = fma2(p, f, make_float2(0.9999992847442627f, 0.9999992847442627f));
    return mul2(p, make_float2(__uint_as_float(__float_as_uint(t.x) << 23), __uint_as_float(__float_as_uint(t.y) << 23)));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// ---- the line of work ----
struct Line {                                           // in shared memory
    int begin[kMostSeqs + 1];                           // cost before a sequence
    int keys[kMostSeqs], first[kMostSeqs + 1], slot[kMostSeqs];      // its keys, its first token, its row of the page table
    int warp_sum[32];
};
__device__ __forceinline__ int pages_of(int keys) { return (keys + kPageTokens - 1) / kPageTokens; }
// A sequence's row of the page table, and its keys: none where the row is none.
__device__ __forceinline__ int slot_of(const Args& a, int s) {
    const int slot = a.slots[s];
    return slot >= 0 && slot < a.n_slots ? slot : -1;
}
__device__ __forceinline__ int keys_of(const Args& a, int s, int slot) {
    const int keys = max(0, min(a.kv_len[s], a.max_pages * kPageTokens));       // (read beside the slot, not behind it)
    return slot < 0 ? 0 : keys;
}
__device__ __forceinline__ int tokens_of(const Args& a, const Line& l, int s) { return max(0, min(l.first[s + 1] - l.first[s], a.most)); }

template <int H>
__device__ __forceinline__ int units_of(const Args& a, int tokens) { return (tokens + H * a.per_half - 1) / (H * a.per_half) * a.n_kv; }

// By all threads of a block.
template <int H, int THREADS>
__device__ __forceinline__ void lay_out(const Args& a, Line& l) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (a.n_seqs <= 32) {                               // one warp's work
        if (warp == 0) {
            const bool there = lane < a.n_seqs;
            const int first = there ? max(0, min(a.cu[lane], a.n_tokens)) : 0, then = there ? max(0, min(a.cu[lane + 1], a.n_tokens)) : 0;
            const int slot = there ? slot_of(a, lane) : -1, keys = there ? keys_of(a, lane, slot) : 0;
            const int cost = there ? units_of<H>(a, max(0, min(then - first, a.most))) * (pages_of(keys) + kExtra) : 0;
            int upto = cost;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            if (there) {
                l.begin[lane] = upto - cost;
                l.first[lane] = first;
                l.keys[lane] = keys;
                l.slot[lane] = slot;
                if (lane == a.n_seqs - 1) {
                    l.begin[lane + 1] = upto;
                    l.first[lane + 1] = then;
                }
            }
        }
        __syncthreads();
        return;
    }
    for (int s = tid; s <= a.n_seqs; s += THREADS) {
        l.first[s] = max(0, min(a.cu[s], a.n_tokens));
        if (s < a.n_seqs) {
            l.slot[s] = slot_of(a, s);
            l.keys[s] = keys_of(a, s, l.slot[s]);
        }
    }
    __syncthreads();
    const int each = (a.n_seqs + THREADS - 1) / THREADS, s0 = min(a.n_seqs, tid * each), s1 = min(a.n_seqs, s0 + each);
    int sum = 0;
    for (int s = s0; s < s1; ++s) sum += units_of<H>(a, tokens_of(a, l, s)) * (pages_of(l.keys[s]) + kExtra);
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) l.warp_sum[warp] = upto;
    __syncthreads();
    int run = upto - sum;
    for (int w = 0; w < warp; ++w) run += l.warp_sum[w];
    for (int s = s0; s < s1; ++s) {
        l.begin[s] = run;
        run += units_of<H>(a, tokens_of(a, l, s)) * (pages_of(l.keys[s]) + kExtra);
    }
    if (tid == THREADS - 1) l.begin[a.n_seqs] = run;
    __syncthreads();
}
__device__ __forceinline__ int blocks_used(int total) { return max(1, min((int)gridDim.x, total / kLeast)); }
__device__ __forceinline__ int share_begin(int total, int blocks, int b) { return (int)((int64_t)total * b / blocks); }
__device__ __forceinline__ int block_of(int total, int blocks, int at) {      // the block whose piece holds it
    int b = (int)((int64_t)at * blocks / total);
    while (b + 1 < blocks && share_begin(total, blocks, b + 1) <= at) ++b;
    return b;
}

struct Segment {
    int seq, part, head, page0, pages, all_pages;       // of the unit's pages, page0 .. page0 + pages
    int tokens, row0, keys, history;                    // of the sequence; row0: the first token of the tile
    __device__ __forceinline__ bool whole() const { return pages == all_pages; }
};
// The pieces of units that lie in a block's piece of the line, one after the other; every role of the block walks them for itself.
template <int H>
struct Walk {
    int at, end, s, u;
    __device__ __forceinline__ void start(const Args& a, const Line& l, int lo, int hi) {
        at = lo;
        end = hi;
        int x = 0, y = a.n_seqs - 1;                    // the last sequence that begins at ``lo`` or before
        while (x < y) {
            const int mid = (x + y + 1) >> 1;
            if (l.begin[mid] <= lo) x = mid;
            else y = mid - 1;
        }
        s = x;
        u = lo < hi ? (lo - l.begin[s]) / (pages_of(l.keys[s]) + kExtra) : 0;
    }
    __device__ __forceinline__ bool next(const Args& a, const Line& l, Segment& g) {
        while (at < end) {
            const int n = tokens_of(a, l, s), pages = pages_of(l.keys[s]), cost = pages + kExtra, units = units_of<H>(a, n);
            if (u >= units) {
                ++s;
                u = 0;
                continue;
            }
            const int u0 = l.begin[s] + u * cost, from = max(0, at - u0 - kExtra), to = min(pages, end - u0 - kExtra);
            const bool none = pages == 0 && at == u0;   // a unit without keys is its first place's
            g = Segment{s, u / a.n_kv, u % a.n_kv, from, max(0, to - from), pages, n, u / a.n_kv * H * a.per_half, l.keys[s], l.keys[s] - n};
            ++u;
            at = u0 + cost;
            if (none || to > from) return true;
        }
        return false;
    }
};

template <int D, int H>
__global__ void __launch_bounds__(Sizes<D, H>::kThreads, Sizes<D, H>::kBlocks)
draft_attention_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                               const __grid_constant__ Args a) {
    using Z = Sizes<D, H>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ Line line;
    __shared__ __align__(8) uint64_t q_full[H][Z::kQBufs], k_full[kStages], v_full[kStages], v_ready[kStages], k_empty[kStages], v_empty[kStages], s_full[H][2], p_full[H][2],
        o_done[H][2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, odd[kOdd];               // odd: a segment's number and one (of those with pages), where its own tokens' values hold what is no finite number
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_smem = base, k_smem = q_smem + H * Z::kQBufs * Z::kQ, v_smem = k_smem + kStages * Z::kK;
    constexpr int kScoreWarp = 4 * H, kValueWarp = 5 * H, kLoadWarp = 6 * H, kCleanWarp = 6 * H + 1;
    if (threadIdx.x == 32) {
        asm volatile("prefetch.tensormap [%0];" :: "l"(&map_q) : "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" :: "l"(&map_v) : "memory");
    }
    if (threadIdx.x == 0) {
#pragma unroll 1
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&k_full[s]), 1);
            mbar_init(smem_u32(&v_full[s]), 1);
            mbar_init(smem_u32(&v_ready[s]), 1);
            mbar_init(smem_u32(&k_empty[s]), H);
            mbar_init(smem_u32(&v_empty[s]), H);
        }
#pragma unroll 1
        for (int i = 0; i < H; ++i) {
            for (int b = 0; b < Z::kQBufs; ++b) mbar_init(smem_u32(&q_full[i][b]), 1);
            for (int b = 0; b < 2; ++b) {
                mbar_init(smem_u32(&s_full[i][b]), 1);
                mbar_init(smem_u32(&p_full[i][b]), 4);
                mbar_init(smem_u32(&o_done[i][b]), 1);
            }
        }
        abort_flag = 0;
        for (int i = 0; i < kOdd; ++i) odd[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kScoreWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&tmem_slot)), "r"((uint32_t)Z::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    tcgen05_fence_before();
    lay_out<H, Z::kThreads>(a, line);                   // (ends with a barrier of the block)
    tcgen05_fence_after();
    const uint32_t tmem = tmem_slot;
    const int total = line.begin[a.n_seqs], blocks = blocks_used(total);
    const bool mine = total > 0 && (int)blockIdx.x < blocks;
    const int lo = mine ? share_begin(total, blocks, blockIdx.x) : 0, hi = mine ? share_begin(total, blocks, blockIdx.x + 1) : 0;
    float* const places = a.scratch + (int64_t)gridDim.x * kCutFloats;
    const int64_t place_floats = (int64_t)a.rows * (D + 2);

    auto fail = [&](int code) {
        atomicCAS(&g_error, 0, code);
        atomicExch(&abort_flag, 1);
    };
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
    // Up to 64 rows keep two warps busy: of two blocks on an SM the second has its rows in the tile's upper half, which other warps, on the SM's other schedulers, read
    const int shift = Z::kBlocks == 2 && a.rows <= 64 && blockIdx.x >= gridDim.x / 2 ? 64 : 0;
    Walk<H> walk;
    Segment g;
    walk.start(a, line, lo, hi);

    if (warp == kLoadWarp) {
        // ---- keys and values, a page a step ----
        int st = 0;
        bool ok = true;
#pragma unroll 1
        while (ok && walk.next(a, line, g)) {
            const int* table = a.page_table + (int64_t)line.slot[g.seq] * a.max_pages;
            int ids = 0;                                // 32 page numbers, one a lane
#pragma unroll 1
            for (int i = 0; i < g.pages; ++i, ++st) {
                if ((i & 31) == 0) ids = i + lane < g.pages ? max(0, min(CPM_PAGE(table, g.page0 + i + lane, a.max_pages), a.n_pages - 1)) : 0;
                const int page = __shfl_sync(0xffffffffu, ids, i & 31);
                const int s = st % kStages, ph = (st / kStages) & 1;
                if (!__all_sync(0xffffffffu, wait(k_empty[s], ph ^ 1))) { fail(ERR_K_EMPTY); ok = false; break; }
                if (lane == 0) {
                    mbar_expect_tx(smem_u32(&k_full[s]), Z::kK);
#pragma unroll
                    for (int c = 0; c < Z::kChunks; ++c)
                        tma_load_2d(k_smem + s * Z::kK + c * 64 * 128, &map_k, smem_u32(&k_full[s]), c * 64, (page * a.n_kv + g.head) * kPageTokens);
                }
                if (!__all_sync(0xffffffffu, wait(v_empty[s], ph ^ 1))) {
                    fail(ERR_V_EMPTY);
                    ok = false;
                    mbar_wait_bounded(smem_u32(&k_full[s]), ph);
                    break;
                }
                if (lane == 0) {
                    mbar_expect_tx(smem_u32(&v_full[s]), Z::kV);
                    tma_load_2d(v_smem + s * Z::kV, &map_v, smem_u32(&v_full[s]), 0, (page * a.n_kv + g.head) * D);
                }
                __syncwarp();
            }
        }
        // copies that nobody waits for: none is in flight at the exit
#pragma unroll 1
        for (int x = max(0, st - kStages); x < st; ++x) {
            mbar_wait_bounded(smem_u32(&k_full[x % kStages]), (x / kStages) & 1);
            mbar_wait_bounded(smem_u32(&v_full[x % kStages]), (x / kStages) & 1);
        }
    } else if (warp == kCleanWarp) {
        // ---- values of the step's own tokens and what lies behind them ----
        int st = 0, number = 0;
        bool ok = true;
#pragma unroll 1
        for (; ok && walk.next(a, line, g); number += g.pages > 0) {       // (segments without pages are not waited for)
#pragma unroll 1
            for (int i = 0; i < g.pages; ++i, ++st) {
                const int s = st % kStages, key0 = (g.page0 + i) * kPageTokens;
                if (!__all_sync(0xffffffffu, wait(v_full[s], (st / kStages) & 1))) { fail(ERR_V_FULL); ok = false; break; }
                if (key0 + kPageTokens > g.history) {
                    // a lane has the same eight keys of every channel it looks at: those that there are, and of these the step's own, by word
                    const int j0 = (lane & 7) * 8, keep = g.keys - key0 - j0, own = g.history - key0 - j0;
                    uint32_t there[4], check[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const auto from = [&](int n) { return (2 * e >= n ? 0xffffu : 0u) | (2 * e + 1 >= n ? 0xffff0000u : 0u); };
                        there[e] = ~from(keep);
                        check[e] = from(own) & there[e] & 0x80008000u;
                    }
                    bool found = false;
                    if (own < 8) {
#pragma unroll 8
                        for (int x = 0; x < D / 4; ++x) {
                            const int c = (lane >> 3) + 4 * x;
                            const uint32_t at = v_smem + s * Z::kV + c * 128 + (uint32_t)(((lane & 7) ^ (c & 7)) << 4);
                            uint32_t w[4], bad[4];
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
#pragma unroll
                            for (int e = 0; e < 4; ++e) bad[e] = ((w[e] & 0x7fff7fffu) + 0x00800080u) & check[e];      // an exponent of ones runs over into the sign's bit
                            if (bad[0] | bad[1] | bad[2] | bad[3]) {
                                found = true;
#pragma unroll
                                for (int e = 0; e < 4; ++e) w[e] &= ~((bad[e] >> 15) * 0xffffu);
                            }
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(at), "r"(w[0] & there[0]), "r"(w[1] & there[1]), "r"(w[2] & there[2]), "r"(w[3] & there[3]) : "memory");
                        }
                    }
                    if (found) odd[number % kOdd] = number + 1;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&v_ready[s]));
            }
        }
    } else if (warp >= kScoreWarp && warp < kValueWarp) {
        // ---- a half's queries and scores ----
        const int i = warp - kScoreWarp;
        int st = 0, number = 0;
        bool ok = true;
        const auto load_q = [&](const Segment& x, int n) {
            if (lane == 0) {
                const int b = n % Z::kQBufs;
                const uint32_t to = q_smem + (i * Z::kQBufs + b) * Z::kQ + shift * 128;
                mbar_expect_tx(smem_u32(&q_full[i][b]), Z::kChunks * a.per_half * a.group * 128);
#pragma unroll
                for (int c = 0; c < Z::kChunks; ++c)
                    tma_load_3d(to + c * Z::kQHalf, &map_q, smem_u32(&q_full[i][b]), c * 64, x.head * a.group, line.first[x.seq] + x.row0 + i * a.per_half);
            }
        };
        Segment ahead;
        bool more = walk.next(a, line, g);
        if (more) load_q(g, 0);
        int requested = more ? 1 : 0;
#pragma unroll 1
        while (ok && more) {
            const bool then = walk.next(a, line, ahead);
            if (Z::kQBufs == 2 && then) {               // (the other buffer's products are done: this half's last scores before this segment)
                if (st > 0 && !__all_sync(0xffffffffu, wait(s_full[i][(st - 1) & 1], ((st - 1) >> 1) & 1))) { fail(ERR_S_FULL); break; }
                load_q(ahead, number + 1);
                ++requested;
            }
            if (!__all_sync(0xffffffffu, wait(q_full[i][number % Z::kQBufs], (number / Z::kQBufs) & 1))) { fail(ERR_Q); break; }
            const uint32_t q_at = q_smem + (i * Z::kQBufs + number % Z::kQBufs) * Z::kQ;
#pragma unroll 1
            for (int k0 = 0; k0 < g.pages; ++k0, ++st) {
                const int s = st % kStages;
                if (!__all_sync(0xffffffffu, wait(k_full[s], (st / kStages) & 1))) { fail(ERR_K_FULL); ok = false; break; }
                if (st >= 2 && !__all_sync(0xffffffffu, wait(o_done[i][st & 1], ((st - 2) >> 1) & 1))) { fail(ERR_O_DONE); ok = false; break; }
                tcgen05_fence_after();
                if (elect_one()) {
                    const uint32_t to = tmem + i * 128 + (st & 1) * 64;
#pragma unroll
                    for (int c = 0; c < Z::kChunks; ++c) {
                        const uint64_t da = smem_desc_sw128(q_at + c * Z::kQHalf), db = smem_desc_sw128(k_smem + s * Z::kK + c * 64 * 128);
#pragma unroll
                        for (int k = 0; k < (D - c * 64 < 64 ? (D - c * 64) / 16 : 4); ++k) tcgen05_mma_f16(to, da + 2 * k, db + 2 * k, Z::kIdescQK, (c | k) != 0);
                    }
                    tcgen05_commit(smem_u32(&s_full[i][st & 1]));
                    tcgen05_commit(smem_u32(&k_empty[s]));
                }
                __syncwarp();
            }
            if (!ok) break;
            if (Z::kQBufs == 1 && then) {
                if (st > 0 && !__all_sync(0xffffffffu, wait(s_full[i][(st - 1) & 1], ((st - 1) >> 1) & 1))) { fail(ERR_S_FULL); break; }
                load_q(ahead, number + 1);
                ++requested;
            }
            g = ahead;
            more = then;
            ++number;
        }
#pragma unroll 1
        for (int x = max(0, requested - Z::kQBufs); x < requested; ++x) mbar_wait_bounded(smem_u32(&q_full[i][x % Z::kQBufs]), (x / Z::kQBufs) & 1);
    } else if (warp >= kValueWarp && warp < kLoadWarp) {
        // ---- a half's weighted values ----
        const int i = warp - kValueWarp;
        int st = 0;
        bool ok = true;
#pragma unroll 1
        while (ok && walk.next(a, line, g)) {
#pragma unroll 1
            for (int k0 = 0; k0 < g.pages; ++k0, ++st) {
                const int s = st % kStages;
                if (!__all_sync(0xffffffffu, wait(v_ready[s], (st / kStages) & 1))) { fail(ERR_V_READY); ok = false; break; }
                if (!__all_sync(0xffffffffu, wait(p_full[i][st & 1], (st >> 1) & 1))) { fail(ERR_P_FULL); ok = false; break; }
                tcgen05_fence_after();
                if (elect_one()) {
                    const uint64_t db = smem_desc_sw128(v_smem + s * Z::kV);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tcgen05_mma_f16_ts(tmem + Z::kO + i * D, tmem + i * 128 + (st & 1) * 64 + k * 8, db + 2 * k, Z::kIdescPV, k0 > 0 || k != 0);
                    tcgen05_commit(smem_u32(&o_done[i][st & 1]));
                    tcgen05_commit(smem_u32(&v_empty[s]));
                }
                __syncwarp();
            }
        }
    } else if (warp < 4 * H) {
        // ---- softmax and output: a thread to a row ----
        const int i = warp >> 2, r = (int)(threadIdx.x & 127) - shift;       // the row of its half; below 0: none
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t o_addr = lanes + Z::kO + i * D;
        int st = 0, number = 0;
        bool ok = true;
#pragma unroll 1
        for (; ok && walk.next(a, line, g); number += g.pages > 0) {
            const int in_half = r / a.group, token = g.row0 + i * a.per_half + in_half;
            const bool valid = r >= 0 && in_half < a.per_half && token < g.tokens;
            const bool any = __any_sync(0xffffffffu, valid);
            uint64_t word = 0;                           // the step's tokens that the row sees
            if (valid) {
                word = a.ancestors ? (uint64_t)a.ancestors[line.first[g.seq] + token] : ~0ull >> (63 - token);
                word &= ~0ull >> (64 - g.tokens);
            }
            float m = -INFINITY, l = 0.f;
#pragma unroll 1
            for (int k0 = 0; k0 < g.pages; ++k0, ++st) {
                if (!__all_sync(0xffffffffu, wait(s_full[i][st & 1], (st >> 1) & 1))) {
                    fail(ERR_S_FULL);
                    ok = false;
                    break;
                }
                tcgen05_fence_after();
                if (any) {
                    const uint32_t s_addr = lanes + i * 128 + (st & 1) * 64;
                    const int before = g.history - (g.page0 + k0) * kPageTokens;       // keys of the page that every row sees
                    uint32_t v[2][32];
                    tmem_load_32cols(s_addr, v[0]);
                    tmem_load_32cols(s_addr + 32, v[1]);
                    tmem_load_wait();
                    if (before < kPageTokens) {
                        const uint64_t sees = before > 0 ? word << before | (~0ull >> (64 - before)) : before > -64 ? word >> -before : 0;
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const uint32_t bits = (uint32_t)(sees >> (32 * c));
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!(bits >> e & 1)) v[c][e] = 0xff800000u;
                        }
                    }
                    float most[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        most[c] = -INFINITY;
#pragma unroll
                        for (int e = 0; e < 16; e += 2) most[c] = max3(most[c], __uint_as_float(v[c / 2][16 * (c & 1) + e]), __uint_as_float(v[c / 2][16 * (c & 1) + e + 1]));
                    }
                    const float m_new = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * a.scale_log2;
                    const bool grow = m_new > m + kBehind || (m == -INFINITY && m_new > -INFINITY);
                    if (__any_sync(0xffffffffu, grow)) {
                        const float alpha = grow ? ex2(m - m_new) : 1.f;        // 0 the first time
                        l *= alpha;
                        if (k0 > 0) {
                            // the products of the page before have to be in O
                            if (!__all_sync(0xffffffffu, wait(o_done[i][(st - 1) & 1], ((st - 1) >> 1) & 1))) {
                                fail(ERR_O_DONE);
                                ok = false;
                                break;
                            }
                            tcgen05_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D / 16; ++c) {
                                uint32_t o[16];
                                tmem_load_16cols(o_addr + c * 16, o);
                                tmem_load_wait();
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                                tmem_store_16cols(o_addr + c * 16, o);
                            }
                        }
                        if (grow) m = m_new;
                    }
                    const float use = m == -INFINITY ? 0.f : m;
                    const float2 by = make_float2(a.scale_log2, a.scale_log2), less = make_float2(-use, -use);
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t packed[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float2 x = fma2(make_float2(__uint_as_float(v[c][2 * e]), __uint_as_float(v[c][2 * e + 1])), by, less);
                            const float2 w = (kPoly >> (e & 3) & 1) ? ex2_poly(x) : make_float2(ex2(x.x), ex2(x.y));
                            sum[e & 1] = add2(sum[e & 1], w);
                            packed[e] = pack_bf16(w.x, w.y);
                        }
                        tmem_store_16cols(s_addr + 16 * c, packed);
                    }
                    const float2 both = add2(sum[0], sum[1]);
                    l += both.x + both.y;
                    tmem_store_wait();
                }
                tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[i][st & 1]));
            }
            if (!ok) break;
            // ---- the segment's output, or its part of it ----
            if (g.pages > 0) {
                if (!__all_sync(0xffffffffu, wait(o_done[i][(st - 1) & 1], ((st - 1) >> 1) & 1))) {
                    fail(ERR_O_DONE);
                    break;
                }
                tcgen05_fence_after();
            }
            if (any) {
                const bool whole = g.whole();
                const int64_t at = ((int64_t)(line.first[g.seq] + token) * a.n_heads + g.head * a.group + r % a.group) * D;
                // a part of a unit that an earlier block began lies in the block's first place, one that goes on behind it in the second
                float* const to = places + (2 * (int64_t)blockIdx.x + (g.page0 == 0)) * place_floats + i * a.per_half * a.group + r;
                const bool fix = g.pages > 0 && odd[number % kOdd] == number + 1;
                const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    if (g.pages > 0) {
                        tmem_load_32cols(o_addr + c * 32, o);
                        tmem_load_wait();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0u;
                    }
                    if (!valid) continue;
                    if (fix) {
                        // values that are no finite numbers, to the row that sees them
#pragma unroll 1
                        for (int j = 0; j < g.tokens; ++j) {
                            const int key = g.history + j;
                            if (!(word >> j & 1) || key < g.page0 * kPageTokens || key >= (g.page0 + g.pages) * kPageTokens) continue;
                            const int* table = a.page_table + (int64_t)line.slot[g.seq] * a.max_pages;
                            const int64_t page = max(0, min(CPM_PAGE(table, key / kPageTokens, a.max_pages), a.n_pages - 1));
                            const bf16* from = a.v + value_offset((int)page, g.head, c * 32, key % kPageTokens, a.n_kv, D);
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float x = __bfloat162float(from[e * kPageTokens]);
                                if (!(fabsf(x) < INFINITY)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
                            }
                        }
                    }
                    if (whole) {
                        uint4 y[4];
                        uint32_t* w = reinterpret_cast<uint32_t*>(y);
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float lo_ = __uint_as_float(o[2 * e]), hi_ = __uint_as_float(o[2 * e + 1]);
                            w[e] = pack_bf16(l == 0.f ? lo_ : lo_ * inv, l == 0.f ? hi_ : hi_ * inv);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) *reinterpret_cast<uint4*>(a.out + at + c * 32 + 8 * e) = y[e];
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) to[(c * 32 + e) * a.rows] = __uint_as_float(o[e]);      // (neighbouring rows side by side)
                    }
                }
                if (valid && !whole) {
                    to[D * a.rows] = m;
                    to[(D + 1) * a.rows] = l;
                }
            }
            tcgen05_fence_before();                      // (the next segment's products come behind this warp's next P)
        }
    }
    // ---- the units that begin here, for the kernel that adds up parts ----
    if (warp == kCleanWarp && lane == 0) {
        Cut* const cuts = reinterpret_cast<Cut*>(a.scratch);
        const bool each = by_unit(a, gridDim.x);
        Cut last{(int)blockIdx.x, -1, 0, 0, 0, 0};
        Walk<H> again;
        Segment x;
        again.start(a, line, lo, hi);
        while (again.next(a, line, x)) {
            if (x.page0 > 0) continue;
            const int u = x.part * a.n_kv + x.head;
            const Cut cut{(int)blockIdx.x, x.whole() ? -1 : block_of(total, blocks, line.begin[x.seq] + (u + 1) * (x.all_pages + kExtra) - 1),
                          line.first[x.seq] + x.row0, min(H * a.per_half, x.tokens - x.row0) * a.group, x.head, 0};
            if (each) cuts[(x.seq * a.parts + x.part) * a.n_kv + x.head] = cut;
            else if (cut.last_block >= 0) last = cut;
        }
        if (!each) cuts[blockIdx.x] = last;
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == kScoreWarp) {
        if (*(volatile int*)&abort_flag != 0)            // a product takes less than a microsecond
            for (int x = 0; x < 16; ++x) __nanosleep(20000);
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"((uint32_t)Z::kTmem) : "memory");
    }
}

// Adds up the parts of the units that were cut.  A block has 32 rows of one unit and all or (few units) an eighth of the channels; a warp has an eighth of the channels
// and every second or sixteenth part, a lane a row.
constexpr int kJoinWarps = 16, kEighths = 8;
template <int D, int H>
__global__ void __launch_bounds__(32 * kJoinWarps, 2)
draft_join_tcgen05_kernel(const __grid_constant__ Args a, int grid, int eighths) {       // eighths: of the channels a block has, 1 or 8
    constexpr int C = D / kEighths;
    __shared__ float tops[kJoinWarps][32], sums[kJoinWarps][32], values[kJoinWarps][C][33], weight[kJoinWarps][32];
    __shared__ bf16* to[32];                            // where a row's channels go
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pieces = kEighths / eighths, groups = kJoinWarps / eighths;
    const int r0 = blockIdx.x / pieces * 32, first_eighth = blockIdx.x % pieces * eighths, eighth = first_eighth + warp % eighths, group = warp / eighths;
    const Cut cut = reinterpret_cast<const Cut*>(a.scratch)[blockIdx.y];
    if (by_unit(a, grid)) {                             // (a unit that is none has no Cut)
        const int s = blockIdx.y / (a.parts * a.n_kv), part = blockIdx.y / a.n_kv % a.parts;
        const int first = max(0, min(a.cu[s], a.n_tokens)), n = min(max(0, min(a.cu[s + 1], a.n_tokens) - first), a.most);
        if (part * H * a.per_half >= n) return;
    }
    if (cut.last_block < 0 || r0 >= cut.rows) return;
    const int b0 = cut.first_block, row = min(r0 + lane, cut.rows - 1);
    const float* places = a.scratch + (int64_t)grid * kCutFloats;
    const int64_t place_floats = (int64_t)a.rows * (D + 2);
    float top = -INFINITY, l = 0.f, o[C];
#pragma unroll
    for (int i = 0; i < C; ++i) o[i] = 0.f;
#pragma unroll 2
    for (int b = b0 + group; b <= cut.last_block; b += groups) {
        const float* p = places + (2 * (int64_t)b + (b == b0)) * place_floats + row;
        float v[C];
#pragma unroll
        for (int i = 0; i < C; ++i) v[i] = p[(eighth * C + i) * a.rows];
        const float m = p[D * a.rows], sum = p[(D + 1) * a.rows], now = fmaxf(top, m), use = now == -INFINITY ? 0.f : now, back = ex2(top - use), by = ex2(m - use);
        l = l * back + sum * by;
#pragma unroll
        for (int i = 0; i < C; ++i) o[i] = o[i] * back + v[i] * by;
        top = now;
    }
    tops[warp][lane] = top;
    sums[warp][lane] = l;
#pragma unroll
    for (int i = 0; i < C; ++i) values[warp][i][lane] = o[i];
    __syncthreads();
    // the groups' weights of every row (those of the warps with the block's first eighth stand for their groups)
    const int many = min(groups, cut.last_block - b0 + 1);
    if (warp == 1) to[lane] = a.out + ((int64_t)(cut.token + row / a.group) * a.n_heads + cut.head * a.group + row % a.group) * D + first_eighth * C;
    if (warp == 0) {
        float high = -INFINITY, all = 0.f;
        for (int g = 0; g < many; ++g) high = fmaxf(high, tops[g * eighths][lane]);
        const float use = high == -INFINITY ? 0.f : high;
        for (int g = 0; g < many; ++g) all += sums[g * eighths][lane] * ex2(tops[g * eighths][lane] - use);
        const float inv = all == 0.f ? 1.f : 1.f / all;
        for (int g = 0; g < many; ++g) weight[g][lane] = ex2(tops[g * eighths][lane] - use) * inv;
    }
    __syncthreads();
    // neighbouring lanes finish neighbouring channels of a row
    const auto finish = [&](auto all_of_them) {
        constexpr int N = decltype(all_of_them)::value ? kEighths : 1;       // eighths, in a block of which a row has N * C neighbours
#pragma unroll 4
        for (int x = threadIdx.x; x < 32 * N * C; x += 32 * kJoinWarps) {
            const int r = x / (N * C), c = x % (N * C);
            if (r0 + r >= cut.rows) break;
            float y = 0.f;
            for (int g = 0; g < many; ++g) y += values[g * N + c / C][c % C][r] * weight[g][r];
            to[r][c] = from_f32<bf16>(y);
        }
    };
    if (eighths == 1) finish(std::false_type{});
    else finish(std::true_type{});
}

template <int D, int H>
int attend(const void* q, const void* k, Args a, cudaStream_t stream) {
    using Z = Sizes<D, H>;
    static bool done[kMaxDevices];
    const int status = ensure_dynamic_smem(draft_attention_tcgen05_kernel<D, H>, Z::kSmem, done);
    if (status != CPM_OK) return status;
    const int sms = device_sms();
    if (sms <= 0) return CPM_BAD_ARGUMENT;
    CUtensorMap map_q, map_k, map_v;
    const uint64_t rows = (uint64_t)a.n_pages * a.n_kv;
    if (!make_map_3d_bf16(&map_q, q, D, a.n_heads, a.n_tokens, D * 2, (uint64_t)a.n_heads * D * 2, 64, a.group, a.per_half) ||
        !make_map_2d_bf16(&map_k, k, rows * kPageTokens, D, D * 2, 64, kPageTokens) || !make_map_2d_bf16(&map_v, a.v, rows * D, kPageTokens, kPageTokens * 2, 64, D))
        return CPM_BAD_ARGUMENT;
    const int grid = sms * Z::kBlocks;
    const Args all = a;
    for (int first = 0; first < all.n_seqs; first += kMostSeqs) {
        a.n_seqs = min(kMostSeqs, all.n_seqs - first);
        a.kv_len = all.kv_len + first;
        a.cu = all.cu + first;
        a.slots = all.slots + first;
        cpm_launch(kLaunchAttention, draft_attention_tcgen05_kernel<D, H>, dim3(grid), Z::kThreads, Z::kSmem, stream, map_q, map_k, map_v, a);
        const int units = by_unit(a, grid) ? a.n_seqs * a.parts * a.n_kv : grid, tiles = (a.rows + 31) / 32, eighths = units * tiles * 2 <= sms ? 1 : kEighths;
        cpm_launch(kLaunchAttention, draft_join_tcgen05_kernel<D, H>, dim3(tiles * (kEighths / eighths), units), 32 * kJoinWarps, 0, stream, a, grid, eighths);
    }
    return launch_status();
}

// Tokens of a half, halves of a tile, and rows of a place in the scratch.
struct Shape { int per_half, halves, rows; };
Shape shape_of(int group, int most) {
    const int fit = 128 / group, halves = most > fit ? 2 : 1, per_half = min(fit, most);
    return Shape{per_half, halves, min(halves * per_half, most) * group};
}
int blocks_per_sm(int d, int halves) {
    if (halves == 2) return 1;
    return d == 32 ? Sizes<32, 1>::kBlocks : d == 64 ? Sizes<64, 1>::kBlocks : d == 96 ? Sizes<96, 1>::kBlocks : Sizes<128, 1>::kBlocks;
}

}  // namespace da5

// Reads and clears the error that a kernel recorded (0: none).
CPM_API int cpm_draft_attention_error() {
    int code = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&code, da5::g_error, sizeof(int)) != cudaSuccess) return -1;
    if (code) cudaMemcpyToSymbol(da5::g_error, &zero, sizeof(int));
    return code;
}

// 32-bit floats that a launch needs for the parts of units that are cut.
CPM_API int64_t cpm_draft_attention_scratch_floats(int n_heads, int n_kv, int d, int most) {
    if (n_kv < 1 || n_heads < n_kv || n_heads / n_kv > 128) return 0;
    const da5::Shape s = da5::shape_of(n_heads / n_kv, most);
    return (int64_t)device_sms() * da5::blocks_per_sm(d, s.halves) * (da5::kCutFloats + 2 * (int64_t)s.rows * (d + 2));
}

CPM_API int cpm_draft_attention_tcgen05(const void* q, const void* k, const void* v, void* out, const int* kv_len, const int* cu, const int* slots,
                                        const int* page_table, int n_slots, int max_pages, int n_pages, const int64_t* ancestors, float* scratch, int n_tokens, int n_seqs,
                                        int most, int n_heads, int n_kv, int d, float scale, cudaStream_t stream) {
    if (n_tokens <= 0 || n_seqs <= 0) return CPM_OK;
    if (n_kv < 1 || n_heads < 1 || n_heads % n_kv || n_heads / n_kv > 128 || most < 1 || most > 64 || max_pages < 1 || n_pages < 1 || !(scale > 0.f) || !scratch) return CPM_BAD_ARGUMENT;
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)scratch) & 15) return CPM_BAD_ARGUMENT;
    // the line's cost and a page's first row are counted in 32 bits
    const da5::Shape s = da5::shape_of(n_heads / n_kv, most);
    const int64_t units = (int64_t)((most + s.halves * s.per_half - 1) / (s.halves * s.per_half)) * n_kv;
    if (units * (max_pages + da5::kExtra) * min(n_seqs, da5::kMostSeqs) > 0x7fffffff || (int64_t)n_pages * n_kv * max(d, kPageTokens) > 0x7fffffff ||
        max_pages > 0x7fffffff / kPageTokens)
        return CPM_BAD_ARGUMENT;
    const da5::Args a{(bf16*)out, kv_len, cu, slots, page_table, ancestors, (const bf16*)v, scratch, n_slots, max_pages, n_pages, n_tokens, n_seqs, n_heads, n_kv,
                      n_heads / n_kv, most, s.per_half, s.rows, (most + s.halves * s.per_half - 1) / (s.halves * s.per_half),
                      scale * 1.4426950408889634f};
    const bool two = s.halves == 2;
    switch (d) {
        case 32: return two ? da5::attend<32, 2>(q, k, a, stream) : da5::attend<32, 1>(q, k, a, stream);
        case 64: return two ? da5::attend<64, 2>(q, k, a, stream) : da5::attend<64, 1>(q, k, a, stream);
        case 96: return two ? da5::attend<96, 2>(q, k, a, stream) : da5::attend<96, 1>(q, k, a, stream);
        case 128: return two ? da5::attend<128, 2>(q, k, a, stream) : da5::attend<128, 1>(q, k, a, stream);
        default: return CPM_BAD_ARGUMENT;
    }
}
