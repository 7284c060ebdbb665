// Attention over a cache held in 4 bits:  o = sum_j p_j v_j,  p = softmax(q . k_j * scale)  over the keys a query sees.
//
// The codes are small whole numbers, which fp16 holds exactly, so that both products run on the tensor cores (mma.m16n8k16, fp16
// in, fp32 sums) without rounding a key or a value: with s and m a half row's scale and middle,
//     q . k  = sum over halves of  s_k (q_h . (c - 8)) + m_k sum(q_h)
//     o      = sum over halves of  (p s_v) (c - 8)      + p m_v
// Keys and values are the operand with 16 rows, a tile of 8 * NT queries (query heads of one key-value head, of one or several tokens) the
// one with 8 columns.  A query is divided by a power of two first, which makes it an fp16 number without loss; p s_v is kept between
// 2^-14 and 2^15 in the same way.  bf16 queries: p s_v is rounded to fp16 (11 bits; the output has 8).  fp32 queries: q and p s_v are sums of
// two fp16 numbers (22 bits), which costs a second product each.
//
// A block takes an equal share of all (tile, key-value head, page) units of the launch, in that order, so that a batch of unequal
// sequences leaves no SM idle; a tile that is cut leaves its parts (maximum, sum, weighted values) to a second kernel.  One warp
// brings whole records (a page of one head, 9,216 bytes at d = 128) into shared memory by bulk copies; four warps take 16 tokens of each
// record and keep a softmax of their own, so that nothing synchronises them but the arrival of records.
#include "kv4.cuh"
#include "tcgen05.cuh"

CPM_BOUNDS_TU(kv4_attention)

namespace {

using namespace tc5;

constexpr int kWarps = 4;                              // warps that compute; one more brings the records
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kTileTokens = 64;                        // tokens of a prompt's query tile
constexpr int kMostTiles = 2048;                       // tiles of one launch (their prefix sums lie in shared memory)

__device__ int g_kv4_error;                            // 1: a wait for a record gave up

struct AttendArgs {
    const void* q;
    void* out;
    const uint8_t* records;
    const int *kv_len, *slots, *page_table;
    const int *cu_q, *tile_seq, *tile_row;             // null: one token per sequence
    float* scratch;
    int max_pages, n_tiles, n_heads, n_kv, group, window;
    float scale;
};

// One query tile: its sequence's first query row, tokens, keys, and the pages that any of its queries sees.
struct Tile { int row, tokens, first_pos, kv_len, page0, pages, slot, parts; };

__device__ __forceinline__ Tile tile_of(const AttendArgs& a, int i, int columns) {
    Tile t;
    const int seq = a.tile_seq ? a.tile_seq[i] : i;
    t.kv_len = a.kv_len[seq];
    t.slot = a.slots[seq];
    int q_len = 1, off = 0, base = i;
    if (a.cu_q) {
        base = a.cu_q[seq];
        q_len = a.cu_q[seq + 1] - base;
        off = a.tile_row[i];
    }
    t.row = base + off;
    t.tokens = max(0, min(a.cu_q ? kTileTokens : 1, q_len - off));
    t.first_pos = t.kv_len - q_len + off;              // position of the tile's first token; keys up to its own are seen
    const int keys = min(t.kv_len, t.first_pos + t.tokens);
    t.page0 = a.window ? max(0, t.first_pos - a.window + 1) / kPageTokens : 0;
    t.pages = max(0, (keys + kPageTokens - 1) / kPageTokens - t.page0);
    t.parts = (t.tokens * a.group + columns - 1) / columns;
    return t;
}
// Units of a tile: pages (one where there is none, for the zeros that such a row gets) times parts and key-value heads.
__device__ __forceinline__ int tile_units(const Tile& t, int n_kv) { return max(1, t.pages) * t.parts * n_kv; }

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Waits for a record, with a limit; where a wait has given up before, shortly (for what may still be under way into shared memory).
__device__ __forceinline__ bool wait_record(uint32_t bar, uint32_t parity, bool alive) {
    const uint32_t limit = alive ? kSpinLimit : 4096u;
    for (uint32_t i = 0; i < limit; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    return false;
}

// The eight codes of a word as fp16 numbers c - 8: nibbles 0 and 4, 1 and 5, 2 and 6, 3 and 7.  A nibble put into the low bits of 1024
// gives 1024 + c, one four bits higher 1024 + 16 c; both steps back to c - 8 are exact.
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t (&r)[4]) {
    const __half2 low = __floats2half2_rn(-1032.f, -1032.f), sixteenth = __floats2half2_rn(0.0625f, 0.0625f), high = __floats2half2_rn(-72.f, -72.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t v = w >> (8 * i);
        uint32_t a, b;
        asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(a) : "r"(v));
        asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(b) : "r"(v));
        const __half2 x = __hadd2(*reinterpret_cast<__half2*>(&a), low);
        const __half2 y = __hfma2(*reinterpret_cast<__half2*>(&b), sixteenth, high);
        r[2 * i] = *reinterpret_cast<const uint32_t*>(&x);
        r[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
    }
}
// A lane's words of 16 tokens: word[pair][upper].
template <int D>
__device__ __forceinline__ void load_words(const uint8_t* codes, int slice, int lane, uint32_t (&w)[D / 32][2]) {
    using L = Kv4<D>;
    const uint8_t* p = codes + L::word(slice, 0, lane, 0);
    if constexpr (L::kRun == 2) {
#pragma unroll
        for (int v = 0; v < D / 64; ++v) {
            const uint4 x = *reinterpret_cast<const uint4*>(p + v * 512);
            w[2 * v][0] = x.x; w[2 * v][1] = x.y; w[2 * v + 1][0] = x.z; w[2 * v + 1][1] = x.w;
        }
    } else {
#pragma unroll
        for (int v = 0; v < D / 32; ++v) {
            const uint2 x = *reinterpret_cast<const uint2*>(p + v * 256);
            w[v][0] = x.x; w[v][1] = x.y;
        }
    }
}

// Power of two by which a number is divided so that it lies in [1024, 2048): its exponent less 10, kept where 2^e and 2^-e are finite.
__device__ __forceinline__ int shift_of(float most) {
    const int e = (int)((__float_as_uint(most) >> 23) & 255u) - 127 - 10;
    return most > 0.f && most < INFINITY ? max(-120, min(120, e)) : 0;
}
constexpr int kNoShift = -1000;                        // no value has been seen yet
__device__ __forceinline__ float power2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <int D, int NT, int TERMS>
struct Smem {
    static constexpr int kStages = D >= 96 ? 5 : 8;
    static constexpr int kCols = 8 * NT;
    static constexpr int kQStride = D + 16;            // fp16 numbers a row: rows 32 bytes apart modulo 128
    alignas(128) uint8_t records[kStages][Kv4<D>::kBytes];
    alignas(16) __half q[TERMS][kCols][kQStride];
    alignas(16) float merge[kWarps / 2][kCols][D + 4];
    float merge_m[kWarps][kCols], merge_l[kWarps][kCols];
    float q_sum[kCols][2], factor[kCols];
    int last[kCols];                                   // a column's last key, -1: no such column
    alignas(8) uint64_t full[kStages], empty[kStages];
    int scan[kThreads / 32 + 1];
    int prefix[kMostTiles + 1];
};

// Blocks that take a share: each of them at least two units, since every further part costs the second kernel a read.
__device__ __forceinline__ int sharing_blocks(int64_t units, int blocks) {
    return (int)min((int64_t)blocks, max((int64_t)1, units / 2));
}
__device__ __forceinline__ int64_t share_begin(int64_t units, int sharing, int block) { return units * block / sharing; }
__device__ __forceinline__ int block_of(int64_t unit, int64_t units, int sharing) { return (int)(((unit + 1) * sharing - 1) / units); }

// Prefix sums of the tiles' units; every thread of the block takes part.
__device__ __forceinline__ void sum_tiles(const AttendArgs& a, int columns, int* prefix, int* scan) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int carry = 0;
    for (int i0 = 0; i0 < a.n_tiles; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        const int own = i < a.n_tiles ? tile_units(tile_of(a, i, columns), a.n_kv) : 0;
        int v = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += x;
        }
        if (lane == 31) scan[warp] = v;
        __syncthreads();
        int before = carry, all = carry;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) before += scan[w];
            all += scan[w];
        }
        if (i < a.n_tiles) prefix[i] = before + v - own;
        carry = all;
        __syncthreads();
    }
    if (threadIdx.x == 0) prefix[a.n_tiles] = carry;
    __syncthreads();
}
__device__ __forceinline__ int find_tile(const int* prefix, int n, int unit) {
    int lo = 0, hi = n;                                 // the last tile that begins at or before the unit (empty tiles begin where the next does)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= unit) lo = mid; else hi = mid;
    }
    return lo;
}

// Blocks that an SM has room for: what the registers allow (207 of a thread at d = 128 and 16 columns, 255 for fp32).
constexpr int blocks_per_sm(int d, int nt, int terms) { return nt == 1 ? 3 : terms == 2 && d > 32 ? 1 : 2; }
constexpr int kMostBlocksPerSm = 3;

template <int D> constexpr int64_t part_floats(int columns) { return (int64_t)columns * (D + 2); }

template <typename T, int D, int NT, int TERMS>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(D, NT, TERMS))
kv4_attention_kernel(const __grid_constant__ AttendArgs a) {
    using L = Kv4<D>;
    using S = Smem<D, NT, TERMS>;
    constexpr int COLS = S::kCols, STEPS = D / 16, E = D / 32;
    extern __shared__ uint8_t raw[];
    S& sm = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(raw) + 127) & ~(uintptr_t)127);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            mbar_init(smem_u32(&sm.full[i]), 1);
            mbar_init(smem_u32(&sm.empty[i]), kWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_launch_dependents();
    pdl_wait();
    sum_tiles(a, COLS, sm.prefix, sm.scan);
    const int64_t units = sm.prefix[a.n_tiles];
    const int sharing = sharing_blocks(units, gridDim.x);
    if ((int)blockIdx.x >= sharing || units == 0) return;
    const int64_t begin = share_begin(units, sharing, blockIdx.x), end = share_begin(units, sharing, blockIdx.x + 1);
    int64_t unit = begin;
    int index = find_tile(sm.prefix, a.n_tiles, (int)unit);

    if (warp == kWarps) {
        // ---- the warp that brings records ----
        bool alive = true;
        int it = 0;
        while (unit < end) {
            while (sm.prefix[index + 1] <= unit) ++index;
            const Tile t = tile_of(a, index, COLS);
            const int pages = max(1, t.pages);
            const int at = (int)unit - sm.prefix[index];
            int page = at % pages;
            const int head = (at / pages) % a.n_kv;
            const int stop = (int)min((int64_t)pages, page + (end - unit));
            unit += stop - page;
            const int* table = a.page_table + (int64_t)t.slot * a.max_pages;
            for (; page < stop; page += 32) {
                const int n = min(32, stop - page);
                const int mine = lane < n && t.pages > 0 ? CPM_PAGE(table, t.page0 + page + lane, a.max_pages) : 0;
                for (int i = 0; i < n; ++i, ++it) {
                    const int number = __shfl_sync(0xffffffffu, mine, i);
                    const int stage = it % S::kStages;
                    if (it >= S::kStages && alive)
                        alive = mbar_wait_bounded(smem_u32(&sm.empty[stage]), ((it / S::kStages) & 1) ^ 1);
                    if (lane == 0) {
                        const uint32_t bar = smem_u32(&sm.full[stage]);
                        if (t.pages > 0 && alive) {
                            mbar_expect_tx(bar, L::kBytes);
                            bulk_load(smem_u32(sm.records[stage]), a.records + ((int64_t)number * a.n_kv + head) * L::kBytes, L::kBytes, bar);
                        } else {
                            mbar_arrive(bar);            // a row without keys: nothing to bring
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (!alive && lane == 0) atomicExch(&g_kv4_error, 1);
        return;
    }

    // ---- the warps that compute ----
    const int g = lane >> 2, j = lane & 3;
    bool alive = true;
    int it = 0;
    while (unit < end) {
        while (sm.prefix[index + 1] <= unit) ++index;
        const Tile t = tile_of(a, index, COLS);
        const int pages = max(1, t.pages);
        const int at = (int)unit - sm.prefix[index];
        const int first_page = at % pages, head = (at / pages) % a.n_kv, part = at / pages / a.n_kv;
        const int stop = (int)min((int64_t)pages, first_page + (end - unit));
        const int columns = min(COLS, t.tokens * a.group - part * COLS);

        // queries of the tile: divided by a power of two, in fp16 (TERMS = 2: and what that leaves)
        for (int c = warp; c < COLS; c += kWarps) {
            float x[E];
            const int n = part * COLS + c;
            const int64_t row = ((int64_t)(t.row + n / a.group) * a.n_heads + head * a.group + n % a.group) * D;
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                x[i] = c < columns ? to_f32(reinterpret_cast<const T*>(a.q)[row + lane * E + i]) : 0.f;
                most = fmaxf(most, fabsf(x[i]));
            }
            const int e = shift_of(warp_max(most));
            const float down = power2(-e);
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float y = x[i] * down;
                sum += y;
                const __half h = __float2half_rn(y);
                sm.q[0][c][lane * E + i] = h;
                if constexpr (TERMS == 2) sm.q[1][c][lane * E + i] = __float2half_rn(y - __half2float(h));
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if ((lane & 15) == 0) sm.q_sum[c][lane >> 4] = sum;
            if (lane == 0) {
                sm.factor[c] = power2(e) * a.scale * 1.4426950408889634f;
                sm.last[c] = c < columns ? t.first_pos + n / a.group : -1;
            }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        uint32_t qf[TERMS][STEPS][NT][2];
        float qs[NT][2][2], factor[NT][2];
        int last[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
#pragma unroll
                for (int u = 0; u < TERMS; ++u) {
                    const uint2 v = *reinterpret_cast<const uint2*>(&sm.q[u][8 * n + g][16 * k + 4 * j]);
                    qf[u][k][n][0] = v.x;
                    qf[u][k][n][1] = v.y;
                }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int c = 8 * n + 2 * j + i;
                qs[n][i][0] = sm.q_sum[c][0];
                qs[n][i][1] = sm.q_sum[c][1];
                factor[n][i] = sm.factor[c];
                last[n][i] = sm.last[c];
            }
        }
        const int top = t.first_pos + (part * COLS + columns - 1) / a.group;           // the last key that any column sees
        const int low = t.first_pos + part * COLS / a.group;                           // the last key that every column sees

        float o[STEPS][NT][4], middle[NT][2][2], l[NT][2], m[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[k][n][i] = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                middle[n][i][0] = middle[n][i][1] = l[n][i] = 0.f;
                m[n][i] = -INFINITY;
            }
        }
        int shift[NT][2];                                                               // p s_v is kept divided by 2^shift
#pragma unroll
        for (int n = 0; n < NT; ++n) shift[n][0] = shift[n][1] = kNoShift;

        for (int page = first_page; page < stop; ++page, ++it) {
            const int stage = it % S::kStages;
            if (!wait_record(smem_u32(&sm.full[stage]), (it / S::kStages) & 1, alive) && alive) {
                alive = false;
                atomicExch(&g_kv4_error, 1);
            }
            const uint8_t* rec = sm.records[stage];
            const int token0 = (t.page0 + page) * kPageTokens + 16 * warp;
            // a slice behind every column's last key, or before every window, has nothing to give
            if (token0 <= top && (a.window == 0 || token0 + 15 > low - a.window) && t.pages > 0) {
                const bool masked = token0 + 15 > low || (a.window && token0 <= top - a.window);
                uint2 kp[2], vp[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    kp[r] = *reinterpret_cast<const uint2*>(rec + L::kKeyParams + (16 * warp + g + 8 * r) * 8);
                    vp[r] = *reinterpret_cast<const uint2*>(rec + L::kValueParams + (16 * warp + g + 8 * r) * 8);
                    if (masked && token0 + g + 8 * r > top) kp[r] = vp[r] = make_uint2(0u, 0u);     // what lies there may be no number
                }
                // ---- scores ----
                float s[2][NT][4];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[h][n][i] = 0.f;
                {
                    uint32_t w[E][2];
                    load_words<D>(rec, warp, lane, w);
#pragma unroll
                    for (int p = 0; p < E; ++p) {
                        uint32_t lo[4], hi[4];
                        unpack8(w[p][0], lo);
                        unpack8(w[p][1], hi);
#pragma unroll
                        for (int odd = 0; odd < 2; ++odd) {
                            const int k = 2 * p + odd;
                            const uint32_t frag[4] = {lo[2 * odd], hi[2 * odd], lo[2 * odd + 1], hi[2 * odd + 1]};
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int u = 0; u < TERMS; ++u) mma_f16(s[k * 2 / STEPS][n], frag, qf[u][k][n][0], qf[u][k][n][1]);
                        }
                    }
                }
                float x[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = i >> 1, c = i & 1;
                        float v = s[0][n][i] * kv4_scale(kp[r].x) + s[1][n][i] * kv4_scale(kp[r].y);
                        v += kv4_middle(kp[r].x) * qs[n][c][0] + kv4_middle(kp[r].y) * qs[n][c][1];
                        x[n][i] = v * factor[n][c];
                        if (masked) {
                            const int token = token0 + g + 8 * r;
                            if (token > last[n][c] || (a.window && token <= last[n][c] - a.window)) x[n][i] = -INFINITY;
                        }
                    }
                // ---- the softmax's running maximum: it may lie up to 2^8 behind, so that it seldom moves ----
                bool behind = false;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) behind |= x[n][i] > m[n][i & 1] + 8.f;
                if (__any_sync(0xffffffffu, behind)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float v = fmaxf(x[n][c], x[n][2 + c]);
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
                            const float now = fmaxf(m[n][c], v);
                            const float by = now > -INFINITY ? exp2f(m[n][c] - now) : 1.f;
                            m[n][c] = now;
                            l[n][c] *= by;
                            middle[n][c][0] *= by;
                            middle[n][c][1] *= by;
#pragma unroll
                            for (int k = 0; k < STEPS; ++k) { o[k][n][c] *= by; o[k][n][2 + c] *= by; }
                        }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float by = m[n][i & 1];
                        x[n][i] = masked && x[n][i] == -INFINITY ? 0.f : exp2f(x[n][i] - by);
                        l[n][i & 1] += x[n][i];
                    }
                // ---- the scale of p s_v: moves where a value's scale is more than 2^4 above it ----
                const float sv[2][2] = {{kv4_scale(vp[0].x), kv4_scale(vp[0].y)}, {kv4_scale(vp[1].x), kv4_scale(vp[1].y)}};
                const float most = fmaxf(fmaxf(sv[0][0], sv[0][1]), fmaxf(sv[1][0], sv[1][1]));
                const int e = (int)(__float_as_uint(most) >> 23) - 127;
                bool above = false;
#pragma unroll
                for (int n = 0; n < NT; ++n) above |= e > min(shift[n][0], shift[n][1]) + 4;
                if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            int now = kNoShift;                                        // of the values that the column sees and that are numbers
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const float v = fmaxf(sv[r][0] < INFINITY ? sv[r][0] : 0.f, sv[r][1] < INFINITY ? sv[r][1] : 0.f);
                                if (x[n][2 * r + c] > 0.f) now = max(now, (int)(__float_as_uint(v) >> 23) - 127);
                            }
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) now = max(now, __shfl_xor_sync(0xffffffffu, now, d));
                            now = min(120, now);
                            if (now > shift[n][c]) {
                                now = max(-120, now);
                                const float by = shift[n][c] > kNoShift ? exp2f((float)(shift[n][c] - now)) : 0.f;
                                shift[n][c] = now;
#pragma unroll
                                for (int k = 0; k < STEPS; ++k) { o[k][n][c] *= by; o[k][n][2 + c] *= by; }
                            }
                        }
                }
                // ---- weights times scales, as the operand with tokens along K ----
                uint32_t pf[TERMS][2][NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float down[2] = {shift[n][0] > kNoShift ? power2(-shift[n][0]) : 0.f, shift[n][1] > kNoShift ? power2(-shift[n][1]) : 0.f};
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float x0 = x[n][2 * r], x1 = x[n][2 * r + 1], d0 = x0 * down[0], d1 = x1 * down[1];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float md = kv4_middle(h ? vp[r].y : vp[r].x);
                            float y0 = d0 * sv[r][h], y1 = d1 * sv[r][h], z0 = x0 * md, z1 = x1 * md;
                            if (masked) {                                              // a key that is not seen may have parameters that are no numbers
                                if (x0 == 0.f) y0 = z0 = 0.f;
                                if (x1 == 0.f) y1 = z1 = 0.f;
                            }
                            middle[n][0][h] += z0;
                            middle[n][1][h] += z1;
                            const uint32_t p = pack_half2(y0, y1);
                            pf[0][h][n][r] = transpose8(p);
                            if constexpr (TERMS == 2) {
                                const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&p));
                                pf[TERMS - 1][h][n][r] = transpose8(pack_half2(y0 - back.x, y1 - back.y));
                            }
                        }
                    }
                }
                // ---- weighted values ----
                {
                    uint32_t w[E][2];
                    load_words<D>(rec + L::kValues, warp, lane, w);
#pragma unroll
                    for (int p = 0; p < E; ++p) {
                        uint32_t lo[4], hi[4];
                        unpack8(w[p][0], lo);
                        unpack8(w[p][1], hi);
#pragma unroll
                        for (int odd = 0; odd < 2; ++odd) {
                            const int k = 2 * p + odd;
                            const uint32_t frag[4] = {lo[2 * odd], lo[2 * odd + 1], hi[2 * odd], hi[2 * odd + 1]};
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int u = 0; u < TERMS; ++u) mma_f16(o[k][n], frag, pf[u][k * 2 / STEPS][n][0], pf[u][k * 2 / STEPS][n][1]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.empty[stage]));
        }

        // ---- the four warps' parts become one ----
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], d);
                    middle[n][c][0] += __shfl_xor_sync(0xffffffffu, middle[n][c][0], d);
                    middle[n][c][1] += __shfl_xor_sync(0xffffffffu, middle[n][c][1], d);
                }
        if (g == 0)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    sm.merge_m[warp][8 * n + 2 * j + c] = m[n][c];
                    sm.merge_l[warp][8 * n + 2 * j + c] = l[n][c];
                }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        float all_m[NT][2], all_l[NT][2], by[NT][2], up[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int col = 8 * n + 2 * j + c;
                float v = sm.merge_m[0][col];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) v = fmaxf(v, sm.merge_m[w][col]);
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w)
                    if (sm.merge_m[w][col] > -INFINITY) sum += sm.merge_l[w][col] * exp2f(sm.merge_m[w][col] - v);
                all_m[n][c] = v;
                all_l[n][c] = sum;
                up[n][c] = shift[n][c] > kNoShift ? power2(shift[n][c]) : 0.f;
                by[n][c] = m[n][c] > -INFINITY ? exp2f(m[n][c] - v) : 0.f;
            }
        // channel of a lane's sums: block k, channels 2 g (i < 2) and 2 g + 1
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = i & 1;
                    o[k][n][i] = by[n][c] > 0.f ? (o[k][n][i] * up[n][c] + middle[n][c][k * 2 / STEPS]) * by[n][c] : 0.f;
                }
#pragma unroll
        for (int round = kWarps / 2; round > 0; round >>= 1) {
            if (warp >= round && warp < 2 * round) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < STEPS; ++k)
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            *reinterpret_cast<float2*>(&sm.merge[warp - round][8 * n + 2 * j + c][16 * k + 2 * g]) = make_float2(o[k][n][c], o[k][n][2 + c]);
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (warp < round) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int k = 0; k < STEPS; ++k)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float2 v = *reinterpret_cast<const float2*>(&sm.merge[warp][8 * n + 2 * j + c][16 * k + 2 * g]);
                            o[k][n][c] += v.x;
                            o[k][n][2 + c] += v.y;
                        }
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
        }
        if (warp == 0) {
            const bool whole = first_page == 0 && stop == pages;
            // a part of a tile that an earlier block began lies in the block's first place, one that goes on behind it in the second
            float* mine = a.scratch + ((int64_t)blockIdx.x * 2 + (first_page == 0 ? 1 : 0)) * part_floats<D>(COLS);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int col = 8 * n + 2 * j + c;
                    if (col >= columns) continue;
                    if (whole) {
                        const int q = part * COLS + col;
                        T* out = reinterpret_cast<T*>(a.out) + ((int64_t)(t.row + q / a.group) * a.n_heads + head * a.group + q % a.group) * D;
                        const float inv = all_l[n][c] > 0.f ? 1.f / all_l[n][c] : 0.f;
#pragma unroll
                        for (int k = 0; k < STEPS; ++k) {
                            out[16 * k + 2 * g] = from_f32<T>(o[k][n][c] * inv);
                            out[16 * k + 2 * g + 1] = from_f32<T>(o[k][n][2 + c] * inv);
                        }
                    } else {
                        float* p = mine + (int64_t)col * (D + 2);
#pragma unroll
                        for (int k = 0; k < STEPS; ++k) *reinterpret_cast<float2*>(p + 2 + 16 * k + 2 * g) = make_float2(o[k][n][c], o[k][n][2 + c]);
                        if (g == 0) {
                            p[0] = all_m[n][c];
                            p[1] = all_l[n][c];
                        }
                    }
                }
        }
        unit += stop - first_page;
    }
}

// Adds up the parts of the tiles that were cut: one block per tile, part and key-value head, a warp per column.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(256)
kv4_combine_kernel(const __grid_constant__ AttendArgs a, int blocks) {
    constexpr int COLS = 8 * NT;
    __shared__ int scan[9];
    __shared__ int prefix[kMostTiles + 1];
    pdl_launch_dependents();
    pdl_wait();
    const int index = blockIdx.x;
    const Tile t = tile_of(a, index, COLS);
    if ((int)blockIdx.y >= t.parts * a.n_kv) return;
    sum_tiles(a, COLS, prefix, scan);
    const int64_t units = prefix[a.n_tiles];
    const int sharing = sharing_blocks(units, blocks);
    const int pages = max(1, t.pages);
    const int64_t begin = prefix[index] + (int64_t)blockIdx.y * pages, last = begin + pages - 1;
    const int b0 = block_of(begin, units, sharing), b1 = block_of(last, units, sharing);
    if (b0 == b1) return;                                                                // the block that had it all wrote the output
    const int head = blockIdx.y % a.n_kv, part = blockIdx.y / a.n_kv;
    const int columns = min(COLS, t.tokens * a.group - part * COLS);
    const int lane = threadIdx.x & 31;
    for (int c = threadIdx.x >> 5; c < columns; c += 8) {
        const auto place = [&](int b) { return a.scratch + ((int64_t)b * 2 + (b == b0 ? 1 : 0)) * part_floats<D>(COLS) + (int64_t)c * (D + 2); };
        float top = -INFINITY;
        for (int b = b0 + lane; b <= b1; b += 32) top = fmaxf(top, place(b)[0]);
        top = warp_max(top);
        float l = 0.f, o[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
        for (int b = b0; b <= b1; ++b) {
            const float* p = place(b);
            const float by = p[0] > -INFINITY ? exp2f(p[0] - top) : 0.f;
            l += p[1] * by;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] += by > 0.f ? p[2 + lane + 32 * i] * by : 0.f;
        }
        const int q = part * COLS + c;
        T* out = reinterpret_cast<T*>(a.out) + ((int64_t)(t.row + q / a.group) * a.n_heads + head * a.group + q % a.group) * D;
        const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) out[lane + 32 * i] = from_f32<T>(o[i] * inv);
    }
}

template <typename T, int D, int NT, int TERMS>
int attend(const AttendArgs& a, cudaStream_t stream) {
    static bool done[kMaxDevices];
    constexpr int bytes = (int)sizeof(Smem<D, NT, TERMS>) + 128;
    const int status = ensure_dynamic_smem(kv4_attention_kernel<T, D, NT, TERMS>, bytes, done);
    if (status != CPM_OK) return status;
    const int sms = device_sms();
    if (sms <= 0) return CPM_BAD_ARGUMENT;
    const int blocks = sms * blocks_per_sm(D, NT, TERMS);
    cpm_launch(kLaunchAttention, kv4_attention_kernel<T, D, NT, TERMS>, dim3(blocks), kThreads, bytes, stream, a);
    const int most_tokens = a.cu_q ? kTileTokens : 1;
    const int64_t rows = (int64_t)((most_tokens * a.group + 8 * NT - 1) / (8 * NT)) * a.n_kv;
    if (rows > 65535) return CPM_BAD_ARGUMENT;
    cpm_launch(kLaunchAttention, kv4_combine_kernel<T, D, NT>, dim3(a.n_tiles, (unsigned)rows), 256, 0, stream, a, blocks);
    return launch_status();
}

template <typename T, int D, int TERMS>
int by_columns(const AttendArgs& a, cudaStream_t stream) {
    // one tile of eight columns where a token's heads of a key-value head are no more, else two
    const bool narrow = !a.cu_q && a.group <= 8;
    return narrow ? attend<T, D, 1, TERMS>(a, stream) : attend<T, D, 2, TERMS>(a, stream);
}

template <typename T, int TERMS>
int by_head_size(const AttendArgs& a, int d, cudaStream_t stream) {
    switch (d) {
        case 32: return by_columns<T, 32, TERMS>(a, stream);
        case 64: return by_columns<T, 64, TERMS>(a, stream);
        case 96: return by_columns<T, 96, TERMS>(a, stream);
        case 128: return by_columns<T, 128, TERMS>(a, stream);
        default: return CPM_BAD_ARGUMENT;
    }
}

}  // namespace

// 32-bit floats that a launch needs for the parts of tiles that are cut.
CPM_API int64_t cpm_kv4_attention_scratch_floats(int d) {
    return (int64_t)device_sms() * kMostBlocksPerSm * 2 * 16 * (d + 2);
}
CPM_API int cpm_kv4_attention_most_tiles() { return kMostTiles; }
// Reads and clears the error that a kernel recorded (0: none).
CPM_API int cpm_kv4_attention_error() {
    int code = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&code, g_kv4_error, sizeof(int)) != cudaSuccess) return -1;
    if (code) cudaMemcpyToSymbol(g_kv4_error, &zero, sizeof(int));
    return code;
}

CPM_API int cpm_kv4_attention(const void* q, const void* records, void* out, const int* kv_len, const int* slots, const int* page_table,
                              int max_pages, const int* cu_q, const int* tile_seq, const int* tile_row, int n_tiles, float* scratch, int n_heads,
                              int n_kv, int d, int window, float scale, int dtype, cudaStream_t stream) {
    if (n_tiles <= 0) return CPM_OK;
    if (n_tiles > kMostTiles || n_heads < 1 || n_kv < 1 || n_heads % n_kv || window < 0) return CPM_BAD_ARGUMENT;
    if ((cu_q == nullptr) != (tile_seq == nullptr) || (cu_q == nullptr) != (tile_row == nullptr)) return CPM_BAD_ARGUMENT;
    if ((uintptr_t)records & 15) return CPM_BAD_ARGUMENT;
    const AttendArgs a{q, out, (const uint8_t*)records, kv_len, slots, page_table, cu_q, tile_seq, tile_row, scratch, max_pages, n_tiles, n_heads, n_kv,
                       n_heads / n_kv, window, scale};
    return dtype == CPM_BF16 ? by_head_size<bf16, 1>(a, d, stream) : by_head_size<float, 2>(a, d, stream);
}
