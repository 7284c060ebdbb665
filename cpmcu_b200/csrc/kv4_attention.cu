// Attention over a cache held in 4 bits:  o = sum_j p_j v_j,  p = softmax(q . k_j * scale)  over the keys a query sees.
//
// The codes are small whole numbers, which fp16 holds exactly, so that both products run on the tensor cores (mma.m16n8k16, fp16
// in, fp32 sums) without rounding a key or a value: with s and m a half row's scale and middle,
//     q . k  = sum over halves of  s_k (q_h . (c - 8)) + m_k sum(q_h)
//     o      = sum over halves of  (p s_v) (c - 8)      + p m_v
// Keys and values are the operand with 16 rows, a tile of 8 * NT queries (query heads of one key-value head, of one or several tokens) the
// one with 8 columns.  A query is divided by a power of two first, which makes it an fp16 number without loss; p s_v is kept below
// 2^15 in the same way.  bf16 queries: p s_v is rounded to fp16 (11 bits; the output has 8), of which it keeps fewer below 2^-14 of the column's largest p
// and scale, an error of 2^-25 of these.  fp32 queries: q and p s_v are sums of two fp16 numbers (22 bits; a third would cost a third product); p s_v
// is taken 2^10 larger, so that the second number of a weight has all its bits down to 2^-13 of the largest and is off by 2^-35 of it below, and
// a slice's products are added to the sums by ordinary additions, since the tensor core cuts its sums off, a bias that grows with the slices and that
// counts where codes and middles nearly cancel.  Error against 64 bits, of the result's norm, without these two, with them, and of fp32 throughout: 40,000
// keys 4.6e-6, 8.9e-7, 2.1e-7, values that do not average to nothing 1.8e-7, 9.2e-8, 6.4e-8, scales over some e^4 1.1e-6, 2.4e-7, 2.1e-7.
//
// One block an SM.  A batch's rows of pages (a tile's, of one key-value head) lie in a line, of which every block takes a piece of equal cost, so that
// unequal sequences leave no SM idle; few rows have blocks of their own.  A row that several blocks share is put together by a second kernel.  Four
// warps take 16 tokens each of a page, and the block's two to four groups of four warps every second to fourth page.  A warp brings its tokens into a
// ring of its own by asynchronous 16-byte copies, of which a lane reads most of what it copied itself, and keeps a softmax of its own, so that nothing
// synchronises the warps until a row ends.  (Bulk copies of a slice's four pieces took longer than the arithmetic: each needs its addresses in
// uniform registers.  Blocks of four warps, three an SM, leave three times as many parts to add up: 41 us where blocks of twelve took 30, for one
// sequence of 131,071 keys.)
//
// 32 heads on 2 of 128, bf16: 1,000 keys 12 us, 131,071 keys 25 us (1.5 TB/s of records); 64 sequences of 1 to 8,192 keys, 16 heads on 2 of 64,
// 28 us (1.6 TB/s); 5 of 300 to 2,500 keys, fp32, 9 us; 200 of 1 to 4,000, 32 heads on 8 of 128, 165 us (2.8 TB/s); prompts of 2,048 tokens behind 4,101
// keys, 16 heads on 2: bf16 of 32 and 96 340 and 532 us, fp32 of 32, 64 and 96 456, 627 and 760, 32 heads on 2 of 128 1,659.  Bound, where there are many keys, by
// instructions: a slice of 16 tokens costs a warp some 500, of which unpacking the codes is a third; where there are few, by the way to the first
// key: 2 us for lengths and shares, 1 for page numbers, 1 for queries, 2 for the first slice and 2 for the parts, whose instructions
// come from L2, and 2.5 for the second kernel.
#include "kv4.cuh"

CPM_BOUNDS_TU(kv4_attention)

namespace {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

constexpr int kSlices = 4;                             // warps to a page
constexpr int kTileTokens = 64;                        // tokens of a prompt's query tile
constexpr int kMostTiles = 512;                        // tiles of one launch (what they are lies in shared memory)

struct AttendArgs {
    const void* q;
    void* out;
    const uint8_t* records;
    const int *kv_len, *slots, *page_table;
    const int *cu_q, *tile_seq, *tile_row;             // null: one token per sequence
    float* scratch;
    int max_pages, n_tiles, n_heads, n_kv, group, window;
    float scale, per_group, per_kv;                    // 1 / group, 1 / n_kv
};

// n / m for 0 <= n < 2^20 and 1 / m: the quotient's error, below 2^-3 / m, stays away from the next whole number, which is 1 / (2 m) off.  (A division
// of whole numbers is some twenty instructions, all of which a block of a few pages fetches from L2.)
__device__ __forceinline__ int quotient(int n, float per) { return (int)(((float)n + 0.5f) * per); }

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
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst), "l"(src) : "memory");
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

// Two fp32 numbers in a register pair: one instruction for both.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 both(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void store2(float* p, float lo, float hi) { *reinterpret_cast<float2*>(p) = make_float2(lo, hi); }
__device__ __forceinline__ void store2(bf16* p, float lo, float hi) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(lo, hi); }
// 2^x; below 2^-126 zero, which no sum of weights up to 2^8 notices.
__device__ __forceinline__ float fast_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
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
__device__ __forceinline__ void load_words(const uint8_t* codes, int lane, uint32_t (&w)[D / 32][2]) {
    using L = Kv4<D>;
    const uint8_t* p = codes + L::word(0, 0, lane, 0);
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
__device__ __forceinline__ float inverse_power2(float p) { return __uint_as_float(0x7f000000u - __float_as_uint(p)); }      // of a power of two
__device__ __forceinline__ float power2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// How far p s_v may lie from where it is put: the running maximum 2^kScoreLag behind, the largest scale kScaleLag above the one that has been fitted,
// which is put at 2^kUp; together 2^15.
template <int TERMS> constexpr float kScoreLag = TERMS == 2 ? 3.f : 8.f;
template <int TERMS> constexpr float kScaleLag = TERMS == 2 ? 4.f : 16.f;
template <int TERMS> constexpr int kUp = TERMS == 2 ? 10 : 0;

// Warps of a block, by what the registers allow: 16 with up to 128 registers a thread, 12 with 168, 8 with 255.
constexpr int warps_of(int d, int nt, int terms) { return nt == 1 ? 16 : terms == 2 && d > 32 ? 8 : 12; }

template <int D, int NT, int TERMS>
struct Smem {
    static constexpr int kWarps = warps_of(D, NT, TERMS);
    static constexpr int kStages = D < 96 ? 6 : 3;
    static constexpr int kCols = 8 * NT;
    static constexpr int kQStride = D + 16;            // fp16 numbers a row: rows 32 bytes apart modulo 128
    // 16 tokens of a record: key codes, value codes, key parameters, value parameters
    static constexpr int kStage = 2 * Kv4<D>::kSlice + 256;
    static constexpr int kChunks = kStage / 16, kPieces = (kChunks + 31) / 32;
    alignas(128) uint8_t ring[kWarps][kStages][kStage];
    alignas(16) __half q[TERMS][kCols][kQStride];
    // what the warps leave at a row's end: their sums as they lie in the registers (16 channels of 8 columns after the other, a lane's four
    // numbers together), and of each column the maximum, the sum of weights, both halves' middles, and the factor of the sums
    alignas(16) float merge[kWarps][NT][D / 16][32][4];
    alignas(16) float merge_m[kWarps][kCols], merge_l[kWarps][kCols], merge_mid[2][kWarps][kCols], merge_up[kWarps][kCols];
    float end_m[kCols], end_l[kCols], end_mid[2][kCols];
    float q_sum[kCols][2], factor[kCols];
    int last[kCols];                                   // a column's last key, -1: no such column
    int scan[kWarps];
    int last_block;                                    // of the block's row, where it has one only, else -1
    int prefix[kMostTiles + 1];
    Tile tiles[kMostTiles];
};

// A row of pages (a tile's, of one key-value head and part) costs a block its pages and some more, for the queries that it prepares and the parts
// that it adds up.  All rows lie one behind the other in a line of such costs, a row's extra cost first.  (Extra cost of 2, 4 and 8 pages for each group
// of warps: 64 sequences of up to 8,192 keys, 16 heads on 2 of 64, 31.0, 27.6 and 29.5 us; 200 of up to 4,000, 32 on 8 of 128, 172, 163 and 177.)
constexpr int extra_cost(int groups) { return 4 * groups; }
// Sharing by cost: each of the blocks takes a piece of the line, wherever rows begin or end; fewer blocks where there is little.
struct Shares { int sharing, each, more; };            // the first ``more`` blocks have one more than ``each``
__device__ __forceinline__ Shares shares_of(int cost, int groups, int blocks) {
    const int least = groups + extra_cost(groups) / 4, sharing = min(blocks, max(1, (cost + least - 1) / least));
    return Shares{sharing, cost / sharing, cost % sharing};
}
__device__ __forceinline__ int share_begin(const Shares& s, int block) { return block * s.each + min(block, s.more); }
__device__ __forceinline__ int block_of(const Shares& s, int at) {
    const int longer = s.more * (s.each + 1);
    return at < longer ? at / (s.each + 1) : s.more + (at - longer) / s.each;
}
// Sharing by rows: a block works on one row alone, a row has a block or more by its number of pages.  Possible where there is a block for every row of
// single tokens, and taken where the longest piece of a row is no more than 5/4 of a piece of the line, in which a block may end one row and begin
// another: us by rows and by the line, 32 heads on 2 of 128, 2,000 keys each: 5 sequences 11.9 and 15.0, 18 17.3 and 20.5, 36 24.1 and 28.6, 72 29.0 and
// 42.7; 1 to 4,000 keys: 18 17.3 and 20.8, 36 (28 pages against 21) 28.5 and 28.1, 72 (63 against 42) 42.4 and 41.8.
__host__ __device__ __forceinline__ int rows_of_tile(const AttendArgs& a, int columns) { return a.n_kv * ((a.group + columns - 1) / columns); }
__host__ __device__ __forceinline__ bool few_rows(const AttendArgs& a, int columns, int blocks) {
    return !a.cu_q && (int64_t)a.n_tiles * rows_of_tile(a, columns) <= blocks;
}

// The tiles and the prefix sums of their rows' costs; every thread of the block takes part.  (A row without keys counts as one page, for the
// zeros that it gets.)
__device__ __forceinline__ void sum_tiles(const AttendArgs& a, int columns, int extra, Tile* tiles, int* prefix, int* scan) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int carry = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < a.n_tiles; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        int own = 0;
        if (i < a.n_tiles) {
            const Tile t = tile_of(a, i, columns);
            tiles[i] = t;
            own = (extra + max(1, t.pages)) * t.parts * a.n_kv;
        }
        int v = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += x;
        }
        if (a.n_tiles <= 32) {                              // one warp has them all
            if (i < a.n_tiles) prefix[i] = v - own;
            if (threadIdx.x == 31) prefix[a.n_tiles] = v;
            __syncthreads();
            return;
        }
        if (lane == 31) scan[warp] = v;
        __syncthreads();
        int before = carry, all = carry;
#pragma unroll 1
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
__device__ __forceinline__ int find_tile(const int* prefix, int n, int at) {
    int lo = 0, hi = n;                                 // the last tile that begins there or before (empty tiles begin where the next does)
#pragma unroll 1
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= at) lo = mid; else hi = mid;
    }
    return lo;
}

// Scratch: a head of kHeadInts numbers for every block, then two parts a block.  A part holds for each column the weighted values, the
// maximum and the sum.  A row that several blocks share has its head, for the kernel that adds up, from the block that begins it: in the row's place
// where there is a head for every row, else in that block's.
struct CutRow { int first_block, last_block, row, part, head, columns; };
constexpr int kHeadInts = 8;
template <int D> constexpr int kPartStride = D + 4;
template <int D>
__device__ __forceinline__ float* part_of(const AttendArgs& a, int blocks, int block, bool goes_on, int columns) {
    return a.scratch + (int64_t)blocks * kHeadInts + ((int64_t)block * 2 + (goes_on ? 1 : 0)) * columns * kPartStride<D>;
}

template <typename T, int D, int NT, int TERMS>
__global__ void __launch_bounds__(32 * warps_of(D, NT, TERMS), 1)
kv4_attention_kernel(const __grid_constant__ AttendArgs a) {
    using L = Kv4<D>;
    using S = Smem<D, NT, TERMS>;
    constexpr int COLS = S::kCols, STEPS = D / 16, E = D / 32, STAGES = S::kStages, WARPS = S::kWarps, GROUPS = WARPS / kSlices;
    constexpr bool Q_IN_REGISTERS = NT == 1 && TERMS == 1;      // else they are read again for every 16 tokens: 32 registers more would leave room for a block less
    extern __shared__ __align__(128) uint8_t raw[];
    S& sm = *reinterpret_cast<S*>(raw);                  // (no arithmetic on the address: the compiler would lose that it is shared memory)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, slice = warp % kSlices, turn = warp / kSlices;      // its tokens of a page, and of how many pages the how-manieth
    // The kernel that joins the parts is let in by the blocks' ends alone.  Let in at their start its blocks waited on the SMs through all of this one,
    // and in a decode step the products of few rows around it came late: ms a step of 8 layers, 32 heads on 2 of 128, behind 4,096 tokens, at their start
    // and at their ends: 1 row 1.26 and 0.87, 8 rows 1.87 and 1.03, 64 rows 1.45 and 1.32 (a cache in bf16: 0.84, 1.06 and 1.33).
    pdl_wait();
    constexpr int EXTRA = extra_cost(GROUPS);
    sum_tiles(a, COLS, EXTRA, sm.tiles, sm.prefix, sm.scan);
    const int cost = sm.prefix[a.n_tiles];
    int begin = 0, end = 0, start = 0;                                                    // the block's piece of the line, and its first tile
    const bool few = few_rows(a, COLS, gridDim.x);
    const int per_tile = rows_of_tile(a, COLS);
    const Shares shares = shares_of(cost, GROUPS, gridDim.x);
    // a row of n pages has 1 + n / each blocks, but no more than have a page for each of their groups
    int each = 0;
    const auto blocks_of = [&](int pages) { return min(1 + pages / each, (pages + GROUPS - 1) / GROUPS); };
    bool by_rows = false;
    if (few) {
        const int rows = a.n_tiles * per_tile, spare = (int)gridDim.x - rows;
        each = spare > 0 ? (cost - rows * EXTRA + spare - 1) / spare : 0x40000000;
        int longest = 0;
#pragma unroll 1
        for (int i = lane; i < a.n_tiles; i += 32) {
            const int pages = max(1, sm.tiles[i].pages), n = blocks_of(pages);
            longest = max(longest, (pages + n - 1) / n);
        }
        longest = __reduce_max_sync(0xffffffffu, longest);
        by_rows = 4 * (int64_t)longest <= 5 * (int64_t)(shares.each + 1);
    }
    if (by_rows) {
        int block = blockIdx.x;
#pragma unroll 1
        for (int i0 = 0; i0 < a.n_tiles; i0 += 32) {
            const int pages = i0 + lane < a.n_tiles ? max(1, sm.tiles[i0 + lane].pages) : 0;
            const int blocks = pages ? blocks_of(pages) : 0;
            int v = blocks * per_tile;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += x;
            }
            const uint32_t behind = __ballot_sync(0xffffffffu, v > block);
            if (behind) {
                const int from = __ffs(behind) - 1, n = __shfl_sync(0xffffffffu, blocks, from), m = __shfl_sync(0xffffffffu, pages, from);
                block -= __shfl_sync(0xffffffffu, v, from) - n * per_tile;
                start = i0 + from;
                const int row = block / n, k = block - row * n, first = sm.prefix[start] + row * (EXTRA + m);
                begin = first + (k ? EXTRA + k * (m / n) + min(k, m % n) : 0);
                end = first + EXTRA + (k + 1) * (m / n) + min(k + 1, m % n);
                if (threadIdx.x == 0) sm.last_block = (int)blockIdx.x - k + n - 1;
                break;
            }
            block -= __shfl_sync(0xffffffffu, v, 31);
        }
    } else {
        if ((int)blockIdx.x < shares.sharing) {
            begin = share_begin(shares, blockIdx.x);
            end = share_begin(shares, blockIdx.x + 1);
            start = find_tile(sm.prefix, a.n_tiles, begin);
        }
        if (threadIdx.x == 0) {
            sm.last_block = -1;
            if (!few) reinterpret_cast<CutRow*>(a.scratch + (int64_t)blockIdx.x * kHeadInts)->last_block = -1;
        }
    }
    if (begin >= end) return;
    // The row of pages at a place of the line: its tile, its number among the tile's, and which of its pages are the block's.
    const auto walk = [&](int& at, int& index, uint32_t& row, int& first, int& stop) {
#pragma unroll 1
        while (sm.prefix[index + 1] <= at) ++index;
        const int pages = max(1, sm.tiles[index].pages), in = at - sm.prefix[index];
        row = (uint32_t)in / (uint32_t)(EXTRA + pages);
        const int within = in - row * (EXTRA + pages);
        first = max(0, within - EXTRA);
        stop = min(pages, within + end - at - EXTRA);
        at += min(EXTRA + pages - within, end - at);
    };

    // ---- what the warp has asked for: it runs ahead of what it works on by the ring's length, across the borders of rows ----
    // (of the block's pages of a row, every GROUPS-th from ``turn`` on)
    int ask_at = begin, ask_index = start, ask_page = 0, ask_stop = 0, ask_ids = 0, ask_base = 0, ask_first = 0, asked = 0;
    const int* ask_table = a.page_table;
    const uint8_t* ask_records = a.records;
    bool ask_any = false;
    // where in a record the lane's i-th 16 bytes of a slice come from: key codes, value codes, key parameters, value parameters
    const auto ask_from = [&](int i) {
        const int c = 32 * i + lane;
        return c < D / 2 ? slice * L::kSlice + 16 * c : c < D ? L::kValues + slice * L::kSlice + 16 * (c - D / 2)
             : (c < D + 8 ? L::kKeyParams : L::kValueParams - 128) + slice * 128 + 16 * (c - D);
    };
    const auto ask = [&]() {
        if (ask_page >= ask_stop && ask_at < end) {        // the next row that has a page for the warp
            uint32_t row = 0;
#pragma unroll 1
            while (ask_page >= ask_stop && ask_at < end) {
                walk(ask_at, ask_index, row, ask_page, ask_stop);
                ask_page += turn;
            }
            ask_any = sm.tiles[ask_index].pages > 0;
            ask_first = sm.tiles[ask_index].page0;
            ask_table = a.page_table + (int64_t)sm.tiles[ask_index].slot * a.max_pages;
            ask_records = a.records + (int64_t)((int)row - quotient(row, a.per_kv) * a.n_kv) * L::kBytes;
            ask_base = ask_page - 32 * GROUPS;
        }
        if (ask_page < ask_stop) {
            if (ask_page - ask_base >= 32 * GROUPS) {      // the next 32 page numbers, one a lane
                ask_base = ask_page;
                const int i = ask_page + lane * GROUPS;
                ask_ids = i < ask_stop && ask_any ? CPM_PAGE(ask_table, ask_first + i, a.max_pages) : 0;
            }
            const int number = __shfl_sync(0xffffffffu, ask_ids, (ask_page - ask_base) / GROUPS);
            if (ask_any) {                                 // (a row without keys: nothing to bring)
                const uint8_t* from = ask_records + (int64_t)number * a.n_kv * L::kBytes;
                const uint32_t to = smem_u32(sm.ring[warp][asked]) + lane * 16;
#pragma unroll
                for (int i = 0; i < S::kPieces; ++i)
                    if (32 * i + 31 < S::kChunks || lane < S::kChunks - 32 * i) copy16(to + 512 * i, from + ask_from(i));
            }
            ask_page += GROUPS;
            if (++asked == STAGES) asked = 0;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) ask();

    // ---- what it works on.  One loop over slices, with a tile's beginning and end inside: every part of the code is there once, since a
    // block runs most of it a few times only and the first run of an instruction comes from L2 (80 KB of unrolled code took 25 us for one page) ----
    const int g = lane >> 2, j = lane & 3;
    int at = begin, index = start, stage = 0;
    uint2 qf[Q_IN_REGISTERS ? STEPS : 1];
    // of a lane's two columns of every eight: q's sums, the factor of the scores, minus the running maximum, the sum of weights, the
    // power of two that p s_v is multiplied by, and the sums of p m_v
    f32x2 q_sum[NT][2], factor[NT], minus[NT], sum[NT], down[NT], middle[NT][2];
    float o[STEPS][NT][4];
    float limit = 0.f;                                                                 // a value's scale above it makes ``down`` move
    uint32_t blank = 0;                                                                // bit 2 n + c: the column has seen no key yet
    const auto q_fragment = [&](int u, int k, int n) { return *reinterpret_cast<const uint2*>(&sm.q[u][8 * n + g][16 * k + 4 * j]); };

#pragma unroll 1
    while (at < end) {
        // ---- a row of pages begins ----
        uint32_t in_tile;
        int first_page, stop;
        walk(at, index, in_tile, first_page, stop);
        if (stop <= first_page) break;                                                  // only a part of a row's extra cost is left
        const Tile t = sm.tiles[index];
        const int pages = max(1, t.pages), part = quotient(in_tile, a.per_kv), head = (int)in_tile - part * a.n_kv;
        const int columns = min(COLS, t.tokens * a.group - part * COLS), row = t.row;
        const int key0 = t.page0 * kPageTokens + 16 * slice;
        const int low = t.first_pos + quotient(part * COLS, a.per_group);                               // the last key that every column sees
        const int top = t.pages > 0 ? t.first_pos + quotient(part * COLS + columns - 1, a.per_group) : -1;      // the last that any column sees
        // queries: divided by a power of two, in fp16 (TERMS = 2: and what that leaves).  All columns at once, some threads to each
        if (threadIdx.x < 16 * COLS) {
            constexpr int PER = 16, EP = D / PER;
            const int c = threadIdx.x / PER, n = part * COLS + c, token = quotient(n, a.per_group), from = threadIdx.x % PER * EP;
            const T* q = reinterpret_cast<const T*>(a.q) + ((int64_t)(row + token) * a.n_heads + head * a.group + n - token * a.group) * D + from;
            float x[EP], most = 0.f;
            if constexpr (EP % 4 == 0) {
#pragma unroll
                for (int i = 0; i < EP; i += 4) {
                    const float4 v = c < columns ? load4(q + i) : make_float4(0.f, 0.f, 0.f, 0.f);
                    x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < EP; ++i) x[i] = c < columns ? to_f32(q[i]) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < EP; ++i) most = fmaxf(most, fabsf(x[i]));
#pragma unroll
            for (int d = 1; d < PER; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
            const int e = shift_of(most);
            const float by = power2(-e);
            float total = 0.f;
#pragma unroll
            for (int i = 0; i < EP; i += 2) {
                const float y0 = x[i] * by, y1 = x[i + 1] * by;
                total += y0 + y1;
                const __half2 h = __floats2half2_rn(y0, y1);
                *reinterpret_cast<__half2*>(&sm.q[0][c][from + i]) = h;
                if constexpr (TERMS == 2) *reinterpret_cast<__half2*>(&sm.q[1][c][from + i]) = __floats2half2_rn(y0 - __low2float(h), y1 - __high2float(h));
            }
#pragma unroll
            for (int d = 1; d < PER / 2; d <<= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
            if (threadIdx.x % (PER / 2) == 0) sm.q_sum[c][threadIdx.x % PER / (PER / 2)] = total;
            if (from == 0) {
                sm.factor[c] = power2(e) * a.scale * 1.4426950408889634f;
                sm.last[c] = c < columns ? t.first_pos + token : -1;
            }
        }
        __syncthreads();
        if constexpr (Q_IN_REGISTERS)
#pragma unroll
            for (int k = 0; k < STEPS; ++k) qf[k] = q_fragment(0, k, 0);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int c = 8 * n + 2 * j;
            q_sum[n][0] = pair(sm.q_sum[c][0], sm.q_sum[c + 1][0]);
            q_sum[n][1] = pair(sm.q_sum[c][1], sm.q_sum[c + 1][1]);
            factor[n] = pair(sm.factor[c], sm.factor[c + 1]);
            minus[n] = sum[n] = down[n] = middle[n][0] = middle[n][1] = pair(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[k][n][i] = 0.f;
        }
        limit = -1.f;
        blank = 0xffffffffu;

#pragma unroll 1
        for (int page = first_page + turn; page < stop; page += GROUPS) {
            ask();                                                                         // into the place that the last slice left
            asm volatile("cp.async.wait_group %0;" :: "n"(STAGES - 1) : "memory");
            __syncwarp();
            const uint8_t* rec = sm.ring[warp][stage];
            if (++stage == STAGES) stage = 0;
            const int token0 = key0 + page * kPageTokens;
            // a slice behind every column's last key, or before every window, has nothing to give
            if (token0 <= top && (a.window == 0 || token0 + 15 > low - a.window)) {
                uint2 kp[2], vp[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    kp[r] = *reinterpret_cast<const uint2*>(rec + 2 * L::kSlice + (g + 8 * r) * 8);
                    vp[r] = *reinterpret_cast<const uint2*>(rec + 2 * L::kSlice + 128 + (g + 8 * r) * 8);
                }
                uint32_t seen = 0xffffffffu;                                               // bit 4 n + 2 r + c: row g + 8 r is seen by the lane's column c
                if (token0 + 15 > low || (a.window && token0 <= top - a.window)) {
                    seen = 0;
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int token = token0 + g + 8 * r;
                        if (token > top) kp[r] = vp[r] = make_uint2(0u, 0u);                // what lies there may be no number
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const int last = sm.last[8 * n + 2 * j + c];
                                if (token <= last && (a.window == 0 || token > last - a.window)) seen |= 1u << (4 * n + 2 * r + c);
                            }
                        // A row that only some columns see and that is no number would reach the others as 0 * NaN: it goes to
                        // those that see it here, and is nobody's afterwards; of a value half a row alone, whose other half and whose key stay.
                        const bool kbad = !(fabsf(kv4_scale(kp[r].x)) + fabsf(kv4_middle(kp[r].x)) + fabsf(kv4_scale(kp[r].y)) + fabsf(kv4_middle(kp[r].y)) < INFINITY);
                        const bool bad0 = kbad || !(fabsf(kv4_scale(vp[r].x)) + fabsf(kv4_middle(vp[r].x)) < INFINITY);
                        const bool bad1 = kbad || !(fabsf(kv4_scale(vp[r].y)) + fabsf(kv4_middle(vp[r].y)) < INFINITY);
                        if (bad0 || bad1) {
                            if (bad0) vp[r].x = 0u;
                            if (bad1) vp[r].y = 0u;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const f32x2 poison = pair(seen >> (4 * n + 2 * r) & 1 ? NAN : 0.f, seen >> (4 * n + 2 * r + 1) & 1 ? NAN : 0.f);
                                if (bad0) middle[n][0] = add2(middle[n][0], poison);
                                if (bad1) middle[n][1] = add2(middle[n][1], poison);
                                if (kbad) seen &= ~(3u << (4 * n + 2 * r));
                            }
                            if (kbad) kp[r] = make_uint2(0u, 0u);
                        }
                    }
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
                    load_words<D>(rec, lane, w);
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
                                for (int u = 0; u < TERMS; ++u) {
                                    const uint2 b = Q_IN_REGISTERS ? qf[Q_IN_REGISTERS ? k : 0] : q_fragment(u, k, n);
                                    mma_f16(s[k * 2 / STEPS][n], frag, b.x, b.y);
                                }
                        }
                    }
                }
                float x[NT][4], highest = -INFINITY;                                       // scores (of 2^x) less the running maximum
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const f32x2 s0 = pair(kv4_scale(kp[r].x), kv4_scale(kp[r].x)), s1 = pair(kv4_scale(kp[r].y), kv4_scale(kp[r].y));
                    const f32x2 m0 = pair(kv4_middle(kp[r].x), kv4_middle(kp[r].x)), m1 = pair(kv4_middle(kp[r].y), kv4_middle(kp[r].y));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const f32x2 v = fma2(pair(s[0][n][2 * r], s[0][n][2 * r + 1]), s0, fma2(pair(s[1][n][2 * r], s[1][n][2 * r + 1]), s1, fma2(m0, q_sum[n][0], mul2(m1, q_sum[n][1]))));
                        const float2 e = both(fma2(v, factor[n], minus[n]));
                        x[n][2 * r] = seen & (1u << (4 * n + 2 * r)) ? e.x : -INFINITY;
                        x[n][2 * r + 1] = seen & (2u << (4 * n + 2 * r)) ? e.y : -INFINITY;
                        highest = fmaxf(highest, fmaxf(x[n][2 * r], x[n][2 * r + 1]));
                    }
                }
                const float sv[2][2] = {{kv4_scale(vp[0].x), kv4_scale(vp[0].y)}, {kv4_scale(vp[1].x), kv4_scale(vp[1].y)}};
                const float largest = fmaxf(fmaxf(sv[0][0], sv[0][1]), fmaxf(sv[1][0], sv[1][1]));
                // ---- the running maximum may lie behind, and ``down`` fit smaller scales, so that both seldom move ----
                if (__any_sync(0xffffffffu, highest > kScoreLag<TERMS> || !(largest <= limit))) {
                    limit = INFINITY;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float2 old = both(minus[n]), was2 = both(down[n]);
                        float now[2], next[2], by[2], shrink[2];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float high = -INFINITY, most = 0.f;
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const bool there = seen & ((1u << c) << (4 * n + 2 * r));
                                high = fmaxf(high, x[n][2 * r + c]);
                                if (there) most = fmaxf(most, fmaxf(sv[r][0] < INFINITY ? sv[r][0] : 0.f, sv[r][1] < INFINITY ? sv[r][1] : 0.f));
                            }
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) {
                                high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, d));
                                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
                            }
                            // a column moves by its own keys alone, so that its neighbours' have no part in its rounding
                            const bool first = blank >> (2 * n + c) & 1, move = first || high > kScoreLag<TERMS>;
                            const float less = c ? old.y : old.x, was = c ? was2.y : was2.x;
                            now[c] = move ? high - less : -less;
                            by[c] = first ? 0.f : move ? fast_exp2(-less - now[c]) : 1.f;
                            if (now[c] > -INFINITY) blank &= ~(1u << (2 * n + c));
                            else now[c] = 0.f;
                            // 2^kUp over the power of two below the largest scale that the column has seen (0: none above 0)
                            constexpr float room = kScaleLag<TERMS> * (1 << kUp<TERMS>);
                            const float fit = most > 0.f ? power2(kUp<TERMS> - max(kUp<TERMS> - 120, min(120, (int)(__float_as_uint(most) >> 23) - 127))) : 0.f;
                            next[c] = was == 0.f || most > room * inverse_power2(was) ? fit : was;
                            shrink[c] = was > 0.f ? by[c] * (next[c] * inverse_power2(was)) : by[c];
                            limit = fminf(limit, blank >> (2 * n + c) & 1 ? -1.f : next[c] > 0.f ? room * inverse_power2(next[c]) : 0.f);
#pragma unroll
                            for (int r = 0; r < 2; ++r)
                                if (move) x[n][2 * r + c] = x[n][2 * r + c] - less - now[c];
                        }
                        const f32x2 b = pair(by[0], by[1]), z = pair(shrink[0], shrink[1]);
                        minus[n] = pair(-now[0], -now[1]);
                        down[n] = pair(next[0], next[1]);
                        sum[n] = mul2(sum[n], b);
                        middle[n][0] = mul2(middle[n][0], b);
                        middle[n][1] = mul2(middle[n][1], b);
#pragma unroll
                        for (int k = 0; k < STEPS; ++k)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const float2 y = both(mul2(pair(o[k][n][2 * r], o[k][n][2 * r + 1]), z));
                                o[k][n][2 * r] = y.x;
                                o[k][n][2 * r + 1] = y.y;
                            }
                    }
#pragma unroll
                    for (int d = 1; d < 4; d <<= 1) limit = fminf(limit, __shfl_xor_sync(0xffffffffu, limit, d));
                }
                // ---- weights, and weights times scales as the operand with tokens along K ----
                uint32_t pf[TERMS][2][NT][2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const f32x2 scale[2] = {pair(sv[r][0], sv[r][0]), pair(sv[r][1], sv[r][1])};
                    const f32x2 md[2] = {pair(kv4_middle(vp[r].x), kv4_middle(vp[r].x)), pair(kv4_middle(vp[r].y), kv4_middle(vp[r].y))};
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const f32x2 p = pair(fast_exp2(x[n][2 * r]), fast_exp2(x[n][2 * r + 1])), d = mul2(p, down[n]);
                        sum[n] = add2(sum[n], p);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float2 y = both(mul2(d, scale[h]));
                            middle[n][h] = fma2(p, md[h], middle[n][h]);
                            const uint32_t packed = pack_half2(y.x, y.y);
                            pf[0][h][n][r] = transpose8(packed);
                            if constexpr (TERMS == 2) {
                                const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&packed));
                                pf[TERMS - 1][h][n][r] = transpose8(pack_half2(y.x - back.x, y.y - back.y));
                            }
                        }
                    }
                }
                // ---- weighted values ----
                {
                    uint32_t w[E][2];
                    load_words<D>(rec + L::kSlice, lane, w);
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
                            for (int n = 0; n < NT; ++n) {
                                if constexpr (TERMS == 1) {
                                    mma_f16(o[k][n], frag, pf[0][k * 2 / STEPS][n][0], pf[0][k * 2 / STEPS][n][1]);
                                } else {
                                    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                                    for (int u = TERMS - 1; u >= 0; --u) mma_f16(part, frag, pf[u][k * 2 / STEPS][n][0], pf[u][k * 2 / STEPS][n][1]);
#pragma unroll
                                    for (int i = 0; i < 4; i += 2) {
                                        const float2 y = both(add2(pair(o[k][n][i], o[k][n][i + 1]), pair(part[i], part[i + 1])));
                                        o[k][n][i] = y.x;
                                        o[k][n][i + 1] = y.y;
                                    }
                                }
                            }
                        }
                    }
                }
            }
            __syncwarp();
        }

        // ---- a row, or the block's part of it, ends: the warps' parts become one, eight columns at a time ----
        const bool whole = first_page == 0 && stop == pages;
        // a part of a row that an earlier block began lies in the block's first place, one that goes on behind it in the second
        float* mine = part_of<D>(a, gridDim.x, blockIdx.x, first_page == 0, COLS);
        if (first_page == 0 && threadIdx.x == 0) {
            const bool by_row = few_rows(a, COLS, gridDim.x);
            if (!whole || by_row) {
                const int last = sm.prefix[index] + ((int)in_tile + 1) * (EXTRA + pages) - 1;
                const int last_block = whole ? -1 : sm.last_block >= 0 ? sm.last_block : block_of(shares_of(sm.prefix[a.n_tiles], GROUPS, gridDim.x), last);
                const int place = by_row ? index * rows_of_tile(a, COLS) + (int)in_tile : (int)blockIdx.x;
                *reinterpret_cast<CutRow*>(a.scratch + (int64_t)place * kHeadInts) = CutRow{(int)blockIdx.x, last_block, row, part, head, columns};
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float2 m = both(minus[n]), d = both(down[n]);
            f32x2 l = sum[n], mid[2] = {middle[n][0], middle[n][1]};
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) {
                l = add2(l, __shfl_xor_sync(0xffffffffu, l, i));
                mid[0] = add2(mid[0], __shfl_xor_sync(0xffffffffu, mid[0], i));
                mid[1] = add2(mid[1], __shfl_xor_sync(0xffffffffu, mid[1], i));
            }
            if (g == 0) {
                const int c = 8 * n + 2 * j;
                *reinterpret_cast<float2*>(&sm.merge_m[warp][c]) = make_float2(blank >> (2 * n) & 1 ? -INFINITY : -m.x, blank >> (2 * n + 1) & 1 ? -INFINITY : -m.y);
                *reinterpret_cast<float2*>(&sm.merge_up[warp][c]) = make_float2(d.x > 0.f ? inverse_power2(d.x) : 0.f, d.y > 0.f ? inverse_power2(d.y) : 0.f);
                *reinterpret_cast<float2*>(&sm.merge_l[warp][c]) = both(l);
                *reinterpret_cast<float2*>(&sm.merge_mid[0][warp][c]) = both(mid[0]);
                *reinterpret_cast<float2*>(&sm.merge_mid[1][warp][c]) = both(mid[1]);
            }
#pragma unroll
            for (int k = 0; k < STEPS; ++k)
                *reinterpret_cast<float4*>(sm.merge[warp][n][k][lane]) = make_float4(o[k][n][0], o[k][n][1], o[k][n][2], o[k][n][3]);
        }
        __syncthreads();
#pragma unroll 1
        for (int c = warp; c < columns; c += WARPS) {                                   // a warp to a column, a lane to a warp's part of it
            const bool there = lane < WARPS;
            const int w = lane % WARPS;
            const float m = there ? sm.merge_m[w][c] : -INFINITY, high = warp_max(m), by = m > -INFINITY ? fast_exp2(m - high) : 0.f;
            const float l = warp_sum(there ? sm.merge_l[w][c] * by : 0.f);
            const float mid0 = warp_sum(there ? sm.merge_mid[0][w][c] * by : 0.f), mid1 = warp_sum(there ? sm.merge_mid[1][w][c] * by : 0.f);
            if (there) sm.merge_up[w][c] *= by;
            if (lane == 0) {
                sm.end_m[c] = high;
                sm.end_l[c] = l;
                sm.end_mid[0][c] = mid0;
                sm.end_mid[1][c] = mid1;
            }
        }
        __syncthreads();
#pragma unroll 1
        for (int i = threadIdx.x; i < NT * D * 2; i += 32 * WARPS) {                     // two channels of two columns
            const int n = i / (2 * D), k = i / 32 % STEPS, c = 8 * n + 2 * (i & 3), channel = 16 * k + 2 * (i >> 2 & 7);
            f32x2 y0 = *reinterpret_cast<const f32x2*>(&sm.end_mid[k * 2 / STEPS][c]), y1 = y0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(sm.merge[w][n][k][i & 31]);
                const f32x2 up = *reinterpret_cast<const f32x2*>(&sm.merge_up[w][c]);
                y0 = fma2(x.x, up, y0);
                y1 = fma2(x.y, up, y1);
            }
            const float2 even = both(y0), odd = both(y1);                                // (channel, columns c and c + 1; channel + 1)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (c + e >= columns) break;
                const float lo = e ? even.y : even.x, hi = e ? odd.y : odd.x, l = sm.end_l[c + e];
                if (whole) {
                    const int q = part * COLS + c + e, token = sm.last[c + e] - t.first_pos;
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    store2(reinterpret_cast<T*>(a.out) + ((int64_t)(row + token) * a.n_heads + head * a.group + q - token * a.group) * D + channel, lo * inv, hi * inv);
                } else {
                    float* p = mine + (int64_t)(c + e) * kPartStride<D>;
                    *reinterpret_cast<float2*>(p + channel) = make_float2(lo, hi);
                    if (channel == 0) *reinterpret_cast<float2*>(p + D) = make_float2(sm.end_m[c + e], l);
                }
            }
        }
        __syncthreads();
    }
}

// Adds up the parts of the rows that were cut, one block per row and column; blockIdx.y is the place of the row's head.  A warp has five of its parts
// under way at a time, so that the half of 148 blocks' parts are one round of loads.
constexpr int kCombineWarps = 16, kCombineParts = 5;
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kCombineWarps * 32)
kv4_combine_kernel(const __grid_constant__ AttendArgs a, int blocks) {
    constexpr int COLS = 8 * NT, E = D / 32, STRIDE = COLS * kPartStride<D>;
    __shared__ float tops[kCombineWarps], sums[kCombineWarps], values[kCombineWarps][D];
    pdl_launch_dependents();
    pdl_wait();
    const CutRow cut = *reinterpret_cast<const CutRow*>(a.scratch + (int64_t)blockIdx.y * kHeadInts);
    const int c = blockIdx.x, b0 = cut.first_block, last = cut.last_block;
    if (last < 0 || c >= cut.columns) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* parts = part_of<D>(a, blocks, 0, false, COLS) + c * kPartStride<D>;
    float top = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = 0.f;
#pragma unroll 1
    for (int b = b0 + warp; b <= last; b += kCombineWarps * kCombineParts) {
        float v[kCombineParts][E];
        float2 ml[kCombineParts];
#pragma unroll
        for (int u = 0; u < kCombineParts; ++u) {
            const int x = b + u * kCombineWarps, y = min(x, last);
            const float* p = parts + (2 * y + (y == b0)) * STRIDE;
            ml[u] = *reinterpret_cast<const float2*>(p + D);
            if (x > last) ml[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int i = 0; i < E; ++i) v[u][i] = p[lane + 32 * i];
        }
        float now = top;
#pragma unroll
        for (int u = 0; u < kCombineParts; ++u) now = fmaxf(now, ml[u].x);
        const float back = top > -INFINITY ? exp2f(top - now) : 0.f;
        top = now;
        l *= back;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] *= back;
#pragma unroll
        for (int u = 0; u < kCombineParts; ++u) {
            const float by = ml[u].x > -INFINITY ? exp2f(ml[u].x - now) : 0.f;
            l += ml[u].y * by;
#pragma unroll
            for (int i = 0; i < E; ++i) o[i] += b + u * kCombineWarps <= last ? v[u][i] * by : 0.f;
        }
    }
    if (lane == 0) {
        tops[warp] = top;
        sums[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) values[warp][lane + 32 * i] = o[i];
    __syncthreads();
    if (warp >= E) return;
    const bool there = lane < kCombineWarps;
    const float m = there ? tops[lane % kCombineWarps] : -INFINITY, high = warp_max(m), by = m > -INFINITY ? exp2f(m - high) : 0.f;
    const float total = warp_sum(there ? sums[lane % kCombineWarps] * by : 0.f), inv = total > 0.f ? 1.f / total : 0.f;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kCombineWarps; ++w) v += values[w][32 * warp + lane] * __shfl_sync(0xffffffffu, by, w);
    const int q = cut.part * COLS + c, token = quotient(q, a.per_group);
    reinterpret_cast<T*>(a.out)[((int64_t)(cut.row + token) * a.n_heads + cut.head * a.group + q - token * a.group) * D + 32 * warp + lane] = from_f32<T>(v * inv);
}

template <typename T, int D, int NT, int TERMS>
int attend(const AttendArgs& a, cudaStream_t stream) {
    static bool done[kMaxDevices];
    constexpr int bytes = (int)sizeof(Smem<D, NT, TERMS>);
    static_assert(bytes <= 227 * 1024, "a block's shared memory");
    const int status = ensure_dynamic_smem(kv4_attention_kernel<T, D, NT, TERMS>, bytes, done);
    if (status != CPM_OK) return status;
    const int sms = device_sms();
    if (sms <= 0) return CPM_BAD_ARGUMENT;
    const int blocks = sms;
    cpm_launch(kLaunchAttention, kv4_attention_kernel<T, D, NT, TERMS>, dim3(blocks), 32 * warps_of(D, NT, TERMS), bytes, stream, a);
    const int heads = few_rows(a, 8 * NT, blocks) ? a.n_tiles * rows_of_tile(a, 8 * NT) : blocks;
    cpm_launch(kLaunchAttention, kv4_combine_kernel<T, D, NT>, dim3(8 * NT, heads), kCombineWarps * 32, 0, stream, a, blocks);
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
    return (int64_t)device_sms() * (kHeadInts + 2 * 16 * (d + 4));
}
CPM_API int cpm_kv4_attention_most_tiles() { return kMostTiles; }
CPM_API int cpm_kv4_attention(const void* q, const void* records, void* out, const int* kv_len, const int* slots, const int* page_table,
                              int max_pages, const int* cu_q, const int* tile_seq, const int* tile_row, int n_tiles, float* scratch, int n_heads,
                              int n_kv, int d, int window, float scale, int dtype, cudaStream_t stream) {
    if (n_tiles <= 0) return CPM_OK;
    if (n_tiles > kMostTiles || n_heads < 1 || n_heads > 8192 || n_kv < 1 || n_heads % n_kv || window < 0) return CPM_BAD_ARGUMENT;
    if ((cu_q == nullptr) != (tile_seq == nullptr) || (cu_q == nullptr) != (tile_row == nullptr)) return CPM_BAD_ARGUMENT;
    if (((uintptr_t)records | (uintptr_t)q | (uintptr_t)out) & 15) return CPM_BAD_ARGUMENT;
    const AttendArgs a{q, out, (const uint8_t*)records, kv_len, slots, page_table, cu_q, tile_seq, tile_row, scratch, max_pages, n_tiles, n_heads, n_kv,
                       n_heads / n_kv, window, scale, (float)n_kv / (float)n_heads, 1.f / (float)n_kv};
    return dtype == CPM_BF16 ? by_head_size<bf16, 1>(a, d, stream) : by_head_size<float, 2>(a, d, stream);
}
