// Drawing a token under a temperature, top-k, top-p and min-p from one given number a row.
//
//     w_i = exp((z_i - max z) / T)                      fp32; held as W_i = floor(w_i 2^40), a whole number
//     tokens stand by w from large to small, equal ones by index; of these stay
//         the first k                                   (top_k > 0)
//         of them as many as first reach  p * (their mass)     (top_p < 1)
//         and those with  w_i >= min_p                  (min_p > 0; the largest w is 1)
//     token = the first, by index, whose running sum over the kept W exceeds  floor(u * kept mass)
//     log-probability = (z_token - max z) / T - log(kept mass / 2^40)
//
// Sums are whole numbers, so they do not depend on the order in which thousands of threads form them: the same row and number give the same
// token whatever the launch.  (With fp32 sums the border between two of 70,000 tokens moves by more than their distance.)
//
// A row is read once.  Its weights lie in the shared memory of a cluster of blocks (one to eight; the fewer rows, the more blocks a row).  One
// histogram of the weights' upper bits (32 bins to an octave) holds each bin's number of tokens and, where mass decides, the sum of their lower bits: so the
// bin in which the k-th token lies, or at which the mass is reached, is known exactly.  The tokens in that bin, a few hundred, go to the cluster's first
// block, which finds the border by radix selection; where no more than kRanked tokens are in or above the bin of top-k, all of them go there, each is
// compared with each, and it draws as well.  In the same pass a thread sums what it keeps above the bin, so that the draw looks at few tokens again.
// (A cluster's barrier takes about 2 us, and a look into a neighbour's shared memory half of that: a selection over the whole row with
// all blocks' histograms added up at every step took 41 us for one row of 73,448, bins of counts alone 25, and this 15.)
// 64 rows of 73,448 with settings of their own 38 us, 512 rows of 32,000 by mass alone 117.  What a row cannot do without is its logits, 4 bytes a token
// (10 us of the 117); the instructions bound it, some hundred a token, and the phases in which a cluster's blocks wait for the first.
#include "common.cuh"
#include "philox.cuh"

namespace {

constexpr int kFilterThreads = 512;
constexpr int kFilterWarps = kFilterThreads / 32;
constexpr int kMostBlocks = 8;                         // of a cluster
constexpr int kOctaveBits = 18;                        // bits of a weight below those that number its bin
constexpr int kCoarseBins = 1536;                      // 48 octaves down from 1; what is smaller (less than 2^-40 has no mass) lies in bin 0
constexpr int kFirstBin = (0x3f800000 >> kOctaveBits) + 1 - kCoarseBins;
constexpr int kOwnBins = kCoarseBins / kFilterThreads;
constexpr uint32_t kWhole = 110u << 23;                // bits of 2^-17: from here up a weight times 2^40 is a whole number as it is
constexpr int kFineBins = 1024;                        // of a step of the selection
constexpr int kListed = 2048;                          // tokens that are set apart for the selection
constexpr int kRanked = 256;                           // up to so many the first block compares each with each, and draws without the others
constexpr int kLimbBits = 14;                          // a mass is added in three limbs: 32-bit adds in shared memory are one instruction
constexpr int kMostVocab = 1 << 21;                    // so that a limb's sum over the tokens of a block, an eighth of them, stays within 32 bits

struct FilterArgs {
    const float* logits;
    int64_t ld;
    int vocab, per_block;
    const float *uniform, *temperature, *top_p, *min_p;
    const int *top_k, *seq_key, *step_key, *drawn;
    uint64_t seed;
    int* token;
    float* logprob;
};

// What the first block has found and the others read: the weights to set apart, or the border.
struct Plan {
    uint32_t low, high;                                // bits of the weights to set apart
    int complete;                                      // all from ``low`` up are
    int known;                                         // whether the mass above ``high`` is
    int apart;                                         // whether they are few enough, else their masses go into bins
    uint32_t border;                                   // tokens above it stay, and the first ``ties`` of the ``equal`` ones at it
    uint64_t ties, equal;
};

struct FilterShared {
    alignas(16) uint32_t coarse[kCoarseBins];          // tokens of the row in each bin (in the first block)
    union {
        alignas(16) uint32_t fine[3][kFineBins];
        uint32_t low[2][kCoarseBins];                  // before that: the sums of their weights' bits below the bin's number, by 16 bits
    };
    union {
        struct {
            uint32_t list[kListed];                    // bits of the weights that are set apart, in the first block
            int place[kListed];                        // and their tokens
        };
        alignas(8) uint64_t joined[kFineBins];         // where they are too many: what the other blocks have in each fine bin, in the first block
        uint32_t own[2][kCoarseBins];                  // before that: the block's bins, see count_own
    };
    int listed;
    uint64_t warp_sum[kFilterWarps + 1], warp_sums[3][kFilterWarps + 1];
    uint64_t found_before, found_here;                 // what lies above the bin that was found, and in it
    int found_bin, low_bin, high_bin, cut;
    alignas(8) ArgMax best[kMostBlocks];                          // of the cluster's blocks, which write here
    uint64_t mass[kMostBlocks];
    int count[kMostBlocks];
    Plan plan;
    ArgMax scratch[33];
};

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
__device__ __forceinline__ uint32_t add32(const void* own, uint32_t rank, uint32_t v) {
    uint32_t old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(cluster_address(own, rank)), "r"(v) : "memory");
    return old;
}

// floor(w 2^40) of a weight (0 to 1) by its bits: 24 bits of significand, shifted.
__device__ __forceinline__ uint64_t units_of(uint32_t bits) {
    return ((uint64_t)((bits & 0x7fffffu) | 0x800000u) << 17) >> min(63u, 127u - (bits >> 23));
}

// Of a weight below 2^-17.
__device__ __forceinline__ uint32_t small_units_of(uint32_t bits) {
    return bits < kWhole ? ((bits & 0x7fffffu) | 0x800000u) >> min(31u, 110u - (bits >> 23)) : 0u;
}
__device__ __forceinline__ int bin_of(uint32_t bits) { return max(0, (int)(bits >> kOctaveBits) - kFirstBin); }
__device__ __forceinline__ uint32_t bin_begin(int bin) { return bin > 0 ? (uint32_t)(bin + kFirstBin) << kOctaveBits : 0u; }

// A block's bins: own[1] holds the number of tokens, 15 bits, above the sum of the upper 2 of the 18 bits below a bin's number, own[0] the sum of all 18
// modulo 2^32; with less than 2^15 tokens the one tells how often the other has run over.  Without staged weights: the number alone.
constexpr int kCountBits = 17;
template <bool STAGED>
__device__ __forceinline__ void count_own(FilterShared& sm, uint32_t bits, bool masses) {
    const int bin = bin_of(bits);
    if constexpr (STAGED) {
        atomicAdd(&sm.own[1][bin], 1u << kCountBits | (bits >> (kOctaveBits - 2) & 3u));
        if (masses) atomicAdd(&sm.own[0][bin], bits & ((1u << kOctaveBits) - 1));
    } else {
        atomicAdd(&sm.own[1][bin], 1u);
    }
}
// Adds them to the row's, in the first block.
template <bool STAGED>
__device__ __forceinline__ void add_own(FilterShared& sm, bool masses) {
#pragma unroll 1
    for (int bin = threadIdx.x; bin < kCoarseBins; bin += kFilterThreads) {
        const uint32_t packed = sm.own[1][bin];
        if (!packed) continue;
        add32(&sm.coarse[bin], 0, STAGED ? packed >> kCountBits : packed);
        if (STAGED && masses) {
            const uint64_t least = (uint64_t)(packed & ((1u << kCountBits) - 1)) << (kOctaveBits - 2);
            const uint64_t sum = least + (uint32_t)(sm.own[0][bin] - (uint32_t)least);
            add32(&sm.low[0][bin], 0, (uint32_t)sum & 0xffffu);
            add32(&sm.low[1][bin], 0, (uint32_t)(sum >> 16));
        }
    }
}
// The mass of a bin: exact where its weights' bits have been summed and it lies above 2^-17, else a bound from above or below.
__device__ __forceinline__ uint64_t bin_mass(const FilterShared& sm, int bin, bool summed, bool upper) {
    if (bin == 0) return 0;
    const uint64_t n = sm.coarse[bin], low = summed ? sm.low[0][bin] + ((uint64_t)sm.low[1][bin] << 16) : upper ? n * ((1u << kOctaveBits) - 1) : 0;
    const uint32_t begin = bin_begin(bin);
    const uint64_t v = (n * ((begin & 0x7fffffu) | 0x800000u) + low) << 17 >> (127u - (begin >> 23));
    return upper || begin >= kWhole ? v : v - min(v, n);
}

// Inclusive sums over the block's threads in order; the block's total is left in the last of ``sums``.
__device__ __noinline__ uint64_t block_scan64(uint64_t v, uint64_t* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
        const uint64_t own = lane < kFilterWarps ? sums[lane] : 0;
        uint64_t x = own;
#pragma unroll
        for (int o = 1; o < kFilterWarps; o <<= 1) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncwarp();
        if (lane < kFilterWarps) sums[lane] = x - own;
        if (lane == kFilterWarps - 1) sums[kFilterWarps] = x;
    }
    __syncthreads();
    return v + sums[warp];
}
// The same of three numbers at once.
__device__ __forceinline__ void block_scan64(uint64_t (&v)[3], uint64_t (*sums)[kFilterWarps + 1]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            const uint64_t x = __shfl_up_sync(0xffffffffu, v[n], o);
            if (lane >= o) v[n] += x;
        }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 3; ++n)
        if (lane == 31) sums[n][warp] = v[n];
    __syncthreads();
    if (warp < 3) {
        const uint64_t own = lane < kFilterWarps ? sums[warp][lane] : 0;
        uint64_t x = own;
#pragma unroll
        for (int o = 1; o < kFilterWarps; o <<= 1) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncwarp();
        if (lane < kFilterWarps) sums[warp][lane] = x - own;
        if (lane == kFilterWarps - 1) sums[warp][kFilterWarps] = x;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 3; ++n) v[n] += sums[n][warp];
}
__device__ __forceinline__ uint64_t block_sum64(uint64_t v, FilterShared& sm) {
    block_scan64(v, sm.warp_sum);
    return sm.warp_sum[kFilterWarps];
}

// STAGED: the block's weights lie in shared memory; else (a vocabulary that eight blocks' do not hold) they are formed again from the logits.
template <bool STAGED>
struct Row {
    const float* z;                                    // the block's first logit
    float* w;
    int n;                                             // tokens of the block
    float top, t;
    float inverse;                                     // 1 / t where the quotient by it is exact, else 0
    // (x - top) / t correctly rounded.  For t within 2^60 of 1 by Markstein's method (IBM J. Res. Dev. 34, 1990): with r = 1 / t rounded, q = x r, and
    // the remainder x - q t, which a fused multiply-add gives exactly, q + r (x - q t) rounds to the quotient.  Where it overflows the weight is 0.
    __device__ __forceinline__ float over_t(float x) const {
        if (inverse == 0.f) return __fdiv_rn(x, t);
        const float q = __fmul_rn(x, inverse);
        return __fmaf_rn(__fmaf_rn(-q, t, x), inverse, q);
    }
    __device__ __forceinline__ float form(float x) const {
        if (top == INFINITY) return x == INFINITY ? 1.f : 0.f;
        const float v = expf(over_t(__fsub_rn(x, top)));
        return v >= 0.f ? v : 0.f;                     // a logit that is no number is never drawn
    }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (STAGED) return w[i];
        else return form(z[i]);
    }
};

struct Border { uint32_t bits; uint64_t above, here; };      // a weight, and the count or mass of the tokens above it and at it

// What the block has in a fine bin.
__device__ __forceinline__ uint64_t own_fine(const FilterShared& sm, int bin) {
    uint64_t v = 0;
#pragma unroll
    for (int u = 0; u < 3; ++u) v += (uint64_t)sm.fine[u][bin] << (u * kLimbBits);
    return v;
}
// The bin of sm.fine, counts or masses in limbs, at which the running sum from the last bin down, starting with ``above``, first reaches ``need``: left in
// sm.found_bin, with what lies above it and in it.  ``joined``: with the other blocks' in sm.joined.  Exactly one bin is found, whatever the sums: the last
// one looked at needs not reach ``need``, and the first may be reached before it.
__device__ __noinline__ void find_fine(FilterShared& sm, double need, uint64_t above, bool joined) {
    const int bin = kFineBins - 2 - 2 * threadIdx.x;    // two bins a thread
    uint64_t v[2] = {own_fine(sm, bin + 1), own_fine(sm, bin)};
    if (joined) {
        v[0] += sm.joined[bin + 1];
        v[1] += sm.joined[bin];
    }
    uint64_t upto = above + block_scan64(v[0] + v[1], sm.warp_sum) - v[0] - v[1];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool first = bin + 1 - i == kFineBins - 1, last = bin + 1 - i == 0;
        if ((first || (double)upto < need) && (last || (double)(upto + v[i]) >= need)) {
            sm.found_bin = bin + 1 - i;
            sm.found_before = upto;
            sm.found_here = v[i];
        }
        upto += v[i];
    }
    __syncthreads();
}
__device__ __forceinline__ void clear_fine(FilterShared& sm) {
#pragma unroll 1
    for (int i = threadIdx.x; i < 3 * kFineBins; i += kFilterThreads) sm.fine[0][i] = 0;
    __syncthreads();
}
__device__ __forceinline__ void add_fine(FilterShared& sm, bool mass, int bin, uint32_t bits) {
    if (!mass) {
        atomicAdd(&sm.fine[0][bin], 1u);
        return;
    }
    const uint64_t v = units_of(bits);
    atomicAdd(&sm.fine[0][bin], (uint32_t)v & ((1u << kLimbBits) - 1));
    atomicAdd(&sm.fine[1][bin], (uint32_t)(v >> kLimbBits) & ((1u << kLimbBits) - 1));
    atomicAdd(&sm.fine[2][bin], (uint32_t)(v >> (2 * kLimbBits)));
}
__device__ __forceinline__ int bits_of_range(uint32_t low, uint32_t high) { return max(1, 32 - __clz(high - low - 1)); }

// The weight at which the running count (``mass`` false) or mass of the listed tokens, from the largest weight down, first reaches ``need``.  Looked at are
// the weights of [low, high), which are known to hold it; ``above``: what lies above them.  By the first block alone.
__device__ __noinline__ Border select(FilterShared& sm, bool mass, int listed, double need, uint64_t above, uint32_t low, uint32_t high) {
    uint32_t prefix = 0;
    int done = bits_of_range(low, high);                // key bits from here up are the prefix
#pragma unroll 1
    while (done > 0) {
        const int shift = max(0, done - 10);
        clear_fine(sm);
#pragma unroll 1
        for (int i = threadIdx.x; i < listed; i += kFilterThreads) {
            const uint32_t bits = sm.list[i], key = bits - low;
            if (bits >= low && bits < high && (key >> done) == prefix) add_fine(sm, mass, (key >> shift) & ((1u << (done - shift)) - 1), bits);
        }
        __syncthreads();
        find_fine(sm, need, above, false);
        prefix = (prefix << (done - shift)) | sm.found_bin;
        above = sm.found_before;
        done = shift;
    }
    return Border{low + prefix, above, sm.found_here};
}

// The bin, from the largest weights down, at whose end the number of tokens reaches ``need``: left in sm.found_bin, with the number before it.
__device__ __forceinline__ void find_count(FilterShared& sm, double need) {
    const int top_bin = kCoarseBins - 1 - kOwnBins * threadIdx.x;
    uint64_t here[kOwnBins], sum = 0;
#pragma unroll
    for (int q = 0; q < kOwnBins; ++q) sum += here[q] = sm.coarse[top_bin - q];
    uint64_t upto = block_scan64(sum, sm.warp_sum) - sum;
#pragma unroll
    for (int q = 0; q < kOwnBins; ++q) {
        if ((double)upto < need && (double)(upto + here[q]) >= need) {
            sm.found_bin = top_bin - q;
            sm.found_before = upto;
        }
        upto += here[q];
    }
    __syncthreads();
}
// The bins at whose ends the masses reach ``p`` times all, by their bounds from above (sm.high_bin) and from below (sm.low_bin, with what lies before it in
// sm.found_before): no bin between them can be ruled out.  ``within``: all, or, where the bins' masses are summed, what they do not tell exactly; returned is all.
__device__ __forceinline__ uint64_t find_mass(FilterShared& sm, bool summed, float p, uint64_t within, int last) {
    const int top_bin = kCoarseBins - 1 - kOwnBins * threadIdx.x;
    uint64_t here[2][kOwnBins], v[3] = {0, 0, 0}, sum[2];
#pragma unroll
    for (int q = 0; q < kOwnBins; ++q) {
        v[0] += here[0][q] = bin_mass(sm, top_bin - q, summed, true);
        v[1] += here[1][q] = bin_mass(sm, top_bin - q, summed, false);
        if (summed && bin_begin(top_bin - q) >= kWhole) v[2] += here[1][q];
    }
    sum[0] = v[0];
    sum[1] = v[1];
    if (threadIdx.x == 0) {
        sm.high_bin = kCoarseBins - 1;
        sm.low_bin = last;
    }
    block_scan64(v, sm.warp_sums);
    within += sm.warp_sums[2][kFilterWarps];
    const double need = (double)p * (double)within;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        uint64_t upto = v[n] - sum[n];
#pragma unroll
        for (int q = 0; q < kOwnBins; ++q) {
            if ((double)upto < need && (double)(upto + here[n][q]) >= need) {
                if (n == 0) sm.high_bin = top_bin - q;
                else {
                    sm.low_bin = top_bin - q;
                    sm.found_before = upto;
                }
            }
            upto += here[n][q];
        }
    }
    __syncthreads();
    return within;
}

// Of the tokens at a border that mass decides, how many it takes.
__device__ __forceinline__ uint64_t ties_of(const Border& b, double need, uint64_t* equal) {
    const uint64_t each = max((uint64_t)1, units_of(b.bits)), there = b.here / each;
    uint64_t n = (uint64_t)ceil((need - (double)b.above) / (double)each);
    n = min(max(n, (uint64_t)1), there);
    while (n > 1 && (double)(b.above + (n - 1) * each) >= need) --n;
    while (n < there && (double)(b.above + n * each) < need) ++n;
    *equal = there;
    return n;
}

template <bool STAGED>
__global__ void __launch_bounds__(kFilterThreads, 2)
sample_filtered_kernel(const __grid_constant__ FilterArgs a) {
    extern __shared__ float weights[];
    __shared__ FilterShared sm;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t blocks = cluster_blocks(), rank = cluster_rank();
    const int r = blockIdx.x / blocks, tid = threadIdx.x, lane = tid & 31;
    if (a.drawn && !a.drawn[r]) {                               // another's row (its whole cluster leaves)
        if (rank == 0 && tid == 0) a.logprob[r] = NAN;
        return;
    }
    const int first = min(a.vocab, (int)rank * a.per_block);
    Row<STAGED> row;
    row.n = min(a.vocab, first + a.per_block) - first;
    row.z = a.logits + (int64_t)r * a.ld + first;
    row.w = weights;
    const float t = a.temperature ? a.temperature[r] : 0.f, p = a.top_p ? a.top_p[r] : 1.f;
    int k = a.top_k ? a.top_k[r] : 0;
    float ratio = a.min_p ? a.min_p[r] : 0.f;
    if (p <= 0.f || ratio > 1.f) k = 1;
    // above one: the first token alone, which it would leave out as well; below zero, -0 (weights are compared by their bits) or no number: no limit
    if (!(ratio > 0.f && ratio <= 1.f)) ratio = 0.f;
    const bool by_count = k > 0 && k < a.vocab, by_mass = p < 1.f && p > 0.f && k != 1;
    const float u = a.uniform ? a.uniform[r] : philox_uniform(a.seed, (uint32_t)a.seq_key[r], (uint32_t)a.step_key[r]);

    asm volatile("barrier.cluster.arrive;" ::: "memory");       // (nothing is put into a block that has not begun)

    // the largest logit, lowest index among equals
    ArgMax best{-INFINITY, 0x7fffffff};
    const int whole = ((uintptr_t)row.z & 15) == 0 ? row.n & ~3 : 0;
#pragma unroll 1
    for (int i0 = 4 * tid; i0 < whole; i0 += 16 * kFilterThreads) {
        float4 v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = i0 + 4 * q * kFilterThreads;
            v[q] = i < whole ? *reinterpret_cast<const float4*>(row.z + i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int i = i0 + 4 * q * kFilterThreads;
            if (i >= whole) break;
            if constexpr (STAGED) *reinterpret_cast<float4*>(weights + i) = v[q];
            if (v[q].x > best.v) best = ArgMax{v[q].x, first + i};       // (a thread's tokens come by index)
            if (v[q].y > best.v) best = ArgMax{v[q].y, first + i + 1};
            if (v[q].z > best.v) best = ArgMax{v[q].z, first + i + 2};
            if (v[q].w > best.v) best = ArgMax{v[q].w, first + i + 3};
        }
    }
#pragma unroll 1
    for (int i = whole + tid; i < row.n; i += kFilterThreads) {
        const float v = row.z[i];
        if constexpr (STAGED) weights[i] = v;
        if (v > best.v) best = ArgMax{v, first + i};
    }
    if (by_count || by_mass)
#pragma unroll 1
        for (int i = tid; i < kCoarseBins; i += kFilterThreads) sm.coarse[i] = sm.low[0][i] = sm.low[1][i] = sm.own[0][i] = sm.own[1][i] = 0;
    if (tid == 0) sm.listed = 0;
    best = block_argmax(best, sm.scratch);
    asm volatile("barrier.cluster.wait;" ::: "memory");
    if (tid < (int)blocks) put64(&sm.best[rank], tid, (uint64_t)__float_as_uint(best.v) | (uint64_t)(uint32_t)best.i << 32);
    cluster_sync();
    best = ArgMax{-INFINITY, 0x7fffffff};
#pragma unroll 1
    for (uint32_t b = 0; b < blocks; ++b) best = better(best, sm.best[b]);
    if (best.v == -INFINITY || !(t > 0.f)) {                   // nothing that can be drawn: token 0; a greedy row: the largest
        if (rank == 0 && tid == 0) {
            a.token[r] = best.v == -INFINITY ? 0 : best.i;
            a.logprob[r] = best.v == -INFINITY ? -INFINITY : 0.f;
        }
        return;
    }
    row.top = best.v;
    row.t = t;
    row.inverse = t > 0x1p-60f && t < 0x1p60f ? __frcp_rn(t) : 0.f;

    // weights, their histogram, and (where mass alone decides) their mass.  A thread's tokens are neighbours, an odd number of them, so that sums by
    // thread go by index and a warp's accesses to shared memory are in different banks
    const int strip = (row.n + kFilterThreads - 1) / kFilterThreads | 1, i0 = min(row.n, tid * strip), i1 = min(row.n, i0 + strip);
    const bool summed = STAGED && by_mass && !by_count;        // whether the bins' masses are
    uint64_t own_mass = 0;                                     // of the thread's tokens that bins do not tell exactly
    if (by_count || by_mass) {
        uint32_t small = 0;
#pragma unroll 4
        for (int i = i0; i < i1; ++i) {
            const float w = STAGED ? row.form(weights[i]) : row.at(i);
            if constexpr (STAGED) weights[i] = w;
            count_own<STAGED>(sm, __float_as_uint(w), summed);
            if (summed) small += small_units_of(__float_as_uint(w));
            else if (!STAGED && !by_count) own_mass += units_of(__float_as_uint(w));
        }
        own_mass += small;
    } else if constexpr (STAGED) {
#pragma unroll 2
        for (int i = i0; i < i1; ++i) weights[i] = row.form(weights[i]);
    }
    __syncthreads();
    const auto put_mass = [&](uint64_t own) {                  // the block's sum into the first block's (or every block's) list of sums
        const uint64_t all = block_sum64(own, sm);
        if (tid < (int)blocks) put64(&sm.mass[rank], tid, all);
    };
    const auto all_mass = [&]() {
        uint64_t all = 0;
#pragma unroll 1
        for (uint32_t b = 0; b < blocks; ++b) all += sm.mass[b];
        return all;
    };

    uint32_t border = 0;
    uint64_t ties = ~0ull, equal = 0;
    // of the thread's tokens, those that were set apart (the last one in the lowest bit), and the mass above them; ``sure``: these two tell what it keeps
    uint64_t found = 0, sure_mass = 0;
    bool sure = false;
    const auto each_found = [&](auto&& visit) {
#pragma unroll 1
        for (uint64_t left = found; left;) {
            const int bit = 63 - __clzll(left);
            left &= ~(1ull << bit);
            visit(i1 - 1 - bit);
        }
    };
    if (by_count || by_mass) {
        if (by_mass && !by_count) put_mass(own_mass);
        add_own<STAGED>(sm, summed);
        cluster_sync();
        uint64_t within = by_mass && !by_count ? all_mass() : 0;      // mass of the tokens that top-k leaves (known to the first block alone, unless by_count)
#pragma unroll 1
        for (int round = by_count ? 0 : 1; round < (by_mass ? 2 : 1); ++round) {
            // ---- which weights the border may be among ----
            double need = (double)k;
            const bool last_round = round == (by_mass ? 1 : 0);
            uint64_t above = 0;                                // what lies above them (known to the first block alone)
            uint64_t some = 0;                                 // no fewer tokens than they are (likewise)
            uint32_t low = 0, high = 0, complete = 0;
            bool known = round == 0;                           // whether ``above`` is
            if (rank == 0) {
                if (round == 0) {
                    find_count(sm, need);
                    above = sm.found_before;
                    low = bin_begin(sm.found_bin);
                    some = sm.coarse[sm.found_bin];
                    complete = above + some <= kListed;
                    high = complete ? 0x3f800001u : bin_begin(sm.found_bin + 1);
                } else {
                    // from where the masses reach ``need`` by their bounds from above, to where they do by those from below
                    const int last = bin_of(border);
                    within = find_mass(sm, summed, p, within, last);
                    need = (double)p * (double)within;
                    const int low_bin = max(sm.low_bin, last), high_bin = max(sm.high_bin, low_bin);
                    low = max(border, bin_begin(low_bin));
                    high = bin_begin(high_bin + 1);
                    if (summed && bin_begin(low_bin) >= kWhole) {      // exact so far
                        above = sm.found_before;
                        known = true;
                    }
                    some = sm.coarse[low_bin];
                    if (low_bin < high_bin) {
                        uint64_t count = 0;
                        for (int bin = low_bin + tid; bin <= high_bin; bin += kFilterThreads) count += sm.coarse[bin];
                        some = block_sum64(count, sm);
                    }
                }
            }
            Border b{};
            int listed = 0;
#pragma unroll 1
            while (true) {
                if (rank == 0) {
                    if (some > kListed) {
#pragma unroll 1
                        for (int i = tid; i < kFineBins; i += kFilterThreads) sm.joined[i] = 0;
                        clear_fine(sm);
                    }
                    if (tid == 0) {
                        sm.plan.low = low;
                        sm.plan.high = high;
                        sm.plan.complete = complete;
                        sm.plan.known = known;
                        sm.plan.apart = some <= kListed;
                        sm.listed = 0;
                    }
                }
                cluster_sync();
                low = peer32(&sm.plan.low, 0);
                high = peer32(&sm.plan.high, 0);
                complete = peer32(&sm.plan.complete, 0);
                known = peer32(&sm.plan.known, 0);
                const bool apart = peer32(&sm.plan.apart, 0);
                const int range = bits_of_range(low, high), shift = max(0, range - 10);
                uint64_t over = 0;
                int hits = 0;
                if (!apart && rank > 0) clear_fine(sm);
                sure = STAGED && apart && (last_round || complete) && __float_as_uint(ratio) <= high;
                found = 0;
                const bool weigh = !known || sure;
#pragma unroll 4
                for (int i = i0; i < i1; ++i) {
                    const uint32_t bits = __float_as_uint(row.at(i));
                    const bool hit = bits - low < high - low;
                    if (STAGED) found = found << 1 | hit;
                    else hits += hit;
                    if (hit && !apart) add_fine(sm, round > 0, (bits - low) >> shift, bits);
                    if (weigh && bits >= high) over += units_of(bits);
                }
                if (STAGED) hits = __popcll(found);
                sure_mass = over;
                if (!known) put_mass(over);
                if (apart) {
                    // ---- the tokens themselves to the first block: a warp asks for room once, and then goes through its tokens again ----
                    const int all = __reduce_add_sync(0xffffffffu, hits);
                    if (all) {
                        uint32_t at = lane == 0 ? add32(&sm.listed, 0, all) : 0;
                        at = __shfl_sync(0xffffffffu, at, 0);
                        int before = hits;
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) {
                            const int x = __shfl_up_sync(0xffffffffu, before, o);
                            if (lane >= o) before += x;
                        }
                        at += before - hits;
                        const auto put = [&](int i, uint32_t bits) {
                            if (at < kListed) {
                                put32(&sm.list[at], 0, bits);
                                put32(&sm.place[at], 0, first + i);
                            }
                            ++at;
                        };
                        if constexpr (STAGED) {
                            each_found([&](int i) { put(i, __float_as_uint(weights[i])); });
                        } else {
#pragma unroll 1
                            for (int i = i0; i < i1 && hits > 0; ++i) {
                                const uint32_t bits = __float_as_uint(row.at(i));
                                if (bits - low < high - low) {
                                    put(i, bits);
                                    --hits;
                                }
                            }
                        }
                    }
                } else if (rank > 0) {
                    __syncthreads();
#pragma unroll 1
                    for (int i = tid; i < kFineBins; i += kFilterThreads) {
                        const uint64_t v = own_fine(sm, i);          // (the row's limbs could exceed 32 bits)
                        if (v) add64(&sm.joined[i], 0, v);
                    }
                }
                cluster_sync();
                if (!known) above = all_mass();
                known = true;
                if (apart) {
                    listed = min((int)peer32(&sm.listed, 0), kListed);
                    if (rank == 0 && !(complete && listed <= kRanked)) b = select(sm, round > 0, listed, need, complete ? 0 : above, low, high);
                    break;
                }
                // ---- too many for the list (equal weights, or a mass that flat tails make up): their masses in 1,024 bins, and on with one of these ----
                if (rank == 0) {
                    find_fine(sm, need, above, true);
                    // (never beyond the range, so that it stays one, and ``shift`` falls until a single weight is left)
                    low += min((uint32_t)sm.found_bin, (high - low - 1) >> shift) << shift;
                    high = min(high, low + (1u << shift));
                    above = sm.found_before;
                    some = round > 0 ? sm.found_here / max((uint64_t)1, units_of(low)) : sm.found_here;
                    if (tid == 0) sm.plan.apart = shift > 0;
                    b = Border{low, above, sm.found_here};
                }
                cluster_sync();
                if (peer32(&sm.plan.apart, 0) == 0) break;      // a single weight is left
                cluster_sync();                                // (read before the next plan is made)
            }
            if (complete) {
                // ---- all that top-k leaves is here ----
                if (listed <= kRanked) {
                    // The first block goes on alone, but does not end before the others have read what lies in it.
                    asm volatile("barrier.cluster.arrive;" ::: "memory");
                    if (rank > 0) {
                        asm volatile("barrier.cluster.wait;" ::: "memory");
                        return;
                    }
                    // Some threads to a token: how many stand before it, and what mass?
                    int bits_of_tokens = 5;
                    while ((1 << bits_of_tokens) < listed) ++bits_of_tokens;
                    const int share = kFilterThreads >> bits_of_tokens, own = tid / share, part = tid % share;
                    uint64_t* masses = reinterpret_cast<uint64_t*>(sm.fine[0]);
                    if (tid < listed) masses[tid] = units_of(sm.list[tid]);
                    __syncthreads();
                    const bool there = own < listed;
                    const uint32_t bits = there ? sm.list[own] : 0;
                    const int place = there ? sm.place[own] : 0;
                    const uint64_t mass = there ? masses[own] : 0;
                    int count = 0;
                    uint64_t before = 0;
#pragma unroll 4
                    for (int i = part; i < listed; i += share) {
                        const uint32_t other = sm.list[i];
                        const bool ahead = other > bits || (other == bits && sm.place[i] < place);
                        count += ahead;
                        before += ahead ? masses[i] : 0;
                    }
                    for (int o = 1; o < share; o <<= 1) {
                        count += __shfl_xor_sync(0xffffffffu, count, o);
                        before += __shfl_xor_sync(0xffffffffu, before, o);
                    }
                    bool stays = there && count < k;
                    if (by_mass) {
                        within = block_sum64(stays && part == 0 ? mass : 0, sm);
                        stays = stays && (double)before < (double)p * (double)within;
                    }
                    stays = stays && __uint_as_float(bits) >= ratio;
                    const uint64_t total = block_sum64(stays && part == 0 ? mass : 0, sm);
                    if (there && part == 0) masses[own] = stays ? mass : 0;
                    __syncthreads();
                    before = 0;
#pragma unroll 4
                    for (int i = part; i < listed; i += share) before += sm.place[i] < place ? masses[i] : 0;
                    for (int o = 1; o < share; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
                    const uint64_t target = min((uint64_t)((double)u * (double)total), total - 1);
                    if (stays && part == 0 && target >= before && target < before + mass) {
                        a.token[r] = place;
                        a.logprob[r] = (row.top == INFINITY ? 0.f : __fdiv_rn(__fsub_rn(a.logits[(int64_t)r * a.ld + place], row.top), t))
                                     - logf((float)((double)total * (1.0 / 1099511627776.0)));
                    }
                    asm volatile("barrier.cluster.wait;" ::: "memory");
                    return;
                }
                if (rank == 0) {
                    border = b.bits;
                    ties = (uint64_t)k - b.above;
                    equal = b.here;
                    if (by_mass) {
                        uint64_t sum = 0;
#pragma unroll 1
                        for (int i = tid; i < listed; i += kFilterThreads)
                            if (sm.list[i] > border) sum += units_of(sm.list[i]);
                        within = block_sum64(sum, sm) + ties * units_of(border);
                        const double mass_need = (double)p * (double)within;
                        const Border m = select(sm, true, listed, mass_need, 0, border, high);
                        uint64_t there;
                        uint64_t n = ties_of(m, mass_need, &there);
                        if (m.bits == border) n = min(n, ties);
                        border = m.bits;
                        ties = n;
                        equal = there;
                    }
                }
                round = 2;
            } else if (rank == 0) {
                if (round == 0) {
                    border = b.bits;
                    ties = (uint64_t)k - b.above;
                    equal = b.here;
                } else {
                    uint64_t there;
                    uint64_t n = ties_of(b, need, &there);
                    if (b.bits == border) n = min(n, ties);
                    border = b.bits;
                    ties = n;
                    equal = there;
                }
            }
            // ---- known to all ----
            if (rank == 0 && tid == 0) {
                sm.plan.border = border;
                sm.plan.ties = ties;
                sm.plan.equal = equal;
            }
            cluster_sync();
            border = peer32(&sm.plan.border, 0);
            ties = peer64(&sm.plan.ties, 0);
            equal = peer64(&sm.plan.equal, 0);
            if (round == 0 && by_mass) {
                uint64_t sum = 0;                              // (the second round looks at the row's masses anyway)
#pragma unroll 1
                for (int i = i0; i < i1; ++i)
                    if (__float_as_uint(row.at(i)) > border) sum += units_of(__float_as_uint(row.at(i)));
                put_mass(sum);
                cluster_sync();
                within = all_mass() + ties * units_of(border);
                cluster_sync();                                // read before the next sums are put there
            }
        }
    }

    // ---- the draw, by index ----
    if (__float_as_uint(ratio) > border) {                     // min-p leaves fewer
        border = __float_as_uint(ratio);
        ties = equal = 0;
    }
    int cut = 0x7fffffff;                                      // the last token of the thread that may stay at the border
    if (ties < equal) {
        int mine = 0;
#pragma unroll 1
        for (int i = i0; i < i1; ++i) mine += __float_as_uint(row.at(i)) == border;
        const uint64_t upto = block_scan64(mine, sm.warp_sum);
        if (tid < (int)blocks) put32(&sm.count[rank], tid, (uint32_t)sm.warp_sum[kFilterWarps]);
        cluster_sync();
        int64_t left = (int64_t)ties - ((int64_t)upto - mine);     // to keep of the thread's and those behind them
#pragma unroll 1
        for (uint32_t b = 0; b < rank; ++b) left -= sm.count[b];
        if (left < mine) {
            cut = -1;
#pragma unroll 1
            for (int i = i0; i < i1 && left > 0; ++i)
                if (__float_as_uint(row.at(i)) == border) {
                    cut = i;
                    --left;
                }
        }
    }
    const auto kept = [&](int i) -> uint64_t {
        const uint32_t bits = __float_as_uint(row.at(i));
        return bits > border || (bits == border && i <= cut) ? units_of(bits) : 0;
    };
    uint64_t mine = 0;
    if (sure) {
        mine = sure_mass;
        each_found([&](int i) { mine += kept(i); });
    } else {
#pragma unroll 4
        for (int i = i0; i < i1; ++i) mine += kept(i);
    }
    const uint64_t upto = block_scan64(mine, sm.warp_sum);
    if (tid < (int)blocks) put64(&sm.mass[rank], tid, sm.warp_sum[kFilterWarps]);
    cluster_sync();
    uint64_t total = 0, run = upto - mine;
#pragma unroll 1
    for (uint32_t b = 0; b < blocks; ++b) {
        if (b < rank) run += sm.mass[b];
        total += sm.mass[b];
    }
    const uint64_t target = min((uint64_t)((double)u * (double)total), total - 1);
    if (target < run || target >= run + mine) return;
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
        run += kept(i);
        if (run > target) {
            a.token[r] = first + i;
            a.logprob[r] = (row.top == INFINITY ? 0.f : __fdiv_rn(__fsub_rn(row.z[i], row.top), t)) - logf((float)((double)total * (1.0 / 1099511627776.0)));
            return;
        }
    }
}

constexpr int kMostStaged = (113 * 1024 - (int)sizeof(FilterShared) - 1024) / 4;      // weights that a block's half of the shared memory holds
static_assert((kMostStaged + kFilterThreads - 1) / kFilterThreads + 1 <= 64, "a thread's tokens in a mask");
static_assert(kMostStaged < 1 << (32 - kCountBits), "a block's tokens in a packed count");

}  // namespace

CPM_API int cpm_sample_filtered(const float* logits, int64_t ld, int n_rows, int vocab, int* token, float* logprob, const float* uniform,
                                const float* temperature, const int* top_k, const float* top_p, const float* min_p, uint64_t seed,
                                const int* seq_key, const int* step_key, const int* drawn, cudaStream_t stream) {
    if (n_rows <= 0) return CPM_OK;
    if (vocab < 1 || vocab > kMostVocab || n_rows > 0x7fffffff / 8) return CPM_BAD_ARGUMENT;
    if (!uniform && (!seq_key || !step_key)) return CPM_BAD_ARGUMENT;
    const int sms = device_sms();
    // as many blocks a row as run at the same time, and as the weights need; a block of few tokens is not worth its barriers
    int blocks = 8;
    while (blocks > 1 && ((int64_t)n_rows * blocks > 2 * sms || vocab < 1024 * blocks) && (vocab + blocks / 2 - 1) / (blocks / 2) <= kMostStaged - 4) blocks /= 2;
    const int per_block = ((vocab + blocks - 1) / blocks + 3) & ~3;
    const FilterArgs a{logits, ld, vocab, per_block, uniform, temperature, top_p, min_p, top_k, seq_key, step_key, drawn, seed, token, logprob};
    if (per_block <= kMostStaged) {
        static bool done[kMaxDevices];
        const int status = ensure_dynamic_smem(sample_filtered_kernel<true>, kMostStaged * 4, done);
        if (status != CPM_OK) return status;
        cpm_launch_cluster(kLaunchOther, sample_filtered_kernel<true>, dim3(n_rows * blocks), kFilterThreads, (size_t)per_block * 4, stream, blocks, a);
    } else {
        cpm_launch_cluster(kLaunchOther, sample_filtered_kernel<false>, dim3(n_rows * blocks), kFilterThreads, 0, stream, blocks, a);
    }
    return launch_status();
}
