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
// A row is read once.  Its weights lie in the shared memory of a cluster of blocks (one to eight; the fewer rows, the more blocks a row), and every
// step runs there: the k-th weight and the weight at which the mass is reached are found by radix selection on the weight's bits (11 + 10 + 10, of
// which only the first looks at every weight's histogram), counts and masses of the blocks being added over distributed shared memory.
// What a row cannot do without is its logits, 4 bytes a token.
#include "common.cuh"
#include "philox.cuh"

namespace {

constexpr int kFilterThreads = 1024;
constexpr int kBins = 1024;                            // a weight's bits 30..20 end at 1016, the largest weight being 1
constexpr int kLimbBits = 14;                          // a mass is added in three limbs: 32-bit adds in shared memory are one instruction
constexpr int kMostVocab = 1 << 21;                    // so that a limb's sum over a block's tokens stays within 32 bits

struct FilterArgs {
    const float* logits;
    int64_t ld;
    int vocab, per_block;
    const float *uniform, *temperature, *top_p, *min_p;
    const int *top_k, *seq_key, *step_key;
    uint64_t seed;
    int* token;
    float* logprob;
};

struct FilterShared {
    uint32_t bins[3][kBins];
    uint64_t warp_sum[33];
    uint64_t found_before, found_here;                 // what lies above the bin that was found, and in it
    int found_bin;
    ArgMax best;                                       // of this block; read by the others
    uint64_t mass;                                     // likewise
    int count;
    ArgMax scratch[33];
    int cut;
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

__device__ __forceinline__ uint64_t units_of(float w) { return (uint64_t)((double)w * 1099511627776.0); }

__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Inclusive sums over the block's threads in order; the block's total is left in sums[32].
__device__ __forceinline__ uint64_t block_scan64(uint64_t v, uint64_t* sums) {
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
        const uint64_t own = sums[lane];
        uint64_t x = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        sums[lane] = x - own;
        if (lane == 31) sums[32] = x;
    }
    __syncthreads();
    return v + sums[warp];
}

// STAGED: the block's weights lie in shared memory; else (a vocabulary that eight blocks' do not hold) they are formed again from the logits.
template <bool STAGED>
struct Row {
    const float* z;                                    // the block's first logit
    float* w;
    int n;                                             // tokens of the block
    float top, t;
    __device__ __forceinline__ float form(float x) const {
        if (top == INFINITY) return x == INFINITY ? 1.f : 0.f;
        const float v = expf(__fdiv_rn(__fsub_rn(x, top), t));
        return v >= 0.f ? v : 0.f;                     // a logit that is no number is never drawn
    }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (STAGED) return w[i];
        else return form(z[i]);
    }
};

struct Border { uint32_t bits; uint64_t above, here; };      // a weight, and the count or mass of the tokens above it and at it

// The weight at which the running count (MASS false) or mass of the tokens, from the largest weight down, first reaches ``need``; only weights from
// ``least`` up are looked at, and the caller knows that these suffice.
template <bool MASS, bool STAGED>
__device__ Border select(const Row<STAGED>& row, FilterShared& sm, double need, uint32_t least) {
    const uint32_t blocks = cluster_blocks();
    uint32_t prefix = 0;
    uint64_t above = 0, here = 0;
#pragma unroll 1
    for (int level = 0; level < 3; ++level) {
        const int low = level == 0 ? 20 : level == 1 ? 10 : 0;
        for (int i = threadIdx.x; i < kBins; i += kFilterThreads)
#pragma unroll
            for (int u = 0; u < (MASS ? 3 : 1); ++u) sm.bins[u][i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < row.n; i += kFilterThreads) {
            const float w = row.at(i);
            const uint32_t bits = __float_as_uint(w);
            if (bits < least || (level > 0 && (bits >> (low + 10)) != prefix)) continue;
            const int bin = level == 0 ? bits >> 20 : (bits >> low) & (kBins - 1);
            if constexpr (MASS) {
                const uint64_t v = units_of(w);
                atomicAdd(&sm.bins[0][bin], (uint32_t)v & ((1u << kLimbBits) - 1));
                atomicAdd(&sm.bins[1][bin], (uint32_t)(v >> kLimbBits) & ((1u << kLimbBits) - 1));
                atomicAdd(&sm.bins[2][bin], (uint32_t)(v >> (2 * kLimbBits)));
            } else {
                atomicAdd(&sm.bins[0][bin], 1u);
            }
        }
        cluster_sync();
        const int bin = kBins - 1 - threadIdx.x;        // one bin a thread, from the largest weights down
        uint64_t v = 0;
        for (uint32_t b = 0; b < blocks; ++b)
#pragma unroll
            for (int u = 0; u < (MASS ? 3 : 1); ++u) v += (uint64_t)peer32(&sm.bins[u][bin], b) << (u * kLimbBits);
        const uint64_t upto = above + block_scan64(v, sm.warp_sum);
        if ((double)(upto - v) < need && (double)upto >= need) {
            sm.found_bin = bin;
            sm.found_before = upto - v;
            sm.found_here = v;
        }
        cluster_sync();                                 // the bins have been read
        prefix = level == 0 ? sm.found_bin : (prefix << 10) | sm.found_bin;
        above = sm.found_before;
        here = sm.found_here;
    }
    return Border{prefix, above, here};
}

// Sum over the cluster of a number of each block.
__device__ __forceinline__ uint64_t cluster_total(uint64_t own_of_thread, FilterShared& sm) {
    block_scan64(own_of_thread, sm.warp_sum);
    if (threadIdx.x == 0) sm.mass = sm.warp_sum[32];
    cluster_sync();
    uint64_t all = 0;
    for (uint32_t b = 0; b < cluster_blocks(); ++b) all += peer64(&sm.mass, b);
    cluster_sync();
    return all;
}

template <bool STAGED>
__global__ void __launch_bounds__(kFilterThreads)
sample_filtered_kernel(const __grid_constant__ FilterArgs a) {
    extern __shared__ float weights[];
    __shared__ FilterShared sm;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t blocks = cluster_blocks(), rank = cluster_rank();
    const int r = blockIdx.x / blocks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = min(a.vocab, (int)rank * a.per_block);
    Row<STAGED> row;
    row.n = min(a.vocab, first + a.per_block) - first;
    row.z = a.logits + (int64_t)r * a.ld + first;
    row.w = weights;

    // the largest logit, lowest index among equals
    ArgMax best{-INFINITY, 0x7fffffff};
    const int whole = ((uintptr_t)row.z & 15) == 0 ? row.n & ~3 : 0;
    for (int i0 = 4 * tid; i0 < whole; i0 += 16 * kFilterThreads) {
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + 4 * u * kFilterThreads;
            v[u] = i < whole ? *reinterpret_cast<const float4*>(row.z + i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + 4 * u * kFilterThreads;
            if (i >= whole) break;
            if constexpr (STAGED) *reinterpret_cast<float4*>(weights + i) = v[u];
            best = better(best, ArgMax{v[u].x, first + i});
            best = better(best, ArgMax{v[u].y, first + i + 1});
            best = better(best, ArgMax{v[u].z, first + i + 2});
            best = better(best, ArgMax{v[u].w, first + i + 3});
        }
    }
    for (int i = whole + tid; i < row.n; i += kFilterThreads) {
        const float v = row.z[i];
        if constexpr (STAGED) weights[i] = v;
        best = better(best, ArgMax{v, first + i});
    }
    best = block_argmax(best, sm.scratch);
    if (tid == 0) sm.best = best;
    cluster_sync();
    best = ArgMax{-INFINITY, 0x7fffffff};
    for (uint32_t b = 0; b < blocks; ++b) best = better(best, ArgMax{__uint_as_float(peer32(&sm.best.v, b)), (int)peer32(&sm.best.i, b)});
    cluster_sync();
    const float t = a.temperature ? a.temperature[r] : 0.f;
    if (best.v == -INFINITY || !(t > 0.f)) {                   // nothing that can be drawn: token 0; a greedy row: the largest
        if (rank == 0 && tid == 0) {
            a.token[r] = best.v == -INFINITY ? 0 : best.i;
            a.logprob[r] = best.v == -INFINITY ? -INFINITY : 0.f;
        }
        return;
    }
    row.top = best.v;
    row.t = t;
    if constexpr (STAGED) {
        for (int i = tid; i < row.n; i += kFilterThreads) weights[i] = row.form(weights[i]);
        __syncthreads();
    }

    // which tokens stay: those above the border, of those at it the first ``ties``, and of all only from ``ratio`` up
    int k = a.top_k ? a.top_k[r] : 0;
    const float p = a.top_p ? a.top_p[r] : 1.f;
    float ratio = a.min_p ? a.min_p[r] : 0.f;
    if (p <= 0.f || ratio > 1.f) k = 1;
    if (!(ratio <= 1.f)) ratio = 0.f;                          // above one: the first token alone, which it would leave out as well
    uint32_t border = 0;
    uint64_t ties = ~0ull, equal = 0;                          // tokens to keep at the border, and tokens there
    if (k > 0 && k < a.vocab) {
        const Border b = select<false>(row, sm, (double)k, 0u);
        border = b.bits;
        ties = (uint64_t)k - b.above;
        equal = b.here;
    }
    if (p < 1.f && p > 0.f && k != 1) {
        uint64_t own = 0;                                      // mass of the tokens that top-k leaves
        for (int i = tid; i < row.n; i += kFilterThreads) {
            const float w = row.at(i);
            if (__float_as_uint(w) > border || border == 0) own += units_of(w);
        }
        uint64_t within = cluster_total(own, sm);
        if (border) within += ties * units_of(__uint_as_float(border));
        const double need = (double)p * (double)within;
        const Border b = select<true>(row, sm, need, border);
        const uint64_t each = units_of(__uint_as_float(b.bits));
        const uint64_t there = b.here / each;
        uint64_t n = (uint64_t)ceil((need - (double)b.above) / (double)each);
        n = min(max(n, (uint64_t)1), there);
        while (n > 1 && (double)(b.above + (n - 1) * each) >= need) --n;
        while (n < there && (double)(b.above + n * each) < need) ++n;
        if (b.bits == border) n = min(n, ties);
        border = b.bits;
        ties = n;
        equal = there;
    }
    // a warp's tokens are neighbours, so that sums by warp go by index
    const int per_warp = ((row.n + 31) / 32 + 31) & ~31;
    const int w0 = min(row.n, warp * per_warp), w1 = min(row.n, w0 + per_warp);
    int cut = 0x7fffffff;                                      // the last token of the block that may stay at the border
    if (ties < equal) {
        int mine = 0;
        for (int i = w0 + lane; i < w1; i += 32) mine += __float_as_uint(row.at(i)) == border;
        const int of_warp = __reduce_add_sync(0xffffffffu, mine);
        const uint64_t upto = block_scan64(lane == 0 ? of_warp : 0, sm.warp_sum);
        if (tid == 0) {
            sm.count = (int)sm.warp_sum[32];
            sm.cut = 0x7fffffff;
        }
        cluster_sync();
        int64_t left = (int64_t)ties;                          // to keep in this block and behind it
        for (uint32_t b = 0; b < rank; ++b) left -= (int)peer32(&sm.count, b);
        if (left <= 0) {
            cut = -1;
        } else {
            const int64_t before = (int64_t)__shfl_sync(0xffffffffu, upto, 0) - of_warp;
            if (before < left && left < before + of_warp + 1 && of_warp > 0) {
                int64_t seen = before;
                for (int i0 = w0; i0 < w1; i0 += 32) {
                    const int i = i0 + lane;
                    const uint32_t hit = __ballot_sync(0xffffffffu, i < w1 && __float_as_uint(row.at(i)) == border);
                    if (seen + __popc(hit) >= left) {
                        if (lane == 0) sm.cut = i0 + __fns(hit, 0, (int)(left - seen));
                        break;
                    }
                    seen += __popc(hit);
                }
            }
            __syncthreads();
            cut = sm.cut;
        }
        cluster_sync();
    }
    const auto kept = [&](int i) -> uint64_t {
        const float w = row.at(i);
        const uint32_t bits = __float_as_uint(w);
        const bool stays = (bits > border || (bits == border && i <= cut)) && w >= ratio;
        return stays ? units_of(w) : 0;
    };
    uint64_t mine = 0;
    for (int i = w0 + lane; i < w1; i += 32) mine += kept(i);
    const uint64_t of_warp = warp_sum64(mine);
    const uint64_t upto = __shfl_sync(0xffffffffu, block_scan64(lane == 0 ? of_warp : 0, sm.warp_sum), 0);
    if (tid == 0) sm.mass = sm.warp_sum[32];
    cluster_sync();
    uint64_t total = 0, before = 0;
    for (uint32_t b = 0; b < blocks; ++b) {
        const uint64_t m = peer64(&sm.mass, b);
        if (b < rank) before += m;
        total += m;
    }
    cluster_sync();                                            // no block leaves while another may read from it
    const float u = a.uniform ? a.uniform[r] : philox_uniform(a.seed, (uint32_t)a.seq_key[r], (uint32_t)a.step_key[r]);
    const uint64_t target = min((uint64_t)((double)u * (double)total), total - 1);
    uint64_t run = before + upto - of_warp;
    if (of_warp == 0 || target < run || target >= run + of_warp) return;
    for (int i0 = w0; i0 < w1; i0 += 32) {
        const int i = i0 + lane;
        uint64_t v = i < w1 ? kept(i) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t x = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += x;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, run + v > target);
        if (past) {
            if (lane == __ffs(past) - 1) {
                const float z = row.z[i];
                a.token[r] = first + i;
                a.logprob[r] = (row.top == INFINITY ? 0.f : __fdiv_rn(__fsub_rn(z, row.top), t)) - logf((float)((double)total * (1.0 / 1099511627776.0)));
            }
            return;
        }
        run += __shfl_sync(0xffffffffu, v, 31);
    }
}

constexpr int kMostStaged = (227 * 1024 - (int)sizeof(FilterShared) - 1024) / 4;      // weights that a block's shared memory holds

}  // namespace

CPM_API int cpm_sample_filtered(const float* logits, int64_t ld, int n_rows, int vocab, int* token, float* logprob, const float* uniform,
                                const float* temperature, const int* top_k, const float* top_p, const float* min_p, uint64_t seed,
                                const int* seq_key, const int* step_key, cudaStream_t stream) {
    if (n_rows <= 0) return CPM_OK;
    if (vocab < 1 || vocab > kMostVocab || n_rows > 0x7fffffff / 8) return CPM_BAD_ARGUMENT;
    if (!uniform && (!seq_key || !step_key)) return CPM_BAD_ARGUMENT;
    const int sms = device_sms();
    // as many blocks a row as run at the same time, and as the weights need; a block of few tokens is not worth its barriers
    int blocks = 8;
    while (blocks > 1 && ((int64_t)n_rows * blocks > sms || vocab < 1024 * blocks) && (vocab + blocks / 2 - 1) / (blocks / 2) <= kMostStaged - 4) blocks /= 2;
    const int per_block = ((vocab + blocks - 1) / blocks + 3) & ~3;
    const FilterArgs a{logits, ld, vocab, per_block, uniform, temperature, top_p, min_p, top_k, seq_key, step_key, seed, token, logprob};
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
