// Checking drafted tokens against the model's probabilities.
//
// A sequence brings tokens 0 .. n - 1: the last one it has, and drafted ones that follow one another or form a tree.  Row i of the logits says what follows
// token i.  Its filtered distribution is held in whole units of 2^-40 of the likeliest token (sample_filtered.cu): token v has W_v units, all kept ones M.
//     with the probabilities q_i that drafted token i + 1 was drawn from (a chain):
//         Q_v = floor(q_v M);  token x = i + 1 is accepted iff  a_i Q_x < W_x,  that is with probability min(1, p_x / q_x);
//         at the first refusal the sequence goes on with the token at which the running sum of  max(0, W_v - Q_v), by index, exceeds  floor(u_i * its total)
//         (where that is nothing: of W_v); if nothing is refused, with the one drawn from the last row.  What comes out is distributed as the model's own tokens.
//     without (chain or tree): row i has drawn its token by its number u_i; the first child of i that is that token is accepted, and so on from there; the
//         sequence goes on with what the last accepted token's row has drawn.  So drafts change no token, only how many a step gives.
// Sums are whole numbers, so a sequence's tokens depend on nothing but its rows and numbers.
//
// Two launches: one reads every row once, draws its token and notes what its filters keep (cpm_sample_drafts); this one, a cluster of blocks a sequence, looks at
// n logits and probabilities, and reads one row of each again where a token was refused.
#include "filtered.cuh"

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kMostBlocks = 8;
constexpr int kMostTokens = 64;                        // of a sequence: two to a lane

struct VerifyArgs {
    const float* logits;
    int64_t ld;
    const float* probs;                                // null: tokens that have been drawn are compared
    int64_t ldq;
    const float *accept, *uniform, *temperature;
    const int *ids, *cu, *parents, *drawn;
    const float* drawn_logprob;
    const KeptRow* kept;
    int vocab, per_block, n_rows, most;
    int *tokens, *count, *path;
    float* logprob;
};

// A row whose filters are known.
struct Filtered {
    Weigher w;
    KeptRow k;
    __device__ __forceinline__ uint64_t units(int v, float z) const {
        if (k.border == kOneToken) return v == k.cut ? k.total : 0;
        const uint32_t bits = __float_as_uint(w.form(z));
        return bits > k.border || (bits == k.border && v <= k.cut) ? units_of(bits) : 0;
    }
    // What the drafter's probability takes of a token's units (a number that is none: nothing).
    __device__ __forceinline__ uint64_t taken(float q) const { return __double2ull_rz(fmin(fmax((double)q, 0.0), 1.0) * (double)k.total); }
    __device__ __forceinline__ float logprob(float z) const {
        if (k.border == kOneToken) return k.top == -INFINITY ? -INFINITY : 0.f;
        return (k.top == INFINITY ? 0.f : w.over_t(__fsub_rn(z, k.top))) - logf((float)((double)k.total * (1.0 / 1099511627776.0)));
    }
};

__device__ __forceinline__ Filtered filtered(const VerifyArgs& a, int row, float t) {
    Filtered f;
    f.k = a.kept[row];
    f.w.set(f.k.top, t > 0.f ? t : 1.f);
    return f;
}

struct VerifyShared {
    uint64_t warp_sum[kWarps + 1];
    alignas(8) uint64_t mass[kMostBlocks];             // of the cluster's blocks, which write here
    int drawn[kMostTokens];
    int count, last, refused;                          // accepted tokens and the root; the last of them; whether its row is to be drawn again
};

__global__ void __launch_bounds__(kThreads)
verify_drafts_kernel(const __grid_constant__ VerifyArgs a) {
    __shared__ VerifyShared sm;
    pdl_wait();
    const int blocks = (int)cluster_blocks(), rank = (int)cluster_rank(), s = blockIdx.x / blocks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = max(0, min(a.cu[s], a.n_rows)), n = max(0, min(min(a.cu[s + 1], a.n_rows) - first, a.most));
    const float t = a.temperature ? a.temperature[s] : 0.f;

    // ---- the accepted path, by every block for itself (its first warp) ----
    if (warp == 0) {
        const bool mine[2] = {lane < n, lane + 32 < n};
        int id[2], parent[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = lane + 32 * h;
            id[h] = mine[h] ? a.ids[first + i] : -1;
            parent[h] = mine[h] ? (a.parents ? a.parents[first + i] : i - 1) : -2;
            if (!a.probs && mine[h]) sm.drawn[i] = a.drawn[first + i];
        }
        __syncwarp();
        uint64_t accepted = n > 0 ? 1 : 0;              // tokens of the path
        int last = 0, refused = 0;
        if (a.probs) {
            uint32_t bad[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = lane + 32 * h;
                bool ok = true;                         // whether token i + 1 is accepted
                if (i + 1 < n) {
                    const int x = a.ids[first + i + 1];
                    ok = false;
                    if (x >= 0 && x < a.vocab) {
                        const Filtered f = filtered(a, first + i, t);
                        const uint64_t w = f.units(x, a.logits[(int64_t)(first + i) * a.ld + x]), q = f.taken(a.probs[(int64_t)(first + i) * a.ldq + x]);
                        ok = (double)a.accept[first + i] * (double)q < (double)w;
                    }
                }
                bad[h] = __ballot_sync(0xffffffffu, !ok);
            }
            const uint64_t all = (uint64_t)bad[1] << 32 | bad[0];
            const int stop = all ? __ffsll(all) - 1 : n - 1;          // the row whose token was refused, or the last
            if (n > 0) {
                last = stop;
                refused = all != 0;
                accepted = ~0ull >> (63 - stop);
            }
        } else {
#pragma unroll 1
            for (int turn = 1; turn < n; ++turn) {       // (a path has no more tokens than the sequence)
                const int x = sm.drawn[last];
                uint32_t hit[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) hit[h] = __ballot_sync(0xffffffffu, mine[h] && parent[h] == last && lane + 32 * h > last && id[h] == x);
                const uint64_t all = (uint64_t)hit[1] << 32 | hit[0];
                if (!all) break;
                last = __ffsll(all) - 1;
                accepted |= 1ull << last;
            }
        }
        if (rank == 0) {
            const int count = __popcll(accepted);
            // a token of the path stands where as many of it come before; the token behind it is the path's next one's id
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = lane + 32 * h;
                if (mine[h] && accepted >> i & 1) {
                    const int at = __popcll(accepted & ((1ull << i) - 1));
                    a.path[(int64_t)s * a.most + at] = i;
                    if (at > 0) {
                        a.tokens[(int64_t)s * a.most + at - 1] = id[h];
                        const int row = first + (a.probs ? i - 1 : parent[h]);
                        a.logprob[(int64_t)s * a.most + at - 1] =
                            a.probs ? filtered(a, row, t).logprob(a.logits[(int64_t)row * a.ld + id[h]]) : a.drawn_logprob[row];
                    }
                }
            }
            for (int i = lane; i < a.most; i += 32) {
                if (i >= count) {
                    a.tokens[(int64_t)s * a.most + i] = a.path[(int64_t)s * a.most + i] = -1;
                    a.logprob[(int64_t)s * a.most + i] = 0.f;
                }
            }
            if (lane == 0) a.count[s] = count;
        }
        if (lane == 0) {
            sm.count = __popcll(accepted);
            sm.last = last;
            sm.refused = refused;
        }
    }
    __syncthreads();
    const int count = sm.count;
    if (count == 0) return;                             // (the whole cluster leaves)
    const int64_t out = (int64_t)s * a.most + count - 1;
    const int row = first + sm.last;
    if (!sm.refused) {
        if (rank == 0 && tid == 0) {
            a.tokens[out] = a.drawn[row];
            a.logprob[out] = a.drawn_logprob[row];
        }
        return;
    }

    // ---- a token in the place of the refused one ----
    const Filtered f = filtered(a, row, t);
    const int begin = min(a.vocab, rank * a.per_block), end = min(a.vocab, begin + a.per_block);
    const int each = ((end - begin + kWarps - 1) / kWarps + 127) & ~127;             // tokens of a warp, which are neighbours
    const int w0 = min(end, begin + warp * each), w1 = min(end, w0 + each);
    const float *z = a.logits + (int64_t)row * a.ld, *q = a.probs + (int64_t)row * a.ldq;
    const bool whole = (((uintptr_t)(z + w0) | (uintptr_t)(q + w0)) & 15) == 0;
    // four neighbouring tokens' units beyond what the drafter's probability takes; nothing behind the warp's end
    const auto left = [&](int v, uint64_t (&r)[4]) {
        float zz[4], qq[4];
        if (whole && v + 4 <= w1) {
            *reinterpret_cast<float4*>(zz) = *reinterpret_cast<const float4*>(z + v);
            *reinterpret_cast<float4*>(qq) = *reinterpret_cast<const float4*>(q + v);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                zz[e] = v + e < w1 ? z[v + e] : -INFINITY;
                qq[e] = v + e < w1 ? q[v + e] : 1.f;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint64_t w = v + e < w1 ? f.units(v + e, zz[e]) : 0, taken = w ? f.taken(qq[e]) : 0;
            r[e] = w > taken ? w - taken : 0;
        }
    };
    uint64_t sum = 0;
#pragma unroll 2
    for (int v = w0 + 4 * lane; v < w1; v += 128) {
        uint64_t r[4];
        left(v, r);
        sum += r[0] + r[1] + r[2] + r[3];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sm.warp_sum[warp] = sum;
    __syncthreads();
    uint64_t before = 0, block_total = 0;
#pragma unroll 1
    for (int i = 0; i < kWarps; ++i) {
        if (i < warp) before += sm.warp_sum[i];
        block_total += sm.warp_sum[i];
    }
    if (blocks > 1) {
        cluster_sync();                                  // (nothing is put into a block that has not begun)
        if (tid < blocks) put64(&sm.mass[rank], tid, block_total);
        cluster_sync();
    } else {
        if (tid == 0) sm.mass[0] = block_total;
        __syncthreads();
    }
    uint64_t total = 0;
#pragma unroll 1
    for (int b = 0; b < blocks; ++b) {
        if (b < rank) before += sm.mass[b];
        total += sm.mass[b];
    }
    if (total == 0) {                                    // the drafter's probabilities leave nothing: the row's own token
        if (rank == 0 && tid == 0) {
            a.tokens[out] = a.drawn[row];
            a.logprob[out] = a.drawn_logprob[row];
        }
        return;
    }
    const uint64_t target = min((uint64_t)((double)a.uniform[row] * (double)total), total - 1);
    if (target < before || target >= before + sum) return;
#pragma unroll 1
    for (int v0 = w0; v0 < w1; v0 += 128) {
        const int v = v0 + 4 * lane;
        uint64_t r[4] = {0, 0, 0, 0};
        if (v < w1) left(v, r);
        const uint64_t own = r[0] + r[1] + r[2] + r[3];
        uint64_t upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const uint64_t all = __shfl_sync(0xffffffffu, upto, 31);
        if (target < before + all) {
            uint64_t run = before + upto - own;
            if (target >= run && target < run + own) {
                int e = 0;
                while (e < 3 && target >= run + r[e]) run += r[e++];
                a.tokens[out] = v + e;
                a.logprob[out] = f.logprob(z[v + e]);
            }
            return;
        }
        before += all;
    }
}

}  // namespace

// ``kept`` and the draws are what cpm_sample_drafts left for the same rows.  tokens, path int32 and logprob fp32 [seqs, most]: the tokens that a step gives, the
// places of the tokens that stay (the root and the accepted ones), and what is behind ``count`` of them -1, -1 and 0.
CPM_API int cpm_verify_drafts(const float* logits, int64_t ld, int n_rows, int vocab, const int* ids, const int* cu, int n_seqs, int most, const int* parents,
                              const float* probs, int64_t ldq, const float* accept, const float* uniform, const float* temperature, const int* drawn,
                              const float* drawn_logprob, const void* kept, int* tokens, int* count, int* path, float* logprob, cudaStream_t stream) {
    if (n_seqs <= 0) return CPM_OK;
    if (n_rows < 0 || vocab < 1 || most < 1 || most > kMostTokens || n_seqs > 0x7fffffff / kMostBlocks) return CPM_BAD_ARGUMENT;
    if (probs && (parents || !accept || !uniform || !kept)) return CPM_BAD_ARGUMENT;
    int blocks = 1;
    if (probs) {                                         // as many blocks a sequence as run at the same time
        const int sms = device_sms();
        blocks = kMostBlocks;
        while (blocks > 1 && ((int64_t)n_seqs * blocks > 2 * sms || vocab < 2048 * blocks)) blocks /= 2;
    }
    const int per_block = ((vocab + blocks - 1) / blocks + 3) & ~3;
    const VerifyArgs a{logits, ld, probs, ldq, accept, uniform, temperature, ids, cu, parents, drawn, drawn_logprob, (const KeptRow*)kept, vocab, per_block,
                       n_rows, most, tokens, count, path, logprob};
    cpm_launch_cluster(kLaunchOther, verify_drafts_kernel, dim3(n_seqs * blocks), probs ? kThreads : 32, 0, stream, blocks, a);
    return launch_status();
}
