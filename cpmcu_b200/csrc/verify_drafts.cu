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
// What bounds it: the first launch, whose phases wait for one another (sample_filtered.cu).  64 sequences of 5 tokens, vocabulary 73,448, with probabilities: 128 us, 106 of
// them the first launch and 22 this one (37 MB of the refused rows: 6 us from memory, the rest the path before it, two barriers of the cluster and the run that is read
// again); one sequence: 24 us, 15 and 9.  32 trees of 16 tokens, vocabulary 32,000, without probabilities: 74 us, 3 of them this launch.
#include "filtered.cuh"

// Every row's draw (sample_filtered.cu).
CPM_API int cpm_sample_drafts(const float* logits, int64_t ld, int n_rows, int vocab, int* token, float* logprob, const float* uniform, const float* temperature,
                              const int* top_k, const float* top_p, const float* min_p, uint64_t seed, const int* seq_key, const int* step_key,
                              const int* row_seq, const int* positions, const int* cu, int n_seqs, void* kept, cudaStream_t stream);

namespace {

constexpr int kWarps = 16, kThreads = 32 * (kWarps + 1), kMostBlocks = 8;        // and one that writes the path
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
    // Below this a logit less the largest has a weight that is not kept, or no units, for sure: t (log of the border, or of 2^-40, less 1/1000, which is far more than
    // the logarithm, the exponential and these products are off).
    __device__ __forceinline__ float floor_of() const {
        if (k.border == kOneToken || k.top == INFINITY) return -INFINITY;
        return w.t * (fmaxf(logf(__uint_as_float(k.border)), -27.726f) * 1.00001f - 0.001f);
    }
    __device__ __forceinline__ uint64_t units(int v, float z) const {
        if (k.border == kOneToken) return v == k.cut ? k.total : 0;
        const uint32_t bits = __float_as_uint(w.form(z));
        return bits > k.border || (bits == k.border && v <= k.cut) ? units_of(bits) : 0;
    }
    // What the drafter's probability takes of a token's units (a number that is none: nothing).
    __device__ __forceinline__ uint64_t taken(float q) const { return __double2ull_rz((double)fminf(fmaxf(q, 0.f), 1.f) * (double)k.total); }
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
    uint64_t accepted;                                 // the root and the accepted tokens
    int last, refused;                                 // the last of them; whether its row is to be drawn again
};

__global__ void __launch_bounds__(kThreads, 1)
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
                    const Filtered f = filtered(a, first + i, t);
                    ok = false;
                    if (x >= 0 && x < a.vocab) {
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
        if (lane == 0) {
            sm.accepted = accepted;
            sm.last = last;
            sm.refused = refused;
        }
    }
    __syncthreads();
    const uint64_t accepted = sm.accepted;
    const int count = __popcll(accepted);
    // ---- the path, by a warp that has nothing else to do where a row is drawn again ----
    if (rank == 0 && warp == (int)blockDim.x / 32 - 1) {
        // a token of the path stands where as many of it come before; the token behind it is the path's next one's id
#pragma unroll 1
        for (int i = lane; i < n; i += 32) {
            if (!(accepted >> i & 1)) continue;
            const int at = __popcll(accepted & ((1ull << i) - 1));
            a.path[(int64_t)s * a.most + at] = i;
            if (at == 0) continue;
            const int id = a.ids[first + i], row = first + (a.probs || !a.parents ? i - 1 : a.parents[first + i]);
            a.tokens[(int64_t)s * a.most + at - 1] = id;
            a.logprob[(int64_t)s * a.most + at - 1] = a.probs ? filtered(a, row, t).logprob(a.logits[(int64_t)row * a.ld + id]) : a.drawn_logprob[row];
        }
#pragma unroll 1
        for (int i = count + lane; i < a.most; i += 32) {
            a.tokens[(int64_t)s * a.most + i] = a.path[(int64_t)s * a.most + i] = -1;
            a.logprob[(int64_t)s * a.most + i] = 0.f;
        }
        if (lane == 0) a.count[s] = count;
    }
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
    // A warp has up to 32 runs of some times 128 neighbouring tokens, four of which are a lane's; lane g keeps the sum of run g, so that the token's run is known at the end.
    const int per_run = 128 * max(1, ((end - begin + kWarps - 1) / kWarps + 128 * 32 - 1) / (128 * 32));
    const int each = ((end - begin + kWarps - 1) / kWarps + per_run - 1) / per_run * per_run;
    const int w0 = min(end, begin + warp * each), w1 = warp < kWarps ? min(end, w0 + each) : w0;       // (none of the last warp, which has the path)
    const float *z = a.logits + (int64_t)row * a.ld, *q = a.probs + (int64_t)row * a.ldq;
    const bool whole = (((uintptr_t)(z + w0) | (uintptr_t)(q + w0)) & 15) == 0;
    struct Four { float z[4], q[4]; };
    const auto load = [&](int v, Four& x) {              // (nothing behind the warp's end)
        if (whole && v + 4 <= w1) {
            *reinterpret_cast<float4*>(x.z) = __ldg(reinterpret_cast<const float4*>(z + v));
            *reinterpret_cast<float4*>(x.q) = __ldg(reinterpret_cast<const float4*>(q + v));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x.z[e] = v + e < w1 ? z[v + e] : -INFINITY;
                x.q[e] = v + e < w1 ? q[v + e] : 1.f;
            }
        }
    };
    const float least = f.floor_of(), k_top = f.k.top;
    // units beyond what the drafter's probability takes
    const bool quick = f.w.quick() && f.k.border != kOneToken;
    const auto left = [&](int v, const Four& x, uint64_t (&r)[4]) {
        if (quick) {
            // four tokens without a branch between them, if one of the warp's may be kept
            bool any = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) any |= !(__fsub_rn(x.z[e], k_top) < least);
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = 0;
            if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float w = f.w.form_quick(x.z[e]);
                const uint32_t bits = __float_as_uint(w);
                const bool kept = v + e < w1 && (bits > f.k.border || (bits == f.k.border && v + e <= f.k.cut));
                const int64_t d = (int64_t)__float2ull_rz(w * 0x1p40f) - (int64_t)f.taken(x.q[e]);      // (both below 2^62)
                r[e] = kept && d > 0 ? d : 0;
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint64_t w = v + e < w1 && !(__fsub_rn(x.z[e], k_top) < least) ? f.units(v + e, x.z[e]) : 0;
            r[e] = 0;
            if (w) {
                const uint64_t taken = f.taken(x.q[e]);
                r[e] = w > taken ? w - taken : 0;
            }
        }
    };
    const auto warp_total = [](uint64_t v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    constexpr int kAhead = 4;
    uint64_t mine = 0, run_sum = 0;                      // of the lane's run, and the lane's share of the run under way
    int number = 0, filled = 0;
#pragma unroll 1
    for (int v0 = w0; v0 < w1; v0 += 128 * kAhead) {
        Four x[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) load(v0 + 128 * u + 4 * lane, x[u]);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int at = v0 + 128 * u;
            if (at >= w1) break;
            uint64_t r[4];
            left(at + 4 * lane, x[u], r);
            run_sum += r[0] + r[1] + r[2] + r[3];
            if ((filled += 128) == per_run || at + 128 >= w1) {
                const uint64_t all = warp_total(run_sum);
                if (lane == number++) mine = all;
                run_sum = 0;
                filled = 0;
            }
        }
    }
    const uint64_t sum = warp_total(mine);
    if (lane == 0 && warp < kWarps) sm.warp_sum[warp] = sum;
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
    if (warp == kWarps || target < before || target >= before + sum) return;
    uint64_t upto = mine;                                // the run it is in
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    const int run = __ffs(__ballot_sync(0xffffffffu, target < before + upto)) - 1;
    before += __shfl_sync(0xffffffffu, upto - mine, run);
    const int stop = min(w1, w0 + (run + 1) * per_run);
#pragma unroll 1
    for (int v0 = w0 + run * per_run; v0 < stop; v0 += 128) {
        const int v = v0 + 4 * lane;
        Four x;
        uint64_t r[4];
        load(v, x);
        left(v, x, r);
        const uint64_t own = r[0] + r[1] + r[2] + r[3];
        upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const uint64_t all = __shfl_sync(0xffffffffu, upto, 31);
        if (target < before + all) {
            uint64_t from = before + upto - own;
            if (target >= from && target < from + own) {
                int e = 0;
                while (e < 3 && target >= from + r[e]) from += r[e++];
                a.tokens[out] = v + e;
                a.logprob[out] = f.logprob(z[v + e]);
            }
            return;
        }
        before += all;
    }
}

}  // namespace

// rows: 8 bytes a row of the logits (its draw and that one's log-probability), with ``probs`` behind 32 (what its filters keep).  out [3][seqs][most]: the tokens that a
// step gives (int32), the places of the tokens that stay, the root and the accepted ones (int32), and log-probabilities (fp32); what is behind ``count`` of them: -1, -1 and 0.
CPM_API int cpm_verify_drafts(const float* logits, int64_t ld, int n_rows, int vocab, void* rows, const int* ids, const int* row_seq, const int* cu, int n_seqs, int most,
                              const int* parents, const float* probs, int64_t ldq, const float* accept, const float* uniform, const float* temperature,
                              const int* top_k, const float* top_p, const float* min_p, uint64_t seed, const int* seq_key, const int* step_key,
                              const int* positions, int* out, int* count, cudaStream_t stream) {
    if (n_seqs <= 0) return CPM_OK;
    if (n_rows < 0 || vocab < 1 || most < 1 || most > kMostTokens || n_seqs > 0x7fffffff / kMostBlocks) return CPM_BAD_ARGUMENT;
    if ((probs && (parents || !accept || !uniform)) || (!rows && n_rows > 0)) return CPM_BAD_ARGUMENT;
    KeptRow* const kept = probs ? (KeptRow*)rows : nullptr;
    int* const drawn = (int*)((char*)rows + (probs ? sizeof(KeptRow) * n_rows : 0));
    const float* const drawn_logprob = (const float*)(drawn + n_rows);
    const int status = cpm_sample_drafts(logits, ld, n_rows, vocab, drawn, (float*)(drawn + n_rows), uniform, temperature, top_k, top_p, min_p, seed, seq_key, step_key,
                                         row_seq, positions, cu, n_seqs, kept, stream);
    if (status != CPM_OK) return status;
    int* const tokens = out;
    int* const path = out + (int64_t)n_seqs * most;
    float* const logprob = (float*)(out + 2 * (int64_t)n_seqs * most);
    int blocks = 1;
    if (probs) {                                         // as many blocks a sequence as run at the same time, one an SM
        const int sms = device_sms();
        blocks = kMostBlocks;
        while (blocks > 1 && ((int64_t)n_seqs * blocks > sms || vocab < 2048 * blocks)) blocks /= 2;
    }
    const int per_block = ((vocab + blocks - 1) / blocks + 3) & ~3;
    const VerifyArgs a{logits, ld, probs, ldq, accept, uniform, temperature, ids, cu, parents, drawn, drawn_logprob, kept, vocab, per_block,
                       n_rows, most, tokens, count, path, logprob};
    cpm_launch_cluster(kLaunchOther, verify_drafts_kernel, dim3(n_seqs * blocks), probs ? kThreads : 64, 0, stream, blocks, a);
    return launch_status();
}
