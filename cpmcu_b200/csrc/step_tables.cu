// The description of a step, made on the device from the lengths of its requests, and the moving of accepted tokens' keys and values.
//
// Tables: sequence s holds l_s tokens and brings n_s.  With cu the running sum of n, token i of s has the place l_s + i in its sequence's cache, lies in page
// table[slot_s][place / 64], and stands at the position l_s + i, or l_s + its depth in the tree that the parents give; its ancestors are one bit a token.  Pages that
// the new tokens need, ceil((l + n) / 64) - ceil(l / 64), come from a list of free ones in the sequences' order.
// Every block forms both running sums for itself (a few bytes a sequence, out of L2), so that one launch without a barrier between blocks does; a token's
// depth is a walk over at most 64 parents in shared memory.
// Bound by the launch and the two passes over the sequences: 64 sequences of 5 tokens 3.1 us, 512 trees of 64 tokens with their pages handed out 5.0 (1 MB written: 0.14 us).
#include "common.cuh"

namespace {

constexpr int kTableThreads = 256;
constexpr int kMostSeqs = 4096;                         // whose running sums lie in shared memory
constexpr int kTreeTokens = 64;                         // of a sequence with a tree: bits of a word

struct TableArgs {
    const int *lengths, *fresh, *slots, *parents, *free;
    int n_free, n_seqs, n_tokens, n_slots, max_pages;
    int* page_table;
    int *cu, *kv_len, *token_seq, *positions, *places, *taken;
    int64_t *slot_map, *ancestors;
};

__device__ __forceinline__ int pages_of(int64_t tokens) { return (int)((tokens + kPageTokens - 1) / kPageTokens); }

__device__ __forceinline__ int length_of(const TableArgs& a, int s) { return max(0, a.lengths[s]); }

// Exclusive running sums of a pair of numbers a sequence, n_seqs + 1 of them.
__device__ __forceinline__ void sum_up(const TableArgs& a, int* tokens, int* pages) {
    __shared__ int warp_tokens[kTableThreads / 32], warp_pages[kTableThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int each = (a.n_seqs + kTableThreads - 1) / kTableThreads, s0 = min(a.n_seqs, tid * each), s1 = min(a.n_seqs, s0 + each);
    int t = 0, p = 0;
    for (int s = s0; s < s1; ++s) {
        const int n = max(0, a.fresh[s]);
        t += n;
        if (a.taken) p += pages_of((int64_t)length_of(a, s) + n) - pages_of(length_of(a, s));
    }
    int upto_t = t, upto_p = p;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto_t, o), y = __shfl_up_sync(0xffffffffu, upto_p, o);
        if (lane >= o) {
            upto_t += x;
            upto_p += y;
        }
    }
    if (lane == 31) {
        warp_tokens[warp] = upto_t;
        warp_pages[warp] = upto_p;
    }
    __syncthreads();
    int run_t = upto_t - t, run_p = upto_p - p;
    for (int w = 0; w < warp; ++w) {
        run_t += warp_tokens[w];
        run_p += warp_pages[w];
    }
    for (int s = s0; s < s1; ++s) {
        const int n = max(0, a.fresh[s]);
        tokens[s] = run_t;
        run_t += n;
        if (a.taken) {
            pages[s] = run_p;
            run_p += pages_of((int64_t)length_of(a, s) + n) - pages_of(length_of(a, s));
        }
    }
    if (tid == kTableThreads - 1) {
        tokens[a.n_seqs] = run_t;
        if (a.taken) pages[a.n_seqs] = run_p;
    }
    __syncthreads();
}

// Whether the free pages of a sequence are all there (and, whatever the lengths say, within the list: counts of nonsense may run over).
__device__ __forceinline__ bool pages_there(const TableArgs& a, const int* pages, int s) {
    return pages[s] >= 0 && pages[s] <= pages[s + 1] && pages[s + 1] <= a.n_free;
}

__device__ __forceinline__ int sequence_of(const int* cu, int n_seqs, int t) {       // the last whose first token is t or before
    int lo = 0, hi = n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kTableThreads)
step_tables_kernel(const __grid_constant__ TableArgs a) {
    extern __shared__ int sums[];
    __shared__ int up[kTableThreads + kTreeTokens];      // parents of the block's tokens and of those that their sequence has before them
    pdl_wait();
    int *cu = sums, *pages = sums + a.n_seqs + 1;
    sum_up(a, cu, pages);
    const int all = cu[a.n_seqs];
    // ---- what is by sequence, and its new pages ----
    for (int s = blockIdx.x * kTableThreads + threadIdx.x; s <= a.n_seqs; s += gridDim.x * kTableThreads) {
        a.cu[s] = cu[s];
        if (s == a.n_seqs) {
            if (a.taken) *a.taken = pages[s];
            break;
        }
        a.kv_len[s] = length_of(a, s) + cu[s + 1] - cu[s];
        const int slot = a.slots[s], have = pages_of(length_of(a, s));
        if (a.taken && pages_there(a, pages, s) && slot >= 0 && slot < a.n_slots) {      // (a sequence whose pages are not all there gets none)
            for (int i = 0; i < pages[s + 1] - pages[s]; ++i)
                if (have + i < a.max_pages) a.page_table[(int64_t)slot * a.max_pages + have + i] = a.free[pages[s] + i];
        }
    }
    // ---- what is by token ----
    const int t0 = blockIdx.x * kTableThreads, t = t0 + threadIdx.x;
    if (a.parents) {
        for (int i = threadIdx.x; i < kTableThreads + kTreeTokens; i += kTableThreads) {
            const int x = t0 - kTreeTokens + i;
            up[i] = x >= 0 && x < a.n_tokens ? a.parents[x] : -1;
        }
        __syncthreads();
    }
    if (t >= a.n_tokens) return;
    if (t >= all) {                                      // behind the last sequence
        a.token_seq[t] = a.places[t] = a.positions[t] = -1;
        a.slot_map[t] = -1;
        if (a.parents) a.ancestors[t] = 0;
        return;
    }
    const int s = sequence_of(cu, a.n_seqs, t), i = t - cu[s], length = length_of(a, s), place = length + i;
    int depth = i;
    if (a.parents) {
        uint64_t bits = 0;
        depth = 0;
        if (i < kTreeTokens) {
            bits = 1ull << i;
            int at = i;
            while (true) {                               // (a parent comes before its child, so this ends)
                const int p = up[kTreeTokens + threadIdx.x - i + at];
                if (p < 0 || p >= at) break;
                bits |= 1ull << p;
                ++depth;
                at = p;
            }
        }
        a.ancestors[t] = (int64_t)bits;
    }
    a.token_seq[t] = s;
    a.places[t] = place;
    a.positions[t] = length + depth;
    const int column = place / kPageTokens, have = pages_of(length), slot = a.slots[s];
    int64_t at = -1;
    if (place >= 0 && column < a.max_pages && slot >= 0 && slot < a.n_slots) {
        if (!a.taken || column < have) at = a.page_table[(int64_t)slot * a.max_pages + column];
        else if (pages_there(a, pages, s)) at = a.free[pages[s] + column - have];
        if (at >= 0) at = at * kPageTokens + place % kPageTokens;
    }
    a.slot_map[t] = at;
}

// ---------------------------------------------------------------------------
// Keys and values of an accepted path.  Token j of it lies at l + path[j] and goes to l + j.  Paths rise, so that path[j] >= j and what a token is written over has
// been read by a token before it: a block takes one key-value head of one layer and sequence and moves the tokens in groups, read whole before they are written.
// There is nothing to compute; the floor is every moved byte in and out, of which values, stored transposed, lie two or four bytes in a row: each moves 32 bytes both ways.
// 32 layers of one sequence, 4 tokens of 2 heads of 128: 4.3 us, a launch and the chain of three loads; 24 layers of 64 sequences, 5 tokens of 2 of 64: 12.7 us, 3,072 blocks.
// ---------------------------------------------------------------------------
constexpr int kKeepThreads = 128, kKeepLoads = 4, kKeepTensors = 8;

struct KeptTensors {
    struct Pair {
        char *k, *v;                                     // v null: keys alone
        int64_t k_lane, v_lane;                          // bytes of a layer
        int lanes, pages, kv, k_row, dv;                 // k_row: bytes of a key
        int first;                                       // number of the pair's first layer and head in the launch
    } p[kKeepTensors];
    int n;
};
struct KeepArgs {
    const int *lengths, *path, *count, *slots, *page_table;
    int n_slots, max_pages, most;
    const int64_t* rows;                                 // where the step's tokens lie, by token (below 0: nowhere); null: where the page table says
    const int* cu;
    int n_tokens;
};

template <typename K, typename V>
__global__ void __launch_bounds__(kKeepThreads)
keep_drafts_kernel(const __grid_constant__ KeptTensors t, const __grid_constant__ KeepArgs a) {
    __shared__ int64_t from[kTreeTokens], to[kTreeTokens];      // row numbers (page * 64 + place in it); -1: stays
    pdl_wait();
    const int s = blockIdx.y;
    int i = 0;
    while (i + 1 < t.n && (int)blockIdx.x >= t.p[i + 1].first) ++i;
    const KeptTensors::Pair& p = t.p[i];
    const int unit = blockIdx.x - p.first, head = unit % p.kv;
    const int64_t lane = unit / p.kv;
    const int n = min(a.count[s], a.most);
    if (n <= 1) return;                                  // (the first of a path stays where it is)
    if (threadIdx.x < kTreeTokens) {
        const int j = threadIdx.x;
        int64_t src = -1, dst = -1;
        const int x = j < n ? a.path[(int64_t)s * a.most + j] : j;
        const int slot = a.slots[s];
        if (a.rows) {
            const int first = max(0, a.cu[s]), end = min(a.cu[s + 1], a.n_tokens);
            if (j < n && x > j && x < end - first) {         // (and so j)
                const int64_t b = a.rows[first + x], c = a.rows[first + j], rows = (int64_t)p.pages * kPageTokens;
                if (b >= 0 && b < rows && c >= 0 && c < rows) {
                    src = b;
                    dst = c;
                }
            }
        } else if (j < n && x > j && slot >= 0 && slot < a.n_slots) {
            const int* table = a.page_table + (int64_t)slot * a.max_pages;
            const int64_t b = (int64_t)a.lengths[s] + x, c = (int64_t)a.lengths[s] + j;
            if (b / kPageTokens < a.max_pages && c >= 0) {
                const int pb = table[b / kPageTokens], pc = table[c / kPageTokens];
                if (pb >= 0 && pb < p.pages && pc >= 0 && pc < p.pages) {
                    src = (int64_t)pb * kPageTokens + b % kPageTokens;
                    dst = (int64_t)pc * kPageTokens + c % kPageTokens;
                }
            }
        }
        from[j] = src;
        to[j] = dst;
    }
    __syncthreads();
    // ---- keys: runs of k_row bytes ----
    {
        char* base = p.k + lane * p.k_lane;
        const int chunks = p.k_row / (int)sizeof(K), group = max(1, kKeepThreads * kKeepLoads / chunks);
        const auto at = [&](int64_t row, int c) {
            return reinterpret_cast<K*>(base + ((row / kPageTokens * p.kv + head) * kPageTokens + row % kPageTokens) * p.k_row) + c;
        };
        for (int j0 = 1; j0 < n; j0 += group) {
            const int items = min(group, n - j0) * chunks;
            for (int first = 0; first < items; first += kKeepThreads * kKeepLoads) {      // (more than one turn where a key alone is longer)
                K v[kKeepLoads];
#pragma unroll
                for (int u = 0; u < kKeepLoads; ++u) {
                    const int x = first + u * kKeepThreads + threadIdx.x;
                    if (x < items && from[j0 + x / chunks] >= 0) v[u] = *at(from[j0 + x / chunks], x % chunks);
                }
                __syncthreads();
#pragma unroll
                for (int u = 0; u < kKeepLoads; ++u) {
                    const int x = first + u * kKeepThreads + threadIdx.x;
                    if (x < items && from[j0 + x / chunks] >= 0) *at(to[j0 + x / chunks], x % chunks) = v[u];
                }
                __syncthreads();
            }
        }
    }
    if (!p.v) return;
    // ---- values: one number a channel, neighbouring threads on neighbouring tokens ----
    {
        V* base = reinterpret_cast<V*>(p.v + lane * p.v_lane);
        const auto at = [&](int64_t row, int c) { return base + ((row / kPageTokens * p.kv + head) * p.dv + c) * kPageTokens + row % kPageTokens; };
        const int group = min(n - 1, 8);                 // tokens that are read before any of them is written
        for (int j0 = 1; j0 < n; j0 += group) {
            const int here = min(group, n - j0), items = here * p.dv;
            // channels do not meet: a group's turn over all of them may be cut anywhere between channels
            const int turn = kKeepThreads * kKeepLoads / here * here;
            for (int first = 0; first < items; first += turn) {
                V v[kKeepLoads];
#pragma unroll
                for (int u = 0; u < kKeepLoads; ++u) {
                    const int y = u * kKeepThreads + threadIdx.x, x = first + y;
                    if (y < turn && x < items && from[j0 + x % here] >= 0) v[u] = *at(from[j0 + x % here], x / here);
                }
                __syncthreads();
#pragma unroll
                for (int u = 0; u < kKeepLoads; ++u) {
                    const int y = u * kKeepThreads + threadIdx.x, x = first + y;
                    if (y < turn && x < items && from[j0 + x % here] >= 0) *at(to[j0 + x % here], x / here) = v[u];
                }
            }
            __syncthreads();
        }
    }
}

}  // namespace

// All tables of one step in ``room``, one behind the other: slot map int64 [tokens], with ``parents`` ancestors int64 [tokens], sequences, positions and places int32
// [tokens], key counts [seqs], offsets [seqs + 1], and the number of pages wanted from ``free`` [1] (written if there is such a list).  Pages beyond the table's width are not
// written.
CPM_API int cpm_step_tables(const int* lengths, const int* fresh, const int* slots, int n_seqs, int n_tokens, int* page_table, int n_slots, int max_pages,
                            const int* parents, const int* free, int n_free, int hand_out, void* room, cudaStream_t stream) {
    if (n_seqs < 1 || n_seqs > kMostSeqs || n_tokens < 0 || max_pages < 1 || n_free < 0 || !room || ((uintptr_t)room & 7)) return CPM_BAD_ARGUMENT;
    if (!free && n_free > 0) return CPM_BAD_ARGUMENT;
    int64_t* const slot_map = (int64_t*)room;
    int64_t* const ancestors = parents ? slot_map + n_tokens : nullptr;
    int* const token_seq = (int*)(slot_map + (parents ? 2 : 1) * (int64_t)n_tokens);
    int *const positions = token_seq + n_tokens, *const places = positions + n_tokens, *const kv_len = places + n_tokens, *const cu = kv_len + n_seqs;
    const TableArgs a{lengths, fresh, slots, parents, free, n_free, n_seqs, n_tokens, n_slots, max_pages, page_table, cu, kv_len, token_seq, positions, places,
                      hand_out ? cu + n_seqs + 1 : nullptr, slot_map, ancestors};
    const int blocks = (max(n_tokens, n_seqs + 1) + kTableThreads - 1) / kTableThreads;
    cpm_launch(kLaunchOther, step_tables_kernel, dim3(blocks), kTableThreads, (size_t)(n_seqs + 1) * 8, stream, a);
    return launch_status();
}

// pairs: n times {keys, values or 0, bytes of a layer's keys, of its values, layers, pages, key-value heads, bytes of a key, value channels}, each a 64-bit number.
// ``element``: bytes of a number.  ``rows`` with ``cu`` and n_tokens, or null: see KeepArgs.
CPM_API int cpm_keep_drafts(const int64_t* pairs, int n_pairs, int element, const int* lengths, const int* path, const int* count, const int* slots,
                            const int* page_table, int n_slots, int max_pages, int n_seqs, int most, const int64_t* rows, const int* cu, int n_tokens, cudaStream_t stream) {
    if (n_pairs < 0 || n_pairs > kKeepTensors || n_seqs < 0 || n_seqs > 65535 || most < 1 || most > kTreeTokens || max_pages < 1) return CPM_BAD_ARGUMENT;
    if (element != 2 && element != 4) return CPM_BAD_ARGUMENT;
    if (n_seqs == 0 || most == 1) return CPM_OK;
    KeptTensors t = {};
    int64_t units = 0, bits = 0;
    for (int i = 0; i < n_pairs; ++i) {
        const int64_t* p = pairs + 9 * i;
        if (p[4] < 0 || p[5] < 0 || p[5] > 0x7fffffff || p[6] < 1 || p[7] < element || p[8] < 0 || p[7] > (1 << 20) || p[8] > (1 << 20)) return CPM_BAD_ARGUMENT;
        t.p[i] = KeptTensors::Pair{reinterpret_cast<char*>(p[0]), reinterpret_cast<char*>(p[1]), p[2], p[3], (int)p[4], (int)p[5], (int)p[6], (int)p[7], (int)p[8],
                                   (int)units};
        units += p[4] * p[6];
        bits |= p[0] | p[2] | p[7];
        if (units > 0x7fffffff) return CPM_BAD_ARGUMENT;
    }
    if (units == 0) return CPM_OK;
    t.n = n_pairs;
    if (rows && !cu) return CPM_BAD_ARGUMENT;
    const KeepArgs a{lengths, path, count, slots, page_table, n_slots, max_pages, most, rows, cu, n_tokens};
    const dim3 grid((unsigned)units, n_seqs);
    const bool whole = (bits & 15) == 0;                 // keys that begin and end on 16 bytes
    if (element == 2) {
        if (whole) cpm_launch(kLaunchOther, keep_drafts_kernel<uint4, uint16_t>, grid, kKeepThreads, 0, stream, t, a);
        else cpm_launch(kLaunchOther, keep_drafts_kernel<uint16_t, uint16_t>, grid, kKeepThreads, 0, stream, t, a);
    } else {
        if (whole) cpm_launch(kLaunchOther, keep_drafts_kernel<uint4, uint32_t>, grid, kKeepThreads, 0, stream, t, a);
        else cpm_launch(kLaunchOther, keep_drafts_kernel<uint32_t, uint32_t>, grid, kKeepThreads, 0, stream, t, a);
    }
    return launch_status();
}
