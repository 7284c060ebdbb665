// Attention of a few tokens a sequence over the paged cache, in fp32 arithmetic: the 32-bit path, and the plain twin of the tensor-core kernel.
//
//     o_t = sum_j p_j v_j,  p = softmax over the keys j that token t sees of  q_t . k_j * scale
//
// A sequence of kv_len keys brings its last n tokens at once.  A token sees every key before them, and of the n either those up to itself or those whose bit is
// set in its word of 64 (its ancestors in a tree of drafted tokens, and itself).  A sequence whose slot is none has no keys.  A row that sees nothing gives zeros.  What a key holds that a row does not see
// never reaches it, whatever it is: scores are replaced, and of the tokens' own values (and what lies behind them in their page), which rows see or not, those that
// are no finite numbers are taken out of the tile and added to the rows that see them at the end.
//
// All query heads of a key-value head and all tokens are rows of one matrix (row = token * group + head), so that a sequence's keys are read once for
// 64 rows and not once a token.  A block takes 32 or 64 rows and a share of the pages: scores of 64 keys (a thread: 8 rows of one or two keys), the softmax (a warp: an
// eighth of the rows), weighted values (a thread: some rows of one channel), all operands in shared memory.  Few rows and many keys: the pages are shared out over blocks, whose
// parts a second kernel adds up.
//
// Bound by FMA and shared memory, and with few rows by the chain of one page: 3 sequences of 300 to 2,500 keys, 7 tokens of 16 heads on 2 of 64 in fp32 take 27 us, of which
// a page is 10 to 11 (scores 4.7, softmax 2.1, values 3 to 4); the keys and values alone would be a microsecond.  Blocks of 32 rows took 33 us there, of 64 27.
#include "common.cuh"

CPM_BOUNDS_TU(draft_attention)

namespace {

constexpr int kThreads = 256;
constexpr int kLine = kPageTokens + 4;                  // floats of a row of scores, and of a channel's values

struct DraftArgs {
    const void *q, *k, *v;
    void* out;
    const int *kv_len, *cu, *slots, *page_table;
    const int64_t* ancestors;                           // null: every token sees those up to itself
    float* parts;                                       // [share][token][head][d + 2]: values, maximum, sum; null: one share
    int n_slots, max_pages, n_pages, n_tokens, n_heads, n_kv, group, d, most;
    float scale;
};

// floats of a key's line: an odd number of 16 bytes, so that neighbouring keys' lie in different banks
__host__ __device__ constexpr int key_line(int d) { return (d / 4) % 2 ? d : d + 4; }
__host__ __device__ constexpr int draft_smem_floats(int rows, int d) {
    return rows * d + kPageTokens * key_line(d) + d * kLine + rows * kLine + 3 * rows;
}

// J: rows of a block by 32, and keys of a thread.  RPT: rows that a thread adds up of one channel: 32 J / RPT groups of threads have 8 RPT / J channels.
template <typename T, int RPT, int J>
__global__ void __launch_bounds__(kThreads)
draft_attention_kernel(const __grid_constant__ DraftArgs a) {
    constexpr int kRows = 32 * J;
    extern __shared__ __align__(16) float draft_smem[];
    __shared__ int odd;                                 // whether a value among the step's tokens is no finite number
    const int d = a.d, line = key_line(d), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    float *qs = draft_smem, *ks = qs + kRows * d, *vs = ks + kPageTokens * line, *ps = vs + d * kLine, *top = ps + kRows * kLine, *sum = top + kRows, *back = sum + kRows;
    pdl_launch_dependents();
    pdl_wait();
    const int s = blockIdx.y, head_kv = blockIdx.x % a.n_kv, r0 = blockIdx.x / a.n_kv * kRows;
    const int begin = max(0, min(a.cu[s], a.n_tokens)), n = max(0, min(min(a.cu[s + 1], a.n_tokens) - begin, a.most));
    const int rows = min(kRows, n * a.group - r0);
    if (rows <= 0) return;
    const int slot = a.slots[s], held = a.kv_len[s];
    const int kv_len = slot >= 0 && slot < a.n_slots ? max(0, min(held, a.max_pages * kPageTokens)) : 0, history = kv_len - n;       // (negative: the first tokens are none of the keys)
    const int n_keys = a.ancestors ? kv_len : min(kv_len, history + (r0 + rows - 1) / a.group + 1);
    const int all = (n_keys + kPageTokens - 1) / kPageTokens, share = (all + gridDim.z - 1) / gridDim.z;
    const int page0 = min(all, (int)blockIdx.z * share), page1 = min(all, page0 + share);
    const int* table = a.page_table + (int64_t)slot * a.max_pages;           // (followed where there are keys)
    const T *q = static_cast<const T*>(a.q), *k = static_cast<const T*>(a.k), *v = static_cast<const T*>(a.v);

    // whether row r sees key j of the step's tokens
    const auto sees = [&](int r, int j) {
        const int token = (r0 + r) / a.group;
        return a.ancestors ? (bool)((uint64_t)a.ancestors[begin + token] >> (j - history) & 1) : j - history <= token;
    };
    const auto row_of = [&](int r) { return ((int64_t)(begin + (r0 + r) / a.group) * a.n_heads + head_kv * a.group + (r0 + r) % a.group); };
    for (int i = tid; i < kRows * (d / 4); i += kThreads) {
        const int r = i / (d / 4), c = i % (d / 4) * 4;
        *reinterpret_cast<float4*>(qs + r * d + c) = r < rows ? load4(q + row_of(r) * d + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (tid < kRows) {
        top[tid] = -INFINITY;
        sum[tid] = 0.f;
    }
    if (tid == 0) odd = 0;
    const int channel = tid % (8 * RPT / J), o0 = tid / (8 * RPT / J) * RPT;     // of the weighted values: a channel, and rows from o0 on
    float o[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i) o[i] = 0.f;

#pragma unroll 1
    for (int page = page0; page < page1; ++page) {
        const int64_t number = max(0, min(CPM_PAGE(table, page, a.max_pages), a.n_pages - 1));
        const int key0 = page * kPageTokens;
        __syncthreads();                                // the last page's values have been used
        const T* from = k + page_row_offset((int)number, head_kv, 0, a.n_kv, d);
#pragma unroll 4
        for (int i = tid; i < kPageTokens * (d / 4); i += kThreads) {
            const int j = i / (d / 4), c = i % (d / 4) * 4;
            *reinterpret_cast<float4*>(ks + j * line + c) = load4(from + j * d + c);
        }
        const T* values = v + value_offset((int)number, head_kv, 0, 0, a.n_kv, d);
        const bool own = key0 + kPageTokens > history;  // tokens of the step, or what lies behind them
#pragma unroll 4
        for (int i = tid; i < d * (kPageTokens / 4); i += kThreads) {
            const int c = i / (kPageTokens / 4), j = i % (kPageTokens / 4) * 4;
            float4 x = load4(values + c * kPageTokens + j);
            if (own) {
                float* e = reinterpret_cast<float*>(&x);
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (key0 + j + u >= kv_len) e[u] = 0.f;
                    else if (key0 + j + u >= history && !(fabsf(e[u]) < INFINITY)) {
                        e[u] = 0.f;
                        odd = 1;
                    }
            }
            *reinterpret_cast<float4*>(vs + c * kLine + j) = x;
        }
        __syncthreads();
        // ---- scores: eight rows of one or two keys ----
        {
            const int j = tid % (kPageTokens / J), first = tid / (kPageTokens / J) * 8;
            float x[J][8];
#pragma unroll
            for (int u = 0; u < J; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[u][i] = 0.f;
#pragma unroll 2
            for (int c = 0; c < d; c += 4) {
                float4 kk[J];
#pragma unroll
                for (int u = 0; u < J; ++u) kk[u] = *reinterpret_cast<const float4*>(ks + (j + 32 * u) * line + c);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 qq = *reinterpret_cast<const float4*>(qs + (first + i) * d + c);
#pragma unroll
                    for (int u = 0; u < J; ++u) {
                        x[u][i] = fmaf(qq.x, kk[u].x, x[u][i]);
                        x[u][i] = fmaf(qq.y, kk[u].y, x[u][i]);
                        x[u][i] = fmaf(qq.z, kk[u].z, x[u][i]);
                        x[u][i] = fmaf(qq.w, kk[u].w, x[u][i]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < J; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int key = key0 + j + 32 * u;
                    const bool seen = first + i < rows && key < kv_len && (key < history || sees(first + i, key));
                    ps[(first + i) * kLine + j + 32 * u] = seen ? x[u][i] * a.scale : -INFINITY;
                }
        }
        __syncthreads();
        // ---- softmax: a warp an eighth of the rows, a lane two keys ----
#pragma unroll
        for (int i = 0; i < kRows / 8; ++i) {
            if (warp * (kRows / 8) + i >= rows) break;
            const int r = warp * (kRows / 8) + i;
            const float x0 = ps[r * kLine + lane], x1 = ps[r * kLine + 32 + lane];
            const float was = top[r], now = fmaxf(was, warp_max(fmaxf(x0, x1))), use = now == -INFINITY ? 0.f : now;
            const float p0 = expf(x0 - use), p1 = expf(x1 - use), by = was == -INFINITY ? 0.f : expf(was - use), all_p = warp_sum(p0 + p1);
            ps[r * kLine + lane] = p0;
            ps[r * kLine + 32 + lane] = p1;
            if (lane == 0) {
                top[r] = now;
                back[r] = by;
                sum[r] = sum[r] * by + all_p;
            }
        }
        __syncthreads();
        // ---- weighted values: one channel of some rows ----
        if (channel < d) {
#pragma unroll
            for (int i = 0; i < RPT; ++i) o[i] *= back[o0 + i];
#pragma unroll 2
            for (int j = 0; j < kPageTokens; j += 4) {
                const float4 x = *reinterpret_cast<const float4*>(vs + channel * kLine + j);
#pragma unroll
                for (int i = 0; i < RPT; ++i) {
                    const float4 p = *reinterpret_cast<const float4*>(ps + (o0 + i) * kLine + j);
                    o[i] = fmaf(p.x, x.x, o[i]);
                    o[i] = fmaf(p.y, x.y, o[i]);
                    o[i] = fmaf(p.z, x.z, o[i]);
                    o[i] = fmaf(p.w, x.w, o[i]);
                }
            }
        }
    }
    __syncthreads();
    if (channel >= d) return;
    if (odd) {
        // values that are no finite numbers, to the rows that see them
#pragma unroll 1
        for (int j = max(max(0, history), page0 * kPageTokens); j < min(n_keys, page1 * kPageTokens); ++j) {
            const int64_t number = max(0, min(CPM_PAGE(table, j / kPageTokens, a.max_pages), a.n_pages - 1));
            const float x = to_f32(v[value_offset((int)number, head_kv, channel, j % kPageTokens, a.n_kv, d)]);
            if (fabsf(x) < INFINITY) continue;
            for (int i = 0; i < RPT; ++i)
                if (o0 + i < rows && sees(o0 + i, j)) o[i] += x;
        }
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int r = o0 + i;
        if (r >= rows) break;
        const int64_t row = row_of(r);
        if (a.parts) {
            float* to = a.parts + ((int64_t)blockIdx.z * a.n_tokens * a.n_heads + row) * (d + 2);
            to[channel] = o[i];
            if (channel == 0) {
                to[d] = top[r];
                to[d + 1] = sum[r];
            }
        } else {
            static_cast<T*>(a.out)[row * d + channel] = from_f32<T>(sum[r] == 0.f ? o[i] : o[i] / sum[r]);
        }
    }
}

// Adds up the shares of a row: a block a row, a warp every eighth share.  Rows of no sequence are left as they are.
template <typename T>
__global__ void __launch_bounds__(kThreads)
draft_join_kernel(const __grid_constant__ DraftArgs a, int shares) {
    constexpr int kWarps = kThreads / 32, kDims = 8;      // d <= 256
    __shared__ float values[kWarps][32 * kDims];
    pdl_launch_dependents();
    pdl_wait();
    const int s = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = a.d;
    const int begin = max(0, min(a.cu[s], a.n_tokens)), n = max(0, min(min(a.cu[s + 1], a.n_tokens) - begin, a.most));
    if ((int)blockIdx.x >= n * a.n_heads) return;
    const int64_t row = (int64_t)begin * a.n_heads + blockIdx.x, apart = (int64_t)a.n_tokens * a.n_heads * (d + 2);
    const float* part = a.parts + row * (d + 2);
    // a lane has the maximum and the sum of two shares, and their weight in the result
    float m[2], w[2], l = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) m[h] = lane + 32 * h < shares ? part[(lane + 32 * h) * apart + d] : -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h) w[h] = lane + 32 * h < shares ? part[(lane + 32 * h) * apart + d + 1] : 0.f;
    const float top = warp_max(fmaxf(m[0], m[1])), use = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float by = expf(m[h] - use);
        l += w[h] * by;
        w[h] = by;
    }
    l = warp_sum(l);
    float o[kDims];
#pragma unroll
    for (int i = 0; i < kDims; ++i) o[i] = 0.f;
#pragma unroll 4
    for (int z = warp; z < shares; z += kWarps) {
        const float by = __shfl_sync(0xffffffffu, z < 32 ? w[0] : w[1], z & 31);
#pragma unroll
        for (int i = 0; i < kDims; ++i)
            if (lane + 32 * i < d) o[i] = fmaf(part[z * apart + lane + 32 * i], by, o[i]);
    }
#pragma unroll
    for (int i = 0; i < kDims; ++i)
        if (lane + 32 * i < d) values[warp][lane + 32 * i] = o[i];
    __syncthreads();
    const int c = threadIdx.x;
    if (c >= d) return;
    float y = 0.f;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) y += values[x][c];
    static_cast<T*>(a.out)[row * d + c] = from_f32<T>(l == 0.f ? y : y / l);
}

template <typename T, int RPT, int J>
int launch(const DraftArgs& a, int n_seqs, int shares, cudaStream_t stream) {
    static bool done[kMaxDevices];
    const int most_bytes = draft_smem_floats(32 * J, 8 * RPT / J) * 4, status = ensure_dynamic_smem(draft_attention_kernel<T, RPT, J>, most_bytes, done);
    if (status != CPM_OK) return status;
    const int64_t tiles = (int64_t)((a.most * a.group + 32 * J - 1) / (32 * J)) * a.n_kv;
    if (tiles > 0x7fffffff || n_seqs > 65535) return CPM_BAD_ARGUMENT;
    cpm_launch(kLaunchAttention, draft_attention_kernel<T, RPT, J>, dim3((unsigned)tiles, n_seqs, shares), kThreads, (size_t)draft_smem_floats(32 * J, a.d) * 4, stream, a);
    if (shares > 1) {
        if ((int64_t)a.most * a.n_heads > 0x7fffffff) return CPM_BAD_ARGUMENT;
        cpm_launch(kLaunchAttention, draft_join_kernel<T>, dim3((unsigned)(a.most * a.n_heads), n_seqs), kThreads, 0, stream, a, shares);
    }
    return launch_status();
}

// Rows of a block: 64 where there are more than 32 and a thread's sums of 64 rows have room in its registers.
__host__ constexpr bool wide_rows(int most, int group, int d) { return most * group > 32 && d <= 128; }

template <typename T>
int by_size(const DraftArgs& a, int n_seqs, int shares, cudaStream_t stream) {
    const bool wide = wide_rows(a.most, a.group, a.d);
    if (a.d <= 32) return wide ? launch<T, 8, 2>(a, n_seqs, shares, stream) : launch<T, 4, 1>(a, n_seqs, shares, stream);
    if (a.d <= 64) return wide ? launch<T, 16, 2>(a, n_seqs, shares, stream) : launch<T, 8, 1>(a, n_seqs, shares, stream);
    if (a.d <= 128) return wide ? launch<T, 32, 2>(a, n_seqs, shares, stream) : launch<T, 16, 1>(a, n_seqs, shares, stream);
    return launch<T, 32, 1>(a, n_seqs, shares, stream);
}

}  // namespace

// q, out [tokens, heads, d]; k [pages, kv, 64, d], v [pages, kv, d, 64]; ``parts``: shares * tokens * heads * (d + 2) floats where there is more than one share.
CPM_API int cpm_draft_attention_generic(const void* q, const void* k, const void* v, void* out, const int* kv_len, const int* cu, const int* slots,
                                        const int* page_table, int n_slots, int max_pages, int n_pages, const int64_t* ancestors, float* parts, int shares, int n_tokens,
                                        int n_seqs, int most, int n_heads, int n_kv, int d, float scale, int dtype, cudaStream_t stream) {
    if (n_tokens <= 0 || n_seqs <= 0) return CPM_OK;
    if (d < 4 || d > 256 || d % 4 || n_kv < 1 || n_heads < 1 || n_heads % n_kv || most < 1 || most > 64 || max_pages < 1 || max_pages > 0x7fffffff / kPageTokens || n_pages < 1) return CPM_BAD_ARGUMENT;
    if (shares < 1 || shares > 64 || (shares > 1) != (parts != nullptr)) return CPM_BAD_ARGUMENT;
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) return CPM_BAD_ARGUMENT;
    const DraftArgs a{q, k, v, out, kv_len, cu, slots, page_table, ancestors, parts, n_slots, max_pages, n_pages, n_tokens, n_heads, n_kv, n_heads / n_kv, d, most, scale};
    return dtype == CPM_BF16 ? by_size<bf16>(a, n_seqs, shares, stream) : by_size<float>(a, n_seqs, shares, stream);
}
