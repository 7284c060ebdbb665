// Storing keys and values into the 4-bit cache, and reading them back.
//
// Store: q and k of a token are rotated (pairs (c, c + d/2), angle = position * inv_freq[c], cos and sin times ``magnitude``), q goes out in the
// compute type, k and v become codes.  Of these a warp takes one head row; a lane holds d/32 neighbouring channels, so that a pair's other half
// and a half row's 16 lanes are one shuffle away.  The codes meet in shared memory, from where lanes write whole words (keys:
// a token's own; values: 16 bits, for the other half of the word is the neighbouring token's, which another block may be writing).
// What a token cannot do without: its projections, q out, d + 16 bytes per key-value head.
// 2,048 tokens of 32 heads on 2 of 128: 9.1 us (fp32 10.7) and 3.1 for reading them back, 12.4 one behind the other, 3.1 TB/s; 64 tokens of 16 heads on 2 of
// 64: 2.8 and 1.9, 4.5 one behind the other.  Bound by latency: a block's
// tokens are one, and its angles (sincosf) and its rows' loads lie in one chain; with all rows alike, a warp to a row, it took 15.6 us.
#include "kv4.cuh"

CPM_BOUNDS_TU(kv4_store)

namespace {

constexpr int kStoreWarps = 8;

template <typename T, int E>
__device__ __forceinline__ void load_row(const T* p, float (&x)[E]) {
    if constexpr (E == 4) {
        const float4 v = load4(p);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = to_f32(p[i]);
    }
}
template <typename T, int E>
__device__ __forceinline__ void store_row(T* p, const float (&x)[E]) {
    if constexpr (E == 4) {
        store4(p, make_float4(x[0], x[1], x[2], x[3]));
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) p[i] = from_f32<T>(x[i]);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kStoreWarps * 32)
rope_store_kv4_kernel(const T* __restrict__ qkv, T* __restrict__ q_out, uint8_t* __restrict__ records, const int* __restrict__ positions,
                      const int* __restrict__ token_seq, const int* __restrict__ slots, const int* __restrict__ page_table, int max_pages,
                      const float* __restrict__ inv_freq, float magnitude, int n_heads, int n_kv, int rows_per_block) {
    using L = Kv4<D>;
    constexpr int E = D / 32, HALF = D / 2;
    __shared__ float cs[HALF], sn[HALF];
    __shared__ alignas(8) uint8_t codes[kStoreWarps][D];
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pos = positions[t];
    const int n_all = n_heads + (records ? 2 * n_kv : 0);
    const int begin = blockIdx.y * rows_per_block, end = min(n_all, begin + rows_per_block);
    const T* row = qkv + (int64_t)t * (n_heads + 2 * n_kv) * D;
    // q: half a warp to a row, a lane to E pairs of channels, the same ones in every row; the first row is on its way while the angles are formed
    const int c0 = (lane & 15) * E, q_end = min(end, n_heads);
    int hq = begin + 2 * warp + (lane >> 4);
    float qa[E], qb[E];
    const auto load_q = [&]() {
        if (hq >= q_end) return;
        load_row<T, E>(row + (int64_t)hq * D + c0, qa);
        load_row<T, E>(row + (int64_t)hq * D + HALF + c0, qb);
    };
    load_q();
    if (inv_freq) {
        for (int c = threadIdx.x; c < HALF; c += blockDim.x) {
            float s, k;
            sincosf((float)pos * inv_freq[c], &s, &k);
            cs[c] = __fmul_rn(k, magnitude);
            sn[c] = __fmul_rn(s, magnitude);
        }
        __syncthreads();
    }
    if (hq < q_end) {
        float k[E], n[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            k[i] = inv_freq ? cs[c0 + i] : 1.f;
            n[i] = inv_freq ? sn[c0 + i] : 0.f;
        }
#pragma unroll 1
        while (hq < q_end) {
            float a[E], b[E];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                a[i] = inv_freq ? __fsub_rn(__fmul_rn(qa[i], k[i]), __fmul_rn(qb[i], n[i])) : qa[i];
                b[i] = inv_freq ? __fadd_rn(__fmul_rn(qb[i], k[i]), __fmul_rn(qa[i], n[i])) : qb[i];
            }
            T* to = q_out + ((int64_t)t * n_heads + hq) * D + c0;
            hq += 2 * kStoreWarps;
            load_q();
            store_row<T, E>(to, a);
            store_row<T, E>(to + HALF, b);
        }
    }
    if (end <= n_heads) return;
    uint8_t* const page = records + (int64_t)CPM_PAGE(page_table + (int64_t)slots[token_seq[t]] * max_pages, pos / kPageTokens, max_pages) * n_kv * L::kBytes;
    // k and v: a warp to a row, the last warps first, which have had the fewest rows of q
    for (int h = max(begin, n_heads) + kStoreWarps - 1 - warp; h < end; h += kStoreWarps) {
        float x[E];
        load_row<T, E>(row + (int64_t)h * D + lane * E, x);
        if (inv_freq && h < n_heads + n_kv) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float other = __shfl_xor_sync(0xffffffffu, x[i], 16);
                const int c = (lane & 15) * E + i;
                // the lower half: x cos - other sin; the upper one: x cos + other sin
                const float a = __fmul_rn(x[i], cs[c]), b = __fmul_rn(other, sn[c]);
                x[i] = lane < 16 ? __fsub_rn(a, b) : __fadd_rn(a, b);
            }
        }
        const bool values = h >= n_heads + n_kv;
        const int head = h - n_heads - (values ? n_kv : 0);
        float lo = x[0], hi = x[0];
#pragma unroll
        for (int i = 1; i < E; ++i) { lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]); }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        float sum = 0.f;                                    // a channel that is no number makes its half row one too
#pragma unroll
        for (int i = 0; i < E; ++i) sum += x[i] * 0.f;
        const bool bad = __ballot_sync(0xffffffffu, sum != 0.f) & (lane < 16 ? 0xffffu : 0xffff0000u);
        const uint32_t par = bad ? 0x7fc07fc0u : kv4_parameters(lo, hi);
        const float m = kv4_middle(par), inverse = kv4_inverse(kv4_scale(par));
#pragma unroll
        for (int i = 0; i < E; ++i) codes[warp][lane * E + i] = (uint8_t)kv4_code(x[i], m, inverse);
        __syncwarp();
        const int tok = pos % kPageTokens, slice = tok >> 4, r = tok & 15, upper = r >> 3;
        uint8_t* rec = page + (int64_t)head * L::kBytes;
        if ((lane & 15) == 0)
            *reinterpret_cast<uint32_t*>(rec + (values ? L::kValueParams : L::kKeyParams) + tok * 8 + (lane >> 4) * 4) = par;
        if (!values) {
            if (lane < D / 8) {
                const int pair = lane >> 2, j = lane & 3;
                const uint32_t a = *reinterpret_cast<const uint32_t*>(&codes[warp][32 * pair + 4 * j]);
                const uint32_t b = *reinterpret_cast<const uint32_t*>(&codes[warp][32 * pair + 16 + 4 * j]);
                // channels 0, 2 of a in nibbles 0, 1 and channels 1, 3 in nibbles 4, 5; those of b two nibbles higher
                const auto spread = [](uint32_t v) { return (v & 15u) | ((v >> 12) & 0xf0u) | ((v << 8) & 0xf0000u) | ((v >> 4) & 0xf00000u); };
                *reinterpret_cast<uint32_t*>(rec + L::word(slice, pair, (r & 7) * 4 + j, upper)) = spread(a) | (spread(b) << 8);
            }
        } else if (lane < D / 4) {
            const int pair = lane >> 3, g = lane & 7;
            const uint32_t a = *reinterpret_cast<const uint16_t*>(&codes[warp][32 * pair + 2 * g]);
            const uint32_t b = *reinterpret_cast<const uint16_t*>(&codes[warp][32 * pair + 16 + 2 * g]);
            const uint32_t half = (a & 15u) | ((a >> 4) & 0xf0u) | ((b & 15u) << 8) | ((b << 4) & 0xf000u);
            *reinterpret_cast<uint16_t*>(rec + L::kValues + L::word(slice, pair, g * 4 + ((r & 7) >> 1), upper) + 2 * (r & 1)) = (uint16_t)half;
        }
        __syncwarp();
    }
}

// A warp reads one token's row of one key-value head, keys (blockIdx.y even) or values.
template <typename T, int D>
__global__ void __launch_bounds__(kStoreWarps * 32)
kv4_values_kernel(const uint8_t* __restrict__ records, T* __restrict__ k_out, T* __restrict__ v_out, const int* __restrict__ positions,
                  const int* __restrict__ token_seq, const int* __restrict__ slots, const int* __restrict__ page_table, int max_pages,
                  int n_tokens, int n_kv) {
    using L = Kv4<D>;
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * kStoreWarps + (threadIdx.x >> 5);
    if (row >= (int64_t)n_tokens * n_kv * 2) return;
    const int values = (int)(row & 1), head = (int)((row >> 1) % n_kv), t = (int)((row >> 1) / n_kv);
    const int pos = positions[t];
    const int page = CPM_PAGE(page_table + (int64_t)slots[token_seq[t]] * max_pages, pos / kPageTokens, max_pages);
    const uint8_t* rec = records + ((int64_t)page * n_kv + head) * L::kBytes;
    const int tok = pos % kPageTokens, slice = tok >> 4, r = tok & 15, upper = r >> 3;
    const uint2 par = *reinterpret_cast<const uint2*>(rec + (values ? L::kValueParams : L::kKeyParams) + tok * 8);
    const auto value = [&](uint32_t code, int c) { return kv4_value(code & 15u, c < D / 2 ? par.x : par.y); };
    T* out = (values ? v_out : k_out) + ((int64_t)t * n_kv + head) * D;
    if (!values) {
        if (lane < D / 8) {
            const int pair = lane >> 2, j = lane & 3;
            const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + L::word(slice, pair, (r & 7) * 4 + j, upper));
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
                const uint32_t v = w >> (8 * odd);
                const int c = 32 * pair + 16 * odd + 4 * j;
                store4(out + c, make_float4(value(v, c), value(v >> 16, c), value(v >> 4, c), value(v >> 20, c)));
            }
        }
    } else if (lane < D / 4) {
        const int pair = lane >> 3, g = lane & 7;
        const uint32_t w = *reinterpret_cast<const uint16_t*>(rec + L::kValues + L::word(slice, pair, g * 4 + ((r & 7) >> 1), upper) + 2 * (r & 1));
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
            const uint32_t v = w >> (8 * odd);
            const int c = 32 * pair + 16 * odd + 2 * g;
            out[c] = from_f32<T>(value(v, c));
            out[c + 1] = from_f32<T>(value(v >> 4, c));
        }
    }
}

template <typename T, int D>
int store(const void* qkv, void* q_out, void* records, const int* positions, const int* token_seq, const int* slots, const int* page_table,
          int max_pages, const float* inv_freq, float magnitude, int n_tokens, int n_heads, int n_kv, cudaStream_t stream) {
    const int n_all = n_heads + (records ? 2 * n_kv : 0);
    // few tokens: one row a warp, so that the rows of a token fill several blocks
    const int rows = n_tokens >= 64 ? n_all : kStoreWarps;
    const dim3 grid(n_tokens, (n_all + rows - 1) / rows);
    if (grid.y > 65535) return CPM_BAD_ARGUMENT;
    cpm_launch(kLaunchRope, rope_store_kv4_kernel<T, D>, grid, kStoreWarps * 32, 0, stream, (const T*)qkv, (T*)q_out, (uint8_t*)records, positions,
               token_seq, slots, page_table, max_pages, inv_freq, magnitude, n_heads, n_kv, rows);
    return launch_status();
}

template <typename T, int D>
int values(const void* records, void* k_out, void* v_out, const int* positions, const int* token_seq, const int* slots, const int* page_table,
           int max_pages, int n_tokens, int n_kv, cudaStream_t stream) {
    const int64_t rows = (int64_t)n_tokens * n_kv * 2;
    const int64_t blocks = (rows + kStoreWarps - 1) / kStoreWarps;
    if (blocks > 0x7fffffff) return CPM_BAD_ARGUMENT;
    cpm_launch(kLaunchRope, kv4_values_kernel<T, D>, dim3((unsigned)blocks), kStoreWarps * 32, 0, stream, (const uint8_t*)records, (T*)k_out, (T*)v_out,
               positions, token_seq, slots, page_table, max_pages, n_tokens, n_kv);
    return launch_status();
}

}  // namespace

#define KV4_BY_HEAD_SIZE(T, CALL)          \
    switch (d) {                           \
        case 32: return CALL(T, 32);       \
        case 64: return CALL(T, 64);       \
        case 96: return CALL(T, 96);       \
        case 128: return CALL(T, 128);     \
        default: return CPM_BAD_ARGUMENT;  \
    }

CPM_API int cpm_rope_store_kv4(const void* qkv, void* q_out, void* records, const int* positions, const int* token_seq, const int* slots,
                               const int* page_table, int max_pages, const float* inv_freq, float magnitude, int n_tokens, int n_heads, int n_kv,
                               int d, int dtype, cudaStream_t stream) {
    if (n_tokens <= 0) return CPM_OK;
    if (n_heads < 1 || n_kv < 1 || (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)records) & 15)) return CPM_BAD_ARGUMENT;
#define CALL(T, D) store<T, D>(qkv, q_out, records, positions, token_seq, slots, page_table, max_pages, inv_freq, magnitude, n_tokens, n_heads, n_kv, stream)
    if (dtype == CPM_BF16) KV4_BY_HEAD_SIZE(bf16, CALL)
    KV4_BY_HEAD_SIZE(float, CALL)
#undef CALL
}

CPM_API int cpm_kv4_values(const void* records, void* k_out, void* v_out, const int* positions, const int* token_seq, const int* slots,
                           const int* page_table, int max_pages, int n_tokens, int n_kv, int d, int dtype, cudaStream_t stream) {
    if (n_tokens <= 0) return CPM_OK;
    if (n_kv < 1 || (((uintptr_t)records | (uintptr_t)k_out | (uintptr_t)v_out) & 15)) return CPM_BAD_ARGUMENT;
#define CALL(T, D) values<T, D>(records, k_out, v_out, positions, token_seq, slots, page_table, max_pages, n_tokens, n_kv, stream)
    if (dtype == CPM_BF16) KV4_BY_HEAD_SIZE(bf16, CALL)
    KV4_BY_HEAD_SIZE(float, CALL)
#undef CALL
}
