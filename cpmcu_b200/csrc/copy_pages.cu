// Copies of pages inside the cache's tensors: a sequence that is forked takes a copy of its last, partial page, a cache that is
// compacted moves pages into holes.  One launch copies the listed pages in all layers of all tensors; there is nothing to compute, so
// the floor is every byte once in and once out.  A block takes up to kCopyBytes of one page of one layer, and a thread has four
// 16-byte loads under way.
// Closing up a cache of 600 pages (250 moves in 32 layers of keys and values, 1.05 GB in and out): 160 us, 6.5 TB/s; a page of 24 layers for seven further
// answers (6.3 MB) 3.1 us, a launch's own time.
#include "common.cuh"

namespace {

constexpr int kCopyThreads = 256, kCopyLoads = 4;
constexpr int kCopyTensors = 8;

struct PagedTensor {
    char* base;
    int64_t layer_bytes, page_bytes;
    int64_t first_block;        // number of the tensor's first block in the launch
    int n_pages, parts;         // parts: blocks per page and layer
};
struct PagedTensors { PagedTensor t[kCopyTensors]; int n; };

template <typename V>
__global__ void __launch_bounds__(kCopyThreads)
copy_pages_kernel(const __grid_constant__ PagedTensors tensors, const int* __restrict__ src, const int* __restrict__ dst, int n_moves) {
    pdl_launch_dependents();
    pdl_wait();
    int k = 0;
    while (k + 1 < tensors.n && (int64_t)blockIdx.x >= tensors.t[k + 1].first_block) ++k;
    const PagedTensor& a = tensors.t[k];
    int64_t unit = (int64_t)blockIdx.x - a.first_block;
    const int part = (int)(unit % a.parts);
    unit /= a.parts;
    const int move = (int)(unit % n_moves);
    const int64_t layer = unit / n_moves;
    const int from = src[move], to = dst[move];
    if (from < 0 || from >= a.n_pages || to < 0 || to >= a.n_pages || from == to) return;      // no page of this tensor
    const int64_t n = a.page_bytes / (int64_t)sizeof(V);
    const int64_t begin = (int64_t)part * (kCopyThreads * kCopyLoads);
    const V* in = reinterpret_cast<const V*>(a.base + layer * a.layer_bytes + from * a.page_bytes);
    V* out = reinterpret_cast<V*>(a.base + layer * a.layer_bytes + to * a.page_bytes);
    V v[kCopyLoads];
#pragma unroll
    for (int u = 0; u < kCopyLoads; ++u) {
        const int64_t i = begin + u * kCopyThreads + threadIdx.x;
        if (i < n) v[u] = in[i];
    }
#pragma unroll
    for (int u = 0; u < kCopyLoads; ++u) {
        const int64_t i = begin + u * kCopyThreads + threadIdx.x;
        if (i < n) out[i] = v[u];
    }
}

template <typename V>
int launch(const PagedTensors& t, int64_t blocks, const int* src, const int* dst, int n_moves, cudaStream_t stream) {
    if (blocks > 0x7fffffff) return CPM_BAD_ARGUMENT;
    cpm_launch(kLaunchOther, copy_pages_kernel<V>, dim3((unsigned)blocks), kCopyThreads, 0, stream, t, src, dst, n_moves);
    return launch_status();
}

}  // namespace

// tensors: n times {base, bytes of a layer, bytes of a page, layers, pages}, each a 64-bit number.
CPM_API int cpm_copy_pages(const int64_t* tensors, int n_tensors, const int* src, const int* dst, int n_moves, cudaStream_t stream) {
    if (n_tensors < 0 || n_tensors > kCopyTensors || n_moves < 0) return CPM_BAD_ARGUMENT;
    if (n_moves == 0 || n_tensors == 0) return CPM_OK;
    // the widest type that every page of every tensor begins and ends on
    int64_t bits = 0;
    for (int i = 0; i < n_tensors; ++i) bits |= tensors[5 * i] | tensors[5 * i + 1] | tensors[5 * i + 2];
    const int width = (bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : 1;
    PagedTensors all = {};
    int64_t blocks = 0;
    for (int i = 0; i < n_tensors; ++i) {
        const int64_t* t = tensors + 5 * i;
        if (t[2] <= 0 || t[3] < 0 || t[4] < 0 || t[4] > 0x7fffffff) return CPM_BAD_ARGUMENT;
        const int64_t per = (int64_t)kCopyThreads * kCopyLoads * width, parts = (t[2] + per - 1) / per;
        if (parts > 0x7fffffff) return CPM_BAD_ARGUMENT;
        all.t[i] = PagedTensor{reinterpret_cast<char*>(t[0]), t[1], t[2], blocks, (int)t[4], (int)parts};
        blocks += t[3] * parts * n_moves;
    }
    if (blocks == 0) return CPM_OK;
    all.n = n_tensors;
    return width == 16 ? launch<uint4>(all, blocks, src, dst, n_moves, stream)
         : width == 4 ? launch<uint32_t>(all, blocks, src, dst, n_moves, stream)
                      : launch<uint8_t>(all, blocks, src, dst, n_moves, stream);
}
