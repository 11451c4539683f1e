// Moves inside the paged cache: the accepted path of a speculative step (kv_compact) and whole
// pages (kv_copy_pages).  Both only copy bytes.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace gqa_b200 {

constexpr int kCompactThreads = 128;
constexpr int kCompactItems = 8;        // granules a thread holds between the reads and the writes
constexpr int kCompactMaxRows = 1024;   // kCompactThreads * kCompactItems: one column of granules

struct CompactParams {
    void* k_cache;
    void* v_cache;
    const int32_t* table;
    const int32_t* src;        // [batch, n]
    const int32_t* dst;        // [batch] position of entry 0
    long long row_bytes, num_blocks, cap_tokens;
    int n, block_size, max_pages;
    int slice;                 // granules of a row one CTA moves
};

// Byte offset of a sequence's position in the cache, or -1.
__device__ __forceinline__ long long page_row_offset(const CompactParams& p, int b, long long pos) {
    if (pos < 0 || pos >= p.cap_tokens) return -1;
    const int page = (int)(pos / p.block_size);
    const long long phys = __ldg(p.table + (long long)b * p.max_pages + page);
    if (phys < 0 || phys >= p.num_blocks) return -1;
    return (phys * p.block_size + (pos - (long long)page * p.block_size)) * p.row_bytes;
}

// One CTA moves `slice` granules of every listed row of one sequence, of K or of V: all reads,
// a barrier, all writes.  Slices are columns that no other CTA touches, so whatever the list
// holds (a permutation, the same source twice, a source that is another entry's destination),
// every entry gets the row as it was before the call.
// What bounds it: for a few rows a launch and dependent trips to memory (positions, page ids, rows, writes), 4 to 5 us
// for 8 sequences x 5 rows of 2 KB; for 256 x 16 rows, 6.6 to 8 us (2.2 to 2.7 TB/s), its own index arithmetic as well:
// two 64-bit divisions an entry and a division by the run-time width a granule keep 45 % of the issue slots and
// 23 % of the special-function pipe busy.  A thread holds up to eight granules so that its reads are all under
// way before the barrier.
template <typename UNIT>
__global__ void __launch_bounds__(kCompactThreads) kv_compact_kernel(const CompactParams p) {
    __shared__ long long s_from[kCompactMaxRows], s_to[kCompactMaxRows];
    const int b = blockIdx.x;
    char* cache = static_cast<char*>(blockIdx.z ? p.v_cache : p.k_cache);
    const long long first = __ldg(p.dst + b);
    for (int i = threadIdx.x; i < p.n; i += kCompactThreads) {
        long long from = page_row_offset(p, b, __ldg(p.src + (long long)b * p.n + i));
        const long long to = from < 0 ? -1 : page_row_offset(p, b, first + i);
        if (to < 0) from = -1;
        s_from[i] = from;
        s_to[i] = to;
    }
    __syncthreads();
    const long long units = p.row_bytes / (long long)sizeof(UNIT);
    const long long u0 = (long long)blockIdx.y * p.slice;
    const int width = (int)(units - u0 < p.slice ? units - u0 : p.slice);
    const int total = width * p.n;           // <= kCompactThreads * kCompactItems by the launcher's choice
    UNIT held[kCompactItems];
#pragma unroll
    for (int j = 0; j < kCompactItems; ++j) {
        const int idx = threadIdx.x + j * kCompactThreads;
        if (idx < total) {
            const int i = idx / width;
            if (s_from[i] >= 0) held[j] = reinterpret_cast<const UNIT*>(cache + s_from[i])[u0 + idx - i * width];
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kCompactItems; ++j) {
        const int idx = threadIdx.x + j * kCompactThreads;
        if (idx < total) {
            const int i = idx / width;
            if (s_from[i] >= 0) reinterpret_cast<UNIT*>(cache + s_to[i])[u0 + idx - i * width] = held[j];
        }
    }
}

constexpr int kPageCopyThreads = 256;
constexpr int kPageCopyItems = 4;

struct PageCopyParams {
    void* k_cache;
    void* v_cache;
    const int32_t* src;
    const int32_t* dst;
    long long page_units, num_blocks;   // granules of a page
    long long parts;                    // CTAs per page and cache
};

// Four granules of 16 bytes a thread, all read before the first is written.  Bound by memory: 84 us for
// 4096 pages of 2 x 32 KB, 6.4 TB/s, 0.98 of a plain copy's rate; 2.2 us for 16 pages (one launch).
template <typename UNIT>
__global__ void __launch_bounds__(kPageCopyThreads) kv_copy_pages_kernel(const PageCopyParams p) {
    const long long pair = blockIdx.x / p.parts;
    const long long u0 = (blockIdx.x - pair * p.parts) * (kPageCopyThreads * kPageCopyItems) + threadIdx.x;
    const long long from = __ldg(p.src + pair), to = __ldg(p.dst + pair);
    if (from < 0 || from >= p.num_blocks || to < 0 || to >= p.num_blocks) return;
    UNIT* cache = static_cast<UNIT*>(blockIdx.y ? p.v_cache : p.k_cache);
    const UNIT* s = cache + from * p.page_units;
    UNIT* d = cache + to * p.page_units;
    UNIT held[kPageCopyItems];
#pragma unroll
    for (int j = 0; j < kPageCopyItems; ++j)
        if (u0 + j * kPageCopyThreads < p.page_units) held[j] = s[u0 + j * kPageCopyThreads];
#pragma unroll
    for (int j = 0; j < kPageCopyItems; ++j)
        if (u0 + j * kPageCopyThreads < p.page_units) d[u0 + j * kPageCopyThreads] = held[j];
}

}  // namespace gqa_b200
