// Paged attention of several drafted tokens per sequence (a tree), shared parts: parameters, how
// the work is cut, the partial results and the kernel that joins them.
//
// Sequence b has context_lens[b] keys in its pages; the last n = draft_lens[b] of them are its
// drafted tokens, number j at position prefix + j with prefix = context_len - n.  Query row i
// (drafted token i) sees every key before prefix and drafted token j iff bit j of mask[b, i].
// For one kv head the queries are R = tokens * group rows (row r = token r / group, head r % group)
// that all read the same keys, so K and V are read once per block of rows.
//
// How the work is cut.  The 128-key tiles of all sequences, laid end to end, are cut into
// `n_ranges` equal runs; a run is worked on by one CTA for every (kv head, block of rows), with the
// kv head fastest in the CTA number so that CTAs side by side read neighbouring bytes of the same
// pages.  Every CTA derives its run from context_lens itself (nothing is read on the host, no plan
// launch).  A sequence that lies inside one run is finished by its CTA; of the others, every run
// leaves fp32 partials (max, sum, weighted values) that the merge kernel joins in run order, so the
// result does not depend on timing.  Two slots per run suffice: an unfinished piece either begins
// where the run begins (slot 2 r) or ends where it ends (slot 2 r + 1).
#pragma once

#include "gqa_common.cuh"

namespace gqa_b200 {

constexpr int kTreeTile = 128;          // keys of a tile, the unit of the cut
constexpr int kTreeMaxTokens = 64;      // drafted tokens per sequence: bits of a mask word

struct TreeParams {
    const void* q;                // [batch, tokens, q_heads, D]
    const void* k;
    const void* v;
    void* out;                    // [batch, tokens, q_heads, D]
    const int32_t* table;         // [batch, max_pages]
    const int32_t* lens;          // [batch]
    const int32_t* draft_lens;    // [batch] or null: all `tokens`
    const unsigned long long* mask;   // [batch, tokens] or null: a chain (token i sees 0 .. i)
    int4* info;                   // [n_ranges + 1]: where run r begins, see TreeRun
    float2* part_ml;              // [2 * n_ranges][q_heads * tokens] (max in log2 units, sum)
    float* part_acc;              // [2 * n_ranges][q_heads * tokens][D]
    int n_ranges;
    int batch, tokens, q_heads, kv_heads, group, head_dim;
    int rows, row_blocks;         // tokens * group, and into how many blocks of rows it is cut
    int block_size, bs_shift, max_pages;
    long long num_blocks;
    int cap_tokens;
    int tile_rows;                // tensor-core kernel: rows of a query tile (whole tokens, at most 128)
    float scale_log2;
};

__device__ __forceinline__ int tree_len(const TreeParams& p, int b) {
    const int len = __ldg(p.lens + b);
    return len < 0 ? 0 : (len > p.cap_tokens ? p.cap_tokens : len);
}
__device__ __forceinline__ int tree_drafts(const TreeParams& p, int b) {
    if (!p.draft_lens) return p.tokens;
    const int n = __ldg(p.draft_lens + b);
    return n < 0 ? 0 : (n > p.tokens ? p.tokens : n);
}
// Drafted tokens (bits 0 .. n - 1) that row token i < n may see; `word` is its mask word.
__device__ __forceinline__ unsigned long long tree_bits_of(const TreeParams& p, unsigned long long word, int i, int n) {
    const unsigned long long all = n >= 64 ? ~0ull : (1ull << n) - 1ull;
    return (p.mask ? word : (i >= 63 ? ~0ull : (2ull << i) - 1ull)) & all;
}
__device__ __forceinline__ unsigned long long tree_bits(const TreeParams& p, int b, int i, int n) {
    if (i >= n) return 0ull;
    return tree_bits_of(p, p.mask ? __ldg(p.mask + (long long)b * p.tokens + i) : 0ull, i, n);
}
__device__ __forceinline__ int tree_tiles(int len) { return (int)(((long long)len + kTreeTile - 1) / kTreeTile); }
// Physical row (page * block_size + slot) of a position, the page id clamped into the pool.
__device__ __forceinline__ long long tree_phys_row(const TreeParams& p, const int32_t* table_row, int t) {
    int page, slot;
    if (p.bs_shift >= 0) { page = t >> p.bs_shift; slot = t & (p.block_size - 1); }
    else { page = t / p.block_size; slot = t - page * p.block_size; }
    long long phys = __ldg(table_row + page);
    phys = phys < 0 ? 0 : (phys >= p.num_blocks ? p.num_blocks - 1 : phys);
    return phys * p.block_size + slot;
}

// Where a run begins: `b` the sequence that holds its first tile, `first` that tile's number in the
// sequence, `count` tiles in all.
struct TreeRun {
    int b, first;
    long long count;
};

// Run `r` (all threads of the CTA call it).  s_scan: NT / 32 + 4 words of 8 bytes.
template <int NT>
__device__ __forceinline__ TreeRun tree_find_run(const TreeParams& p, int r, long long* s_scan) {
    constexpr int NW = NT / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // inclusive prefix of the tiles of NT sequences from b0 on; the chunk's total in `sum`
    auto scan = [&](int b0, long long& incl, long long& mine, long long& sum) {
        mine = b0 + tid < p.batch ? tree_tiles(tree_len(p, b0 + tid)) : 0;
        incl = mine;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, incl, s);
            if (lane >= s) incl += up;
        }
        __syncthreads();
        if (lane == 31) s_scan[warp] = incl;
        __syncthreads();
        sum = 0;
        long long before = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const long long x = s_scan[w];
            if (w < warp) before += x;
            sum += x;
        }
        incl += before;
    };
    long long incl, mine, sum, total = 0;
    for (int b0 = 0; b0 < p.batch; b0 += NT) {
        scan(b0, incl, mine, sum);
        total += sum;
    }
    const long long start = total * r / p.n_ranges;
    const long long end = total * (r + 1) / p.n_ranges;
    TreeRun run;
    run.count = end - start;
    if (tid == 0) { s_scan[NW] = p.batch; s_scan[NW + 1] = 0; }
    long long base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += NT) {
        if (p.batch > NT) scan(b0, incl, mine, sum);   // (one chunk: the values are still there)
        else __syncthreads();
        const long long lo = base + incl - mine;
        if (mine > 0 && start >= lo && start < base + incl) {
            s_scan[NW] = b0 + tid;
            s_scan[NW + 1] = start - lo;
        }
        base += sum;
        if (base > start) break;
    }
    __syncthreads();
    run.b = (int)s_scan[NW];
    run.first = (int)s_scan[NW + 1];
    return run;
}

// The first CTA of a run tells the merge kernel where it begins.
__device__ __forceinline__ void tree_publish(const TreeParams& p, int r, const TreeRun& run) {
    if (threadIdx.x == 0) p.info[r] = make_int4(run.b, run.first, (int)(run.count > 0), 0);
}

// Rows of sequences without a key are zero.  Called by every CTA of a launch.
template <typename T>
__device__ __forceinline__ void tree_zero_empty(const TreeParams& p) {
    const long long n = (long long)p.tokens * p.q_heads * p.head_dim;
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        if (tree_len(p, b) > 0) continue;
        T* dst = static_cast<T*>(p.out) + b * n;
        for (long long i = threadIdx.x; i < n; i += blockDim.x) dst[i] = from_f32<T>(0.f);
    }
}

// Row index of (kv head, row) within a partial slot.
__device__ __forceinline__ long long tree_part_row(const TreeParams& p, int slot, int kvh, int row) {
    return ((long long)slot * p.kv_heads + kvh) * p.rows + row;
}

// ---------------------------------------------------------------------------
// Merge: CTA column x stands for the boundary between runs x and x + 1.  If it is the first
// boundary inside a sequence, the CTA joins that sequence's partials, in run order.
//   M = max m_r,  out = sum 2^(m_r - M) acc_r / sum 2^(m_r - M) l_r
// One warp per row.  Lane i looks after piece i of a round of 32 (its maximum, sum and weight), then
// the warp adds the pieces' rows four at a time, so that a long sequence's many pieces cost a few
// round trips to memory and not two each (17 pieces x 256 rows: 29 us one after the other).
// VEC: D is a multiple of 4, a lane owns columns 4 lane .. 4 lane + 3 (and + 128).
// ---------------------------------------------------------------------------
constexpr int kTreeMergeWarps = 8;
template <typename T, bool VEC>
__global__ void __launch_bounds__(kTreeMergeWarps * 32) gqa_tree_merge_kernel(const TreeParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int r0 = blockIdx.x;                       // last run before the boundary
    const int4 here = __ldcg(p.info + r0 + 1);
    const int4 prev = __ldcg(p.info + r0);
    if (here.x >= p.batch || here.y == 0) return;    // no tile behind it, or between two sequences
    if (prev.x == here.x && prev.y != 0) return;     // an earlier boundary is inside this sequence too
    const int b = here.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slot0 = 2 * r0 + (prev.x == b ? 0 : 1);   // the first piece; every later one begins its run
    int r1 = r0;                                     // last run that holds a piece of b
    for (;;) {
        const int r = r1 + 1 + lane;
        const bool in = r < p.n_ranges && __ldcg(p.info + r).x == b;
        const unsigned inside = __ballot_sync(0xffffffffu, in);
        if (inside == 0xffffffffu) { r1 += 32; continue; }
        r1 += __ffs(~inside) - 1;
        break;
    }
    const int n_rows = p.rows * p.kv_heads;
    const int D = p.head_dim;
    constexpr int NV = VEC ? 2 : 8;                  // groups of columns of a lane
    constexpr int W = VEC ? 4 : 1;                   // columns of a group
    for (int row = blockIdx.y * kTreeMergeWarps + warp; row < n_rows; row += gridDim.y * kTreeMergeWarps) {
        const int kvh = row / p.rows, rr = row - kvh * p.rows;
        float acc[NV][W], sum = 0.f, mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int c = 0; c < W; ++c) acc[j][c] = 0.f;
        for (int q0 = r0; q0 <= r1; q0 += 32) {
            const int r = q0 + lane;
            long long at = 0;
            float2 ml = make_float2(-INFINITY, 0.f);
            if (r <= r1 && __ldcg(p.info + r).z) {   // (a run without a tile has no piece)
                at = tree_part_row(p, r == r0 ? slot0 : 2 * r, kvh, rr);
                ml = __ldcg(p.part_ml + at);
            }
            const bool use = ml.y != 0.f;            // it saw something (NaN counts)
            float m = use ? ml.x : -INFINITY;
#pragma unroll
            for (int x = 16; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
            const unsigned live = __ballot_sync(0xffffffffu, use);
            if (live == 0) continue;
            const float mn = fmaxf(mx, m);
            const float alpha = mx == -INFINITY ? 0.f : fast_exp2(mx - mn);
            mx = mn;
            const float w = use ? fast_exp2(ml.x - mn) : 0.f;
            float s = use ? w * ml.y : 0.f;
#pragma unroll
            for (int x = 16; x >= 1; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            sum = sum * alpha + s;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int c = 0; c < W; ++c) acc[j][c] *= alpha;
            for (unsigned todo = live; todo;) {
                float x[4][NV][W], wt[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int from = todo ? __ffs(todo) - 1 : 0;
                    const bool has = todo != 0;
                    todo &= todo - 1;
                    wt[u] = __shfl_sync(0xffffffffu, w, from);
                    const float* src = p.part_acc + __shfl_sync(0xffffffffu, at, from) * D;
#pragma unroll
                    for (int j = 0; j < NV; ++j) {
                        const int c = W * (lane + 32 * j);
                        if (!has || c >= D) {
#pragma unroll
                            for (int i = 0; i < W; ++i) x[u][j][i] = 0.f;
                            continue;
                        }
                        if constexpr (VEC) {
                            const float4 t = __ldcg(reinterpret_cast<const float4*>(src + c));
                            x[u][j][0] = t.x; x[u][j][1] = t.y; x[u][j][2] = t.z; x[u][j][3] = t.w;
                        } else {
                            x[u][j][0] = __ldcg(src + c);
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int j = 0; j < NV; ++j)
#pragma unroll
                        for (int c = 0; c < W; ++c) acc[j][c] = fmaf(wt[u], x[u][j][c], acc[j][c]);
            }
        }
        const int tok = rr / p.group, head = kvh * p.group + rr - tok * p.group;
        T* dst = static_cast<T*>(p.out) + (((long long)b * p.tokens + tok) * p.q_heads + head) * D;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const int c = W * (lane + 32 * j) + i;
                if (c < D) dst[c] = from_f32<T>(sum == 0.f ? 0.f : acc[j][i] * inv);
            }
    }
}

}  // namespace gqa_b200
