// Paged attention of several drafted tokens per sequence (a tree), shared parts: parameters, how
// the work is cut, the partial results and the kernel that joins them.
//
// Sequence b has context_lens[b] keys in its pages; the last n = draft_lens[b] of them are its
// drafted tokens, number j at position prefix + j with prefix = context_len - n.  Query row i
// (drafted token i) sees every key before prefix and drafted token j iff bit j of mask[b, i].
// For one kv head the queries are R = tokens * group rows (row r = token r / group, head r % group)
// that all read the same keys, so K and V are read once per block of rows.
//
// How the work is cut.  The tiles (128 keys, or 64) of all sequences, laid end to end, are cut into
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

constexpr int kTreeTile = 128;          // keys of a tile, the unit of the cut (tensor-core kernel)
constexpr int kTreeSimtTile = 64;       // the same for the CUDA-core kernel: short contexts fill more SMs
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

__device__ __forceinline__ int tree_clamp(int n, int top) { return n < 0 ? 0 : (n > top ? top : n); }
__device__ __forceinline__ int tree_len(const TreeParams& p, int b) { return tree_clamp(__ldg(p.lens + b), p.cap_tokens); }
__device__ __forceinline__ int tree_drafts(const TreeParams& p, int b) {
    if (!p.draft_lens) return p.tokens;
    return tree_clamp(__ldg(p.draft_lens + b), p.tokens);
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
__device__ __forceinline__ int tree_tiles(int len, int tile) { return (int)(((unsigned)len + (unsigned)tile - 1u) / (unsigned)tile); }
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
// sequence, `count` tiles in all; `len` and `drafts` of b.  `empties`: some sequence has no key.
struct TreeRun {
    int b, first, len, drafts;
    long long count;
    bool empties;
};

// Run `r` (all threads of the CTA call it).  s_scan: NT / 32 + 4 words of 8 bytes.
template <int NT, int TILE>
__device__ __forceinline__ TreeRun tree_find_run(const TreeParams& p, int r, long long* s_scan) {
    constexpr int NW = NT / 32;
    constexpr long long kEmpty = 1ll << 62;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int len = 0, drafts = 0;
    bool empties = false;
    // inclusive prefix of the tiles of NT sequences from b0 on; the chunk's total in `sum`
    auto scan = [&](int b0, long long& incl, int& mine, long long& sum) {
        const bool in = b0 + tid < p.batch;
        len = in ? tree_len(p, b0 + tid) : 0;
        drafts = in ? tree_drafts(p, b0 + tid) : 0;
        mine = tree_tiles(len, TILE);
        incl = mine;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, incl, s);
            if (lane >= s) incl += up;
        }
        const bool none = __any_sync(0xffffffffu, in && len == 0);
        __syncthreads();
        if (lane == 31) s_scan[warp] = incl | (none ? kEmpty : 0);
        __syncthreads();
        sum = 0;
        long long before = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const long long x = s_scan[w];
            empties |= (x & kEmpty) != 0;
            if (w < warp) before += x & ~kEmpty;
            sum += x & ~kEmpty;
        }
        incl += before;
    };
    long long incl, sum, total = 0;
    int mine;
    for (int b0 = 0; b0 < p.batch; b0 += NT) {
        scan(b0, incl, mine, sum);
        total += sum;
    }
    long long start, end;
    if (total < (1 << 20) && p.n_ranges <= 4000) {     // (a 32-bit division is a good deal shorter)
        start = (unsigned)total * (unsigned)r / (unsigned)p.n_ranges;
        end = (unsigned)total * (unsigned)(r + 1) / (unsigned)p.n_ranges;
    } else {
        start = total * r / p.n_ranges;
        end = total * (r + 1) / p.n_ranges;
    }
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
            s_scan[NW + 2] = len;
            s_scan[NW + 3] = drafts;
        }
        base += sum;
        if (base > start) break;
    }
    __syncthreads();
    run.b = (int)s_scan[NW];
    run.first = (int)s_scan[NW + 1];
    run.len = (int)s_scan[NW + 2];
    run.drafts = (int)s_scan[NW + 3];
    run.empties = empties;
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
// Lane i of a warp looks after run r0 + i (where it begins; the row's maximum, sum and weight there), so
// that a long sequence's many pieces cost a few round trips to memory and not some each; then the warp
// adds the pieces' rows, kTreeMergeRows rows by four pieces at a time.
// Its reads are the partials, 4 D + 8 bytes a row and piece, mostly still in L2; bound by round trips: 6 to
// 8 us alone with 2 pieces a row (144 runs), 4 of them behind the attention kernel's last CTAs; 25 us with 18
// pieces of 2048 rows.  The pieces of a row are one warp's work, so that a single long sequence with one kv head
// pays most: 148 pieces of 8 rows (32 k keys) take 47 us, of 64 rows 57, as long as their attention (44 and 50).
// NV4 > 0: D is a multiple of 4 and at most 128 NV4, a lane owns columns 4 lane .. 4 lane + 3 (and + 128).
// ---------------------------------------------------------------------------
constexpr int kTreeMergeWarps = 8;
constexpr int kTreeMergeRows = 2;                    // rows of a warp at a time
template <typename T, int NV4>
__global__ void __launch_bounds__(kTreeMergeWarps * 32) gqa_tree_merge_kernel(const TreeParams p) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr unsigned ALL = 0xffffffffu;
    const int r0 = blockIdx.x;                       // last run before the boundary
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int4 mine = __ldcg(p.info + min(r0 + lane, p.n_ranges - 1));
    const int b = __shfl_sync(ALL, mine.x, 1), first = __shfl_sync(ALL, mine.y, 1);
    const int prev_b = __shfl_sync(ALL, mine.x, 0), prev_first = __shfl_sync(ALL, mine.y, 0);
    if (b >= p.batch || first == 0) return;          // no tile behind it, or between two sequences
    if (prev_b == b && prev_first != 0) return;      // an earlier boundary is inside this sequence too
    const int slot0 = 2 * r0 + (prev_b == b ? 0 : 1);   // the first piece; every later one begins its run
    // a run whose first tile is b's holds a piece of it, if it has a tile at all (.z)
    auto inside = [&](int q0, int4 info) {
        const int r = q0 + lane;
        return r < p.n_ranges && (r == r0 || info.x == b);
    };
    const int n_rows = p.rows * p.kv_heads;
    const int D = p.head_dim;
    constexpr bool VEC = NV4 > 0;
    constexpr int NV = VEC ? NV4 : 8;                // groups of columns of a lane
    constexpr int W = VEC ? 4 : 1;                   // columns of a group
    constexpr int RW = VEC ? kTreeMergeRows : 1;
    const int step = gridDim.y * kTreeMergeWarps * RW;
    for (int row0 = (blockIdx.y * kTreeMergeWarps + warp) * RW; row0 < n_rows; row0 += step) {
        float acc[RW][NV][W], sum[RW], mx[RW];
#pragma unroll
        for (int k = 0; k < RW; ++k) {
            sum[k] = 0.f;
            mx[k] = -INFINITY;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int c = 0; c < W; ++c) acc[k][j][c] = 0.f;
        }
        for (int q0 = r0; q0 < p.n_ranges; q0 += 32) {
            const int4 info = q0 == r0 ? mine : __ldcg(p.info + min(q0 + lane, p.n_ranges - 1));
            const bool in = inside(q0, info), has = in && info.z != 0;
            const unsigned last_in = __ballot_sync(ALL, in) >> 31;
            const int slot = q0 + lane == r0 ? slot0 : 2 * (q0 + lane);
            // (rows of one kv head or of two: the row number runs on over the heads)
            const long long at = (long long)slot * n_rows + row0;
            float w[RW];
            unsigned live[RW], any = 0;
#pragma unroll
            for (int k = 0; k < RW; ++k) {
                float2 ml = make_float2(-INFINITY, 0.f);
                if (has && row0 + k < n_rows) ml = __ldcg(p.part_ml + at + k);
                const bool use = ml.y != 0.f;        // it saw something (NaN counts)
                float m = use ? ml.x : -INFINITY;
#pragma unroll
                for (int x = 16; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor_sync(ALL, m, x));
                live[k] = __ballot_sync(ALL, use);
                any |= live[k];
                const float mn = fmaxf(mx[k], m);
                const float alpha = mx[k] == -INFINITY ? 0.f : fast_exp2(mx[k] - mn);
                mx[k] = mn;
                w[k] = use ? fast_exp2(ml.x - mn) : 0.f;
                float s = use ? w[k] * ml.y : 0.f;
#pragma unroll
                for (int x = 16; x >= 1; x >>= 1) s += __shfl_xor_sync(ALL, s, x);
                sum[k] = sum[k] * alpha + s;
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int c = 0; c < W; ++c) acc[k][j][c] *= alpha;
            }
            for (unsigned todo = any; todo;) {
                float x[4][RW][NV][W];
                int from[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    from[u] = todo ? __ffs(todo) - 1 : -1;
                    todo &= todo - 1;
                    const long long src = __shfl_sync(ALL, at, from[u] & 31);
#pragma unroll
                    for (int k = 0; k < RW; ++k) {
                        // (a piece that saw nothing may hold anything)
                        const bool load = from[u] >= 0 && (live[k] >> (from[u] & 31) & 1u);
#pragma unroll
                        for (int j = 0; j < NV; ++j) {
                            const int c = W * (lane + 32 * j);
                            if (!load || c >= D) {
#pragma unroll
                                for (int i = 0; i < W; ++i) x[u][k][j][i] = 0.f;
                                continue;
                            }
                            if constexpr (VEC) {
                                const float4 t = __ldcg(reinterpret_cast<const float4*>(p.part_acc + (src + k) * D + c));
                                x[u][k][j][0] = t.x; x[u][k][j][1] = t.y; x[u][k][j][2] = t.z; x[u][k][j][3] = t.w;
                            } else {
                                x[u][k][j][0] = __ldcg(p.part_acc + (src + k) * D + c);
                            }
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int k = 0; k < RW; ++k) {
                        const float wt = __shfl_sync(ALL, w[k], from[u] & 31);
#pragma unroll
                        for (int j = 0; j < NV; ++j)
#pragma unroll
                            for (int c = 0; c < W; ++c) acc[k][j][c] = fmaf(wt, x[u][k][j][c], acc[k][j][c]);
                    }
            }
            if (!last_in) break;                     // the sequence ends within these runs
        }
#pragma unroll
        for (int k = 0; k < RW; ++k) {
            const int row = row0 + k;
            if (row >= n_rows) continue;
            const int kvh = row / p.rows, rr = row - kvh * p.rows;
            const int tok = rr / p.group, head = kvh * p.group + rr - tok * p.group;
            T* dst = static_cast<T*>(p.out) + (((long long)b * p.tokens + tok) * p.q_heads + head) * D;
            const float inv = sum[k] == 0.f ? 0.f : 1.f / sum[k];
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const int c = W * (lane + 32 * j) + i;
                    if (c < D) dst[c] = from_f32<T>(sum[k] == 0.f ? 0.f : acc[k][j][i] * inv);
                }
        }
    }
}

}  // namespace gqa_b200
