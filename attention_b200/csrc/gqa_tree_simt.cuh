// Tree attention on the CUDA cores: every dtype, every head_dim in [1, 256], any alignment, every
// page size.  It is the only kernel for float32 and for rows that are not 16-byte aligned.
//
// One CTA works on one run of tiles (gqa_tree_common.cuh) for one kv head and a block of RB rows.
// Keys go through shared memory 32 at a time as fp32; a thread owns two rows: first LK of their
// scores (keys lx, lx + LX, ...), then, after the softmax step, NJ groups of four output columns.
// The rows of a thread's two jobs are the same and the LX threads of a row pair sit in one warp, so
// the probabilities cross a warp, never the CTA, and the running maxima and sums stay in registers.
// A warp reads a K element once for two rows (RB = 8) to eight (RB = 32): the shared-memory reads,
// not the arithmetic, are what RB amortises, so few rows take the small block and many the large.
// They bound many rows, and with few the loads, which nothing of the CTA overlaps: fp32, D 128, batch 16 of 1 to
// 4 k keys, 8 tokens 280 us (19 TFLOP/s), 32 tokens 1010 us (21); 4 tokens at batch 64 785 us (1.7 TB/s).  A batch of
// four short sequences takes 28 to 35 us, most of it trips to memory (lengths, page ids, keys) and the merge.
#pragma once

#include <type_traits>

#include "gqa_tree_common.cuh"

namespace gqa_b200 {

constexpr int kTreeSimtThreads = 128;
constexpr int kTreeSimtKeys = 32;
static_assert(kTreeSimtTile <= kTreeSimtThreads && kTreeSimtTile % kTreeSimtKeys == 0, "a thread finds a key of a tile");

template <int RB, int DC> struct TreeSimtGeom {
    static constexpr int kLX = 2 * kTreeSimtThreads / RB;      // threads of a row pair
    static constexpr int kLK = kTreeSimtKeys / kLX;            // scores per row and thread
    static constexpr int kNJ = (DC + 4 * kLX - 1) / (4 * kLX); // groups of four columns per thread
    static constexpr int kStride = DC + 4;                     // fp32 words of a row in shared memory
    static constexpr int kPStride = kTreeSimtKeys + 1;
    static constexpr int kSmemBytes = ((RB + 2 * kTreeSimtKeys) * kStride + RB * kPStride) * 4;
    static_assert(kLX <= 32 && kLK >= 1, "a row pair sits in one warp");
};

// N rows of D elements to shared memory as fp32, columns up to DC and rows whose offset is negative as
// zeros, in pieces of type U.  All of a thread's loads are under way before the first is stored (one after
// the other, 16 round trips per 32 keys made most of the kernel's time).
template <typename T, typename U, int DC, int N>
__device__ __forceinline__ void tree_stage_pieces(float* dst, int stride, const T* base, const long long* s_off, int D) {
    constexpr int V = (int)(sizeof(U) / sizeof(T)), C = DC / V;
    constexpr int PER = (N * C + kTreeSimtThreads - 1) / kTreeSimtThreads;
    U raw[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = threadIdx.x + k * kTreeSimtThreads, r = i / C, c = (i - r * C) * V;
        raw[k] = U{};
        if (i < N * C && c < D && s_off[r] >= 0) raw[k] = __ldg(reinterpret_cast<const U*>(base + s_off[r] + c));
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = threadIdx.x + k * kTreeSimtThreads, r = i / C, c = (i - r * C) * V;
        if (i >= N * C) continue;
        const T* e = reinterpret_cast<const T*>(&raw[k]);
        if constexpr (V >= 4) {
#pragma unroll
            for (int j = 0; j < V; j += 4)
                *reinterpret_cast<float4*>(dst + r * stride + c + j) =
                    make_float4(to_f32<T>(e[j]), to_f32<T>(e[j + 1]), to_f32<T>(e[j + 2]), to_f32<T>(e[j + 3]));
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) dst[r * stride + c + j] = to_f32<T>(e[j]);
        }
    }
}
// `piece` bytes divide every row and its address: 16, 4 (two 16-bit elements: 8 tokens on rows of 100
// elements, batch 16, 305 us against 837 with one at a time), or one element.
template <typename T, int DC, int N>
__device__ __forceinline__ void tree_stage_rows(float* dst, int stride, const T* base, const long long* s_off, int D, int piece) {
    if (piece == 16) {
        tree_stage_pieces<T, uint4, DC, N>(dst, stride, base, s_off, D);
    } else if (sizeof(T) == 2 && piece == 4) {
        tree_stage_pieces<T, typename std::conditional<sizeof(T) == 2, unsigned, T>::type, DC, N>(dst, stride, base, s_off, D);
    } else {
#pragma unroll 8
        for (int i = threadIdx.x; i < N * DC; i += kTreeSimtThreads) {
            const int r = i / DC, c = i - r * DC;
            const long long off = s_off[r];
            dst[r * stride + c] = off >= 0 && c < D ? to_f32<T>(base[off + c]) : 0.f;
        }
    }
}

template <typename T, int RB, int DC>
__global__ void __launch_bounds__(kTreeSimtThreads) gqa_tree_simt_kernel(const TreeParams p, const int piece) {
    using G = TreeSimtGeom<RB, DC>;
    constexpr int KN = kTreeSimtKeys, LX = G::kLX, LK = G::kLK, NJ = G::kNJ, ST = G::kStride, PS = G::kPStride;
    extern __shared__ __align__(16) float s_tree[];
    float* s_q = s_tree;                       // [RB][ST]
    float* s_k = s_q + RB * ST;                // [KN][ST]
    float* s_v = s_k + KN * ST;                // [KN][ST]
    float* s_p = s_v + KN * ST;                // [RB][PS]; a key that a row does not see holds -1
    __shared__ long long s_q_off[RB];
    __shared__ long long s_off[kTreeSimtTile];   // of a whole tile's keys: its page ids are one trip to memory
    __shared__ long long s_scan[kTreeSimtThreads / 32 + 4];

    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x;
    const int lx = tid % LX, r0 = tid / LX * 2;
    const int units = p.kv_heads * p.row_blocks;
    const int run_no = blockIdx.x / units, unit = blockIdx.x - run_no * units;
    const int kvh = unit / p.row_blocks, row0 = (unit - kvh * p.row_blocks) * RB;
    const int D = p.head_dim;
    const T* qp = static_cast<const T*>(p.q);
    const T* kp = static_cast<const T*>(p.k) + (long long)kvh * D;
    const T* vp = static_cast<const T*>(p.v) + (long long)kvh * D;

    const TreeRun run = tree_find_run<kTreeSimtThreads, kTreeSimtTile>(p, run_no, s_scan);
    if (run.empties) tree_zero_empty<T>(p);
    if (unit == 0) tree_publish(p, run_no, run);
    long long left = run.count;
    int first = run.first;
    for (int b = run.b; left > 0 && b < p.batch; ++b, first = 0) {
        const int len = tree_len(p, b);
        const int tiles = tree_tiles(len, kTreeSimtTile);
        if (tiles == 0) continue;
        const int take = (int)(left < tiles - first ? left : tiles - first);
        left -= take;
        const bool whole = take == tiles;
        const int t0 = first * kTreeSimtTile, t1 = min(len, (first + take) * kTreeSimtTile);
        const int n = tree_drafts(p, b), prefix = len - n;
        const int32_t* table = p.table + (long long)b * p.max_pages;

        __syncthreads();                       // the piece before has left shared memory
        auto find_keys = [&](int t) {          // pages of the keys t .. t + kTreeSimtTile - 1
            if (tid < kTreeSimtTile)
                s_off[tid] = t + tid < t1 ? tree_phys_row(p, table, t + tid) * p.kv_heads * D : -1;
        };
        if (tid < RB) {
            const int row = row0 + tid, tok = row / p.group;
            s_q_off[tid] = row < p.rows ? (((long long)b * p.tokens + tok) * p.q_heads + kvh * p.group + row - tok * p.group) * D
                                        : -1;
        }
        find_keys(t0);
        __syncthreads();
        tree_stage_rows<T, DC, RB>(s_q, ST, qp, s_q_off, D, piece);

        unsigned long long bits[2];
        bool live[2];
        float m[2], l[2], acc[2][NJ][4];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int row = row0 + r0 + a, tok = row / p.group;
            live[a] = row < p.rows && tok < n;
            bits[a] = row < p.rows ? tree_bits(p, b, tok, n) : 0ull;
            m[a] = -INFINITY;
            l[a] = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[a][j][c] = 0.f;
        }

        for (int t = t0; t < t1; t += KN) {
            const int in_tile = (t - t0) % kTreeSimtTile;
            if (t > t0) {
                __syncthreads();               // the keys before are done with
                if (in_tile == 0) {
                    find_keys(t);
                    __syncthreads();
                }
            }
            tree_stage_rows<T, DC, KN>(s_k, ST, kp, s_off + in_tile, D, piece);
            tree_stage_rows<T, DC, KN>(s_v, ST, vp, s_off + in_tile, D, piece);
            __syncthreads();
            float s[2][LK];
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int i = 0; i < LK; ++i) s[a][i] = 0.f;
#pragma unroll 4
            for (int d = 0; d < DC; d += 4) {
                const float4 q0 = *reinterpret_cast<const float4*>(s_q + r0 * ST + d);
                const float4 q1 = *reinterpret_cast<const float4*>(s_q + (r0 + 1) * ST + d);
#pragma unroll
                for (int i = 0; i < LK; ++i) {
                    const float4 x = *reinterpret_cast<const float4*>(s_k + (lx + LX * i) * ST + d);
                    s[0][i] = fmaf(q0.x, x.x, fmaf(q0.y, x.y, fmaf(q0.z, x.z, fmaf(q0.w, x.w, s[0][i]))));
                    s[1][i] = fmaf(q1.x, x.x, fmaf(q1.y, x.y, fmaf(q1.z, x.z, fmaf(q1.w, x.w, s[1][i]))));
                }
            }
            const bool straddles = t + KN > prefix || t + KN > t1;   // some keys here are hidden from some rows
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                float mx = -INFINITY;
                bool seen[LK];
#pragma unroll
                for (int i = 0; i < LK; ++i) {
                    const int key = t + lx + LX * i;
                    seen[i] = live[a] && key < t1 && (key < prefix || ((bits[a] >> (key - prefix)) & 1ull));
                    s[a][i] = seen[i] ? s[a][i] * p.scale_log2 : -INFINITY;
                    mx = fmaxf(mx, s[a][i]);
                }
#pragma unroll
                for (int x = LX / 2; x >= 1; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                const float mn = fmaxf(m[a], mx);
                const float ref = mn == -INFINITY ? 0.f : mn;
                const float alpha = fast_exp2(m[a] - ref);
                m[a] = mn;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < LK; ++i) {
                    const float w = seen[i] ? fast_exp2(s[a][i] - ref) : 0.f;
                    sum += w;
                    s_p[(r0 + a) * PS + lx + LX * i] = seen[i] ? w : -1.f;
                }
#pragma unroll
                for (int x = LX / 2; x >= 1; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                l[a] = l[a] * alpha + sum;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[a][j][c] *= alpha;
            }
            __syncwarp();
#pragma unroll 2
            for (int key = 0; key < KN; ++key) {
                const float w0 = s_p[r0 * PS + key], w1 = s_p[(r0 + 1) * PS + key];
                // a hidden value may hold anything: it is left out, not multiplied by zero
                const bool use0 = !straddles || !(w0 < 0.f), use1 = !straddles || !(w1 < 0.f);
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int c = 4 * (lx + LX * j);
                    if (c >= DC) continue;
                    const float4 x = *reinterpret_cast<const float4*>(s_v + key * ST + c);
                    if (use0) {
                        acc[0][j][0] = fmaf(w0, x.x, acc[0][j][0]); acc[0][j][1] = fmaf(w0, x.y, acc[0][j][1]);
                        acc[0][j][2] = fmaf(w0, x.z, acc[0][j][2]); acc[0][j][3] = fmaf(w0, x.w, acc[0][j][3]);
                    }
                    if (use1) {
                        acc[1][j][0] = fmaf(w1, x.x, acc[1][j][0]); acc[1][j][1] = fmaf(w1, x.y, acc[1][j][1]);
                        acc[1][j][2] = fmaf(w1, x.z, acc[1][j][2]); acc[1][j][3] = fmaf(w1, x.w, acc[1][j][3]);
                    }
                }
            }
        }

#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int row = row0 + r0 + a;
            if (row >= p.rows) continue;
            const int tok = row / p.group;
            const long long at = tree_part_row(p, 2 * run_no + (b == run.b ? 0 : 1), kvh, row);
            T* dst = static_cast<T*>(p.out) + (((long long)b * p.tokens + tok) * p.q_heads + kvh * p.group + row - tok * p.group) * D;
            if (!whole && lx == 0) p.part_ml[at] = make_float2(m[a], l[a]);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int col = 4 * (lx + LX * j) + c;
                    if (col >= D) continue;
                    if (whole) dst[col] = from_f32<T>(l[a] == 0.f ? 0.f : acc[a][j][c] / l[a]);
                    else p.part_acc[at * D + col] = acc[a][j][c];
                }
        }
    }
}

}  // namespace gqa_b200
