// Tree attention on the 5th-generation tensor cores: fp16 / bf16, rows of a multiple of 16 bytes.
// The kernel is the dense prefill kernel's pipeline (tcgen05.mma with scores, probabilities and
// accumulators in tensor memory) over the pages of a run of tiles (gqa_tree_common.cuh):
//
//   S_X(j,h)[128 x HN]  = Q_X[128 x D] . K(j)[HN keys of half h][D]^T    A, B from shared memory
//   O_X[128 x D]       += P_X(j,h)[128 x HN] . V(j)[HN keys][D]          A from tensor memory, B = V rows as they lie
//
// A CTA holds NQ tiles of up to 128 query rows of one kv head (rows = drafted tokens x heads of the
// group; a tile takes whole tokens, so that one TMA box fetches them) that share every K and V tile of BN keys, worked on in two halves of HN = BN / 2.
//
// What bounds it.  A key of a kv head is 4 D bytes that R rows use for 4 R D flops: up to about
// 256 rows memory is the bound (6.55 TB/s over 148 SMs: 128 keys of D 128 arrive every 2850
// clocks).  Per 128 keys the tensor pipe needs 1024 clocks and the exponentials 1024 clocks for
// each tile of 128 rows, so one tile (NQ 1, R <= 128) hides behind memory and two (NQ 2) just
// about do; with more rows the blocks of 256 run side by side and share the pages through L2.
// The rings (K and V, three tiles each at NQ 1) keep up to 192 KB per SM in flight.
//
// How keys arrive.  By TMA, one box of a page's rows x 64 columns at a time (rows of one kv head,
// 128-byte swizzle, columns behind D as zeros), when pages hold a multiple of 8 rows that divides or
// is divided by the tile.  A warp of cp.async does not get enough bytes in flight for this: one warp
// each for K and V ran at 1.0 TB/s whatever the addresses, 190 clocks per 512 bytes.  Pages of other
// sizes are copied that way all the same, by four warps, a quarter of the rows each (2.3 TB/s).
//
// Warp roles: 4 NQ softmax warps (one thread per query row: TMEM lane = row), the loaders (TMA: one
// warp issues K and V, one issues Q and looks after V; else four warps), NQ warps that issue the MMAs
// of their query tile.  No CTA-wide barrier between the pieces of a run: mbarrier phases run on
// across them, the loaders run ahead into the next piece.
//   q_full / k_full[] / v_full[]     copies have landed        -> MMA warps (v_full: -> the V warp)
//   v_ready[]                        arrivals of the V warp    -> MMA warps
//   q_empty / k_empty[] / v_empty[]  tcgen05.commit of every MMA warp's last use     -> loaders
//   bar_s[X][h]                      tcgen05.commit: S_X(j,h) is in TMEM             -> softmax X
//   bar_p[X][h]                      one arrival per live warp: P_X(j,h) is in TMEM  -> MMA warp X
//   bar_o[X][h]                      tcgen05.commit: P.V of (j,h) is done            -> softmax X
// Warps whose 32 rows lie behind the block's last row take no part (the arrival counts are of the
// live warps); their lanes of S, P and O hold anything and are never read.  Every wait is bounded;
// one that runs out raises the status word and the CTA walks its protocol to the end.
//
// Hidden values.  A drafted token is visible to some rows only, and P = 0 times an infinite V would
// be NaN, as would be what lies in a page behind the sequence's end.  So a warp looks through the V
// rows from the first drafted token on once they are in shared memory: what is not finite becomes zero
// there and is remembered by token (a row that sees such a token adds the value to its sums when it
// stores them), rows behind the end become zero.
//
// Precision: scores and sums in fp32, P rounded to the element type (relative error half a step of
// each probability, as in the other tensor-core kernels), O in fp32.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "gqa_decode_mma.cuh"
#include "gqa_tree_common.cuh"
#include "tcgen05_util.cuh"

namespace gqa_b200 {

constexpr int kTreeBM = 128;            // rows of a query tile
constexpr int kTreeTmemCols = 512;

template <int DP, int NQ, bool TMA> struct TreeTcGeom {
    static constexpr int kBN = DP == 256 ? 64 : 128;             // keys of an inner tile
    static constexpr int kHN = kBN / 2;
    static constexpr int kKB = DP / 64;                          // 128-byte blocks of a row
    static constexpr int kQBytes = kKB * kTreeBM * 128;          // [block][row][128 B]
    static constexpr int kTileBytes = kKB * kBN * 128;
    static constexpr int kStagesK = DP == 64 ? 5 : 3;
    static constexpr int kStagesV = DP == 64 ? 5 : (DP == 256 || NQ == 2) ? 2 : 3;
    static constexpr int kOffK = NQ * kQBytes;
    static constexpr int kOffV = kOffK + kStagesK * kTileBytes;
    static constexpr int kSmemBytes = kOffV + kStagesV * kTileBytes;
    static constexpr int kLoaders = TMA ? 2 : 4;                 // loader warps
    static constexpr int kThreads = (4 * NQ + kLoaders + NQ) * 32;
    static constexpr int kColS = 0;                              // NQ x BN
    static constexpr int kColO = NQ * kBN;                       // NQ x DP
    static_assert(kColO + NQ * DP <= kTreeTmemCols, "TMEM budget");
    static_assert(kSmemBytes > 116 * 1024 && kSmemBytes <= 229376, "one CTA per SM, and it fits");
    static_assert(kTreeTile % kBN == 0, "a tile of the cut is a whole number of inner tiles");
};

// One box of the queries: 64 columns x the heads of kv head `head`'s group x the map's tokens from `token`.
__device__ __forceinline__ void tree_tma_load_q(uint32_t dst, const CUtensorMap* map, int x, int head, int token, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(map), "r"(x), "r"(0), "r"(head), "r"(token), "r"(bar) : "memory");
}
// One box of a page: 64 columns (from column x of a kv head) x the map's rows from physical row y.
__device__ __forceinline__ void tree_tma_load(uint32_t dst, const CUtensorMap* map, int x, int head, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(head), "r"(y), "r"(bar) : "memory");
}
// an arrival with the bytes that TMA copies will bring
__device__ __forceinline__ void mbar_arrive_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// Pieces whose not-finite drafted values are remembered at once.  One loader warp is at most a ring
// of tiles, so five pieces, ahead of another; the softmax warps may still be at three pieces back.
constexpr int kTreeBadRing = 16;

template <typename T, int DP, int NQ, bool TMA>
__global__ void __launch_bounds__((4 * NQ + (TMA ? 2 : 4) + NQ) * 32, 1)
gqa_tree_tc_kernel(const TreeParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, int* status) {
    using G = TreeTcGeom<DP, NQ, TMA>;
    using Ops = MmaOps<T>;
    constexpr int BM = kTreeBM, BN = G::kBN, HN = G::kHN, NSK = G::kStagesK, NSV = G::kStagesV, KB = G::kKB;
    constexpr int NT = G::kThreads;
    constexpr int AB_TYPE = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    constexpr uint32_t EXP_MASK = AB_TYPE ? 0x7f807f80u : 0x7c007c00u;   // exponent bits of a pair of elements
    static_assert(NSK <= 5 && NSV <= NSK, "see kTreeBadRing");

    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ __align__(8) uint64_t s_bar[2 + 2 * NSK + 3 * NSV + 6 * NQ];
    __shared__ long long s_scan[NT / 32 + 4];
    __shared__ unsigned long long s_bad[kTreeBadRing];
    __shared__ uint32_t s_tmem;
    __shared__ int s_dead;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool is_softmax = warp < 4 * NQ, is_load = warp >= 4 * NQ && warp < 4 * NQ + G::kLoaders;
    const int X = is_softmax ? warp >> 2 : 0;
    const int quad = warp & 3;
    const int units = p.kv_heads * p.row_blocks;
    const int run_no = blockIdx.x / units, unit = blockIdx.x - run_no * units;
    const int kvh = unit / p.row_blocks, row0 = (unit - kvh * p.row_blocks) * (NQ * p.tile_rows);
    const int rows_here = min(p.rows - row0, NQ * p.tile_rows);  // >= 1
    const int tiles_live = rows_here > p.tile_rows ? 2 : 1;      // query tiles with a row (NQ 1: one)
    const int warps_a = (min(rows_here, p.tile_rows) + 31) / 32; // live softmax warps of tile A, of B
    const int warps_b = tiles_live > 1 ? (rows_here - p.tile_rows + 31) / 32 : 0;
    const int D = p.head_dim;

    const uint32_t s_base = tc::smem_u32(smem);
    if (s_base & 1023u) {                            // the swizzled tiles need a 1024-byte aligned base
        if (tid == 0) atomicExch(status, 3);
        return;
    }
    const uint32_t sq = s_base, sk = s_base + G::kOffK, sv = s_base + G::kOffV;
    const uint32_t q_full = tc::smem_u32(&s_bar[0]);
    const uint32_t q_empty = tc::smem_u32(&s_bar[1]);
    const uint32_t k_full = tc::smem_u32(&s_bar[2]);
    const uint32_t k_empty = k_full + NSK * 8;
    const uint32_t v_full = k_empty + NSK * 8;
    const uint32_t v_empty = v_full + NSV * 8;
    const uint32_t v_ready = v_empty + NSV * 8;
    const uint32_t bar_s = v_ready + NSV * 8;        // [2 NQ]: query tile x 2 + half
    const uint32_t bar_p = bar_s + NQ * 16;
    const uint32_t bar_o = bar_p + NQ * 16;

    if (warp == 0) { tc::tmem_alloc(tc::smem_u32(&s_tmem), kTreeTmemCols); tc::tmem_relinquish(); }
    if (tid == 0) {
        tc::mbar_init(q_full, TMA ? 1 : 128);
        tc::mbar_init(q_empty, tiles_live);
#pragma unroll
        for (int i = 0; i < NSK; ++i) { tc::mbar_init(k_full + i * 8, TMA ? 1 : 128); tc::mbar_init(k_empty + i * 8, tiles_live); }
#pragma unroll
        for (int i = 0; i < NSV; ++i) {
            tc::mbar_init(v_full + i * 8, 1);
            tc::mbar_init(v_ready + i * 8, TMA ? 32 : 128);
            tc::mbar_init(v_empty + i * 8, tiles_live);
        }
#pragma unroll
        for (int x = 0; x < 2 * NQ; ++x) {
            tc::mbar_init(bar_s + x * 8, 1);
            tc::mbar_init(bar_p + x * 8, x < 2 ? warps_a : (warps_b ? warps_b : 1));
            tc::mbar_init(bar_o + x * 8, 1);
        }
        tc::fence_mbar_init();
#pragma unroll
        for (int i = 0; i < kTreeBadRing; ++i) s_bad[i] = 0ull;
        s_dead = 0;
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = s_tmem;

    pdl_launch_dependents();
    pdl_wait();
    tree_zero_empty<T>(p);
    const TreeRun run = tree_find_run<NT>(p, run_no, s_scan);
    if (unit == 0) tree_publish(p, run_no, run);

    bool alive = true;
    auto wait_bar = [&](uint32_t bar, uint32_t parity) {
        if (tc::mbar_test(bar, parity)) return;
        if (!tc::mbar_wait(bar, parity, s_dead ? 1000ull : 1000000000ull)) {
            s_dead = 1;
            alive = false;
            atomicExch(status, 2);
        }
    };

    // 16-byte chunk of a row that this lane copies, and the rows a pass of the warp covers
    constexpr int CPRW = DP / 8, RPI = 32 / CPRW;
    const int ld_c = lane % CPRW, ld_row0 = lane / CPRW;
    const bool ld_col = ld_c * 8 < D;                            // columns behind D are zeros
    const uint64_t row_bytes = (uint64_t)p.kv_heads * D * 2;
    auto chunk_addr = [&](uint32_t tile, int row, int tile_rows) {
        return tile + (ld_c >> 3) * (tile_rows * 128) + row * 128 + (((ld_c & 7) ^ (row & 7)) << 4);
    };
    constexpr int WR = BN / 4;                                   // rows of a tile each loader warp copies
    const int lw = warp - 4 * NQ;                                // loader warp
    const int page_shift = p.bs_shift;
    auto page_of = [&](int pos) { return page_shift >= 0 ? pos >> page_shift : pos / p.block_size; };
    auto clamp_page = [&](int id) { return id < 0 ? 0ll : ((long long)id >= p.num_blocks ? p.num_blocks - 1 : (long long)id); };
    // TMA: lanes of a warp issue the boxes of a tile, box i = (page i / KB of the tile, block i % KB)
    const int box_rows = p.block_size < BN ? p.block_size : BN;
    const int boxes = BN / (box_rows > 0 ? box_rows : 1) * KB;   // <= 32: pages of 8 rows at least

    int J0 = 0;                                      // running number of the piece's first inner tile
    int piece = 0;
    long long left = run.count;
    int first = run.first;
    // what a piece needs of its sequence is asked for a piece ahead
    const int row = row0 + X * p.tile_rows + quad * 32 + lane;   // softmax threads
    const int tok = row / p.group;
    const bool has_row = quad * 32 + lane < p.tile_rows && row < p.rows;   // (else a dead lane of a live warp)
    int len = 0, nd = 0, len_next = 0, nd_next = 0;
    unsigned long long word = 0ull, word_next = 0ull;
    auto ask_sequence = [&](int b) {
        if (b >= p.batch) return;
        len_next = tree_len(p, b);
        nd_next = tree_drafts(p, b);
        if (is_softmax && p.mask && has_row) word_next = __ldg(p.mask + (long long)b * p.tokens + tok);
    };
    if (left > 0) ask_sequence(run.b);
    for (int b = run.b; left > 0 && b < p.batch; ++b, first = 0) {
        len = len_next;
        nd = nd_next;
        word = word_next;
        ask_sequence(b + 1);
        const int tiles = tree_tiles(len);
        if (tiles == 0) continue;
        const int take = (int)(left < tiles - first ? left : tiles - first);
        left -= take;
        const bool whole = take == tiles;
        const int t0 = first * kTreeTile, t1 = min(len, (first + take) * kTreeTile);
        const int n = (t1 - t0 + BN - 1) / BN;
        const int32_t* table = p.table + (long long)b * p.max_pages;

        if (is_load) {
            // =============================== loaders ===============================
            const int prefix = len - nd;
            // what is not finite among eight elements becomes zero; whether there was any
            auto clean = [&](uint4& x) {
                bool any = false;
                auto word = [&](uint32_t& w) {
                    const uint32_t lo = EXP_MASK & 0xffffu, hi = EXP_MASK & 0xffff0000u;
                    if ((w & lo) == lo) { w &= 0xffff0000u; any = true; }
                    if ((w & hi) == hi) { w &= 0x0000ffffu; any = true; }
                };
                word(x.x); word(x.y); word(x.z); word(x.w);
                return any;
            };
            unsigned long long* const bad = &s_bad[piece % kTreeBadRing];
            if (lw == 1 && lane == 0) s_bad[(piece + 8) % kTreeBadRing] = 0ull;
            if (TMA && lw == 0) {
                // ---- K and V: lane i issues box i of a tile, its page id asked for a tile ahead; pages
                // behind the last used one are left out ----
                const int last_page = page_of(t1 - 1);
                const int my_page = lane / KB, my_col = lane % KB;   // of the tile's pages, blocks of 64 columns
                const uint32_t my_off = my_col * (BN * 128) + my_page * (box_rows * 128);
                auto ask = [&](int t) {
                    const int pg = page_of(t) + my_page;
                    return lane < boxes && pg <= last_page ? __ldg(table + pg) : 0;
                };
                int id = ask(t0);
                for (int j = 0; j < n; ++j) {
                    const int J = J0 + j, t = t0 + j * BN, stage_k = J % NSK, stage_v = J % NSV;
                    const int pg = page_of(t);
                    const bool mine = lane < boxes && pg + my_page <= last_page;
                    // (the offset in the page is 0 unless pages are longer than the tile)
                    const int y = (int)(clamp_page(id) * p.block_size) + (t - pg * p.block_size);
                    const uint32_t bytes = (uint32_t)min(boxes, (last_page - pg + 1) * KB) * (uint32_t)(box_rows * 128);
                    if (J >= NSK) wait_bar(k_empty + stage_k * 8, ((J / NSK) - 1) & 1);
                    if (lane == 0) mbar_arrive_tx(k_full + stage_k * 8, bytes);
                    __syncwarp();
                    if (mine) tree_tma_load(sk + stage_k * G::kTileBytes + my_off, &map_k, my_col * 64, kvh, y, k_full + stage_k * 8);
                    if (J >= NSV) wait_bar(v_empty + stage_v * 8, ((J / NSV) - 1) & 1);
                    if (lane == 0) mbar_arrive_tx(v_full + stage_v * 8, bytes);
                    __syncwarp();
                    if (mine) tree_tma_load(sv + stage_v * G::kTileBytes + my_off, &map_v, my_col * 64, kvh, y, v_full + stage_v * 8);
                    if (j + 1 < n) id = ask(t + BN);
                    __syncwarp();
                }
            } else if (TMA) {
                // ---- Q, then the V tiles as they land ----
                if (piece >= 1) wait_bar(q_empty, (piece - 1) & 1);
                const int box_tok = min(p.tokens, p.tile_rows / p.group);
                if (lane == 0) mbar_arrive_tx(q_full, (uint32_t)(tiles_live * KB * box_tok * p.group * 128));
                __syncwarp();
                if (lane < tiles_live * KB)
                    tree_tma_load_q(sq + lane / KB * G::kQBytes + lane % KB * (BM * 128), &map_q, lane % KB * 64, kvh,
                                    b * p.tokens + (row0 + lane / KB * p.tile_rows) / p.group, q_full);
                __syncwarp();
                for (int j = 0; j < n; ++j) {
                    const int J = J0 + j, t = t0 + j * BN, stage = J % NSV;
                    wait_bar(v_full + stage * 8, (J / NSV) & 1);
                    if (t + BN > prefix) {
                        const uint32_t tile = sv + stage * G::kTileBytes;
#pragma unroll 4
                        for (int r = max(0, prefix - t) + ld_row0; r < BN; r += RPI) {
                            const uint32_t at = chunk_addr(tile, r, BN);
                            uint4 x = make_uint4(0u, 0u, 0u, 0u);
                            bool store = true;
                            if (t + r < t1) {
                                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                             : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
                                store = clean(x);
                                if (store) atomicOr(bad, 1ull << (t + r - prefix));
                            }
                            if (store)
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w)
                                             : "memory");
                        }
                        tc::fence_async_smem();
                    }
                    tc::mbar_arrive(v_ready + stage * 8);
                }
            } else {
                // ---- pages of any size: every warp copies a quarter of the rows ----
                const char* k0 = static_cast<const char*>(p.k) + (size_t)kvh * D * 2 + ld_c * 16;
                const char* v0 = static_cast<const char*>(p.v) + (size_t)kvh * D * 2 + ld_c * 16;
                // The queries of the first piece go first; those of a later one wait for the last scores of
                // the piece before, so up to two tiles of keys (as many as the rings always have room for
                // without this piece's progress) are asked for ahead of them.
                const int q_after = n > 1 ? 1 : 0;
                auto load_q = [&]() {                            // a quarter of the rows; rows behind the last are zeros
                    if (piece >= 1) wait_bar(q_empty, (piece - 1) & 1);
                    const char* qb = static_cast<const char*>(p.q) + ((size_t)b * p.tokens * p.q_heads + kvh * p.group) * D * 2 + ld_c * 16;
                    for (int x = 0; x < tiles_live; ++x) {
                        int r = lw * (BM / 4) + ld_row0;
                        int tk = (row0 + x * p.tile_rows + r) / p.group, g = row0 + x * p.tile_rows + r - tk * p.group;
                        for (int i = 0; i < BM / 4; i += RPI, r += RPI) {
                            const bool valid = r < p.tile_rows && x * p.tile_rows + r < rows_here && ld_col;
                            cp_async16<0>(chunk_addr(sq + x * G::kQBytes, r, BM),
                                          valid ? qb + ((size_t)tk * p.q_heads + g) * D * 2 : static_cast<const char*>(p.q), valid ? 16 : 0, 0);
                            g += RPI;
                            while (g >= p.group) { g -= p.group; ++tk; }
                        }
                    }
                    tc::cp_async_arrive(q_full);
                };
                if (piece == 0) load_q();
                auto ask = [&](int t) {
                    const int pos = t + lw * WR + lane;
                    return pos < t1 && lane < WR ? __ldg(table + page_of(pos)) : 0;
                };
                int id = ask(t0);
                for (int j = 0; j < n; ++j) {
                    const int J = J0 + j, t = t0 + j * BN;
                    const int stage_k = J % NSK, stage_v = J % NSV;
                    const uint32_t tile_k = sk + stage_k * G::kTileBytes, tile_v = sv + stage_v * G::kTileBytes;
                    const int pos = t + lw * WR + lane;
                    const uint32_t mine = (uint32_t)(clamp_page(id) * p.block_size + (pos - page_of(pos) * p.block_size));   // below 2^32: the launcher checks it
                    if (j + 1 < n) id = ask(t + BN);
                    if (J >= NSK) wait_bar(k_empty + stage_k * 8, ((J / NSK) - 1) & 1);
#pragma unroll 8
                    for (int i = 0; i < WR / RPI; ++i) {
                        const int r = i * RPI + ld_row0, row = lw * WR + r;
                        const uint64_t at = __shfl_sync(0xffffffffu, mine, r);
                        const bool valid = t + row < t1 && ld_col;
                        cp_async16<0>(chunk_addr(tile_k, row, BN), valid ? k0 + at * row_bytes : static_cast<const char*>(p.k),
                                      valid ? 16 : 0, 0);
                    }
                    tc::cp_async_arrive(k_full + stage_k * 8);
                    if (J >= NSV) wait_bar(v_empty + stage_v * 8, ((J / NSV) - 1) & 1);
                    if (t + BN <= prefix) {
#pragma unroll 8
                        for (int i = 0; i < WR / RPI; ++i) {
                            const int r = i * RPI + ld_row0, row = lw * WR + r;
                            const uint64_t at = __shfl_sync(0xffffffffu, mine, r);
                            const bool valid = t + row < t1 && ld_col;
                            cp_async16<0>(chunk_addr(tile_v, row, BN), valid ? v0 + at * row_bytes : static_cast<const char*>(p.v),
                                          valid ? 16 : 0, 0);
                        }
                        tc::cp_async_arrive(v_ready + stage_v * 8);
                    } else {
                        // the tile holds drafted tokens: rows pass through registers
#pragma unroll 8
                        for (int i = 0; i < WR / RPI; ++i) {
                            const int r = i * RPI + ld_row0, row = lw * WR + r;
                            const uint64_t at = __shfl_sync(0xffffffffu, mine, r);
                            uint4 x = make_uint4(0u, 0u, 0u, 0u);
                            if (t + row < t1 && ld_col) {
                                x = __ldg(reinterpret_cast<const uint4*>(v0 + at * row_bytes));
                                if (t + row >= prefix && clean(x)) atomicOr(bad, 1ull << (t + row - prefix));
                            }
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(chunk_addr(tile_v, row, BN)),
                                         "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
                        }
                        tc::fence_async_smem();
                        tc::mbar_arrive(v_ready + stage_v * 8);
                    }
                    if (piece > 0 && j == q_after) load_q();
                }
            }
        } else if (!is_softmax) {
            // =============================== MMA warp of query tile x ===============================
            const int x = warp - (4 * NQ + G::kLoaders);
            if (x < tiles_live) {
                const uint32_t elected = tc::elect_one();
                const uint32_t idesc_s = tc::idesc_f16(BM, HN, AB_TYPE);
                const uint32_t idesc_o = tc::idesc_f16(BM, DP, AB_TYPE) | tc::kIdescBMnMajor;
                const uint64_t dq = tc::smem_desc_sw128_kmajor(sq + x * G::kQBytes);
                const uint64_t dk0 = tc::smem_desc_sw128_kmajor(sk);
                const uint64_t dv0 = tc::smem_desc_sw128_mnmajor(sv, BN * 128);
                const uint32_t s_col = tmem + G::kColS + x * BN;
                const uint32_t o_col = tmem + G::kColO + x * DP;
                auto scores_of = [&](int j, int h) {
                    const int J = J0 + j, stage = J % NSK;
                    if (h == 0) {
                        wait_bar(k_full + stage * 8, (J / NSK) & 1);
                        tc::fence_async_smem();
                        tc::tc_fence_after();
                    }
                    const uint64_t dk = dk0 + (uint64_t)((stage * G::kTileBytes + h * HN * 128) >> 4);
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tc::mma_f16_ss_w(elected, s_col + h * HN, dq + (uint64_t)((kb * (BM * 128) + k * 32) >> 4),
                                             dk + (uint64_t)((kb * (BN * 128) + k * 32) >> 4), idesc_s, (kb | k) ? 1u : 0u);
                    }
                    tc::mma_commit_w(elected, bar_s + (x * 2 + h) * 8);
                    if (h == 1) {
                        tc::mma_commit_w(elected, k_empty + stage * 8);
                        if (j == n - 1) tc::mma_commit_w(elected, q_empty);
                    }
                };
                auto pv_of = [&](int j, int h) {
                    const int J = J0 + j, stage = J % NSV;
                    wait_bar(bar_p + (x * 2 + h) * 8, J & 1);
                    if (h == 0) { wait_bar(v_ready + stage * 8, (J / NSV) & 1); tc::fence_async_smem(); }
                    tc::tc_fence_after();
                    const uint64_t dv = dv0 + (uint64_t)((stage * G::kTileBytes + h * (HN / 16) * 2048) >> 4);
#pragma unroll
                    for (int k = 0; k < HN / 16; ++k)
                        tc::mma_f16_ts_w(elected, o_col, s_col + h * HN + k * 8, dv + (uint64_t)((k * 2048) >> 4), idesc_o,
                                         (j | h | k) ? 1u : 0u);
                    tc::mma_commit_w(elected, bar_o + (x * 2 + h) * 8);
                    if (h == 1) tc::mma_commit_w(elected, v_empty + stage * 8);
                };
                wait_bar(q_full, piece & 1);
                scores_of(0, 0);
                scores_of(0, 1);
                for (int j = 0; j < n; ++j) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        // S(j+1, h) takes the columns of P(j, h): P.V(j, h) is queued ahead of it and the
                        // tensor pipe runs this warp's products in order
                        pv_of(j, h);
                        if (j + 1 < n) scores_of(j + 1, h);
                    }
                }
            }
            __syncwarp();
        } else if (quad < (X ? warps_b : warps_a)) {
            // =============================== softmax warps of query tile X ===============================
            const int prefix = len - nd;
            const bool live = has_row && tok < nd;
            const unsigned long long bits = live ? tree_bits_of(p, word, tok, nd) : 0ull;
            const uint32_t lane_sel = (uint32_t)(quad * 32) << 16;
            const uint32_t s_addr = tmem + G::kColS + X * BN + lane_sel;
            const uint32_t o_addr = tmem + G::kColO + X * DP + lane_sel;
            float m_run = -INFINITY, l_run = 0.f;

            for (int j = 0; j < n; ++j) {
                const int J = J0 + j;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    wait_bar(bar_s + (X * 2 + h) * 8, J & 1);
                    tc::tc_fence_after();
                    const int t_base = t0 + j * BN + h * HN;
                    float sc[HN];
#pragma unroll
                    for (int q = 0; q < HN / 32; ++q) {
                        uint32_t r[32];
                        tc::tmem_ld32(s_addr + h * HN + q * 32, r);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 32; ++c) sc[q * 32 + c] = __uint_as_float(r[c]);
                    }
                    const int off = prefix - t_base;             // where the drafted tokens begin in this half
                    if (!live || off < HN) {                     // (t1 <= len: no key is missing before them)
                        unsigned long long w = 0ull;             // bit c: key t_base + c is visible
                        if (live) {
                            if (off >= 64) w = ~0ull;
                            else if (off >= 0) w = (bits << off) | ((1ull << off) - 1ull);
                            else if (off > -64) w = bits >> -off;
                        }
                        const uint32_t w0 = (uint32_t)w, w1 = (uint32_t)(w >> 32);
#pragma unroll
                        for (int c = 0; c < HN; ++c)
                            if (!(((c < 32 ? w0 : w1) >> (c & 31)) & 1u)) sc[c] = -INFINITY;
                    }
                    float mx;
                    {
                        float a0 = sc[0], a1 = sc[1], a2 = sc[2], a3 = sc[3];
#pragma unroll
                        for (int c = 4; c < HN - 4; c += 8) {
                            a0 = tc::max3(a0, sc[c], sc[c + 1]); a1 = tc::max3(a1, sc[c + 2], sc[c + 3]);
                            a2 = tc::max3(a2, sc[c + 4], sc[c + 5]); a3 = tc::max3(a3, sc[c + 6], sc[c + 7]);
                        }
                        a0 = tc::max3(a0, sc[HN - 4], sc[HN - 3]);
                        a1 = tc::max3(a1, sc[HN - 2], sc[HN - 1]);
                        mx = fmaxf(tc::max3(a0, a1, a2), a3) * p.scale_log2;
                    }
                    const bool need = mx > m_run + kRescaleSlack;
                    float alpha = 1.f;
                    if (need) {
                        const float mn = fmaxf(m_run, mx);
                        alpha = m_run == -INFINITY ? 0.f : fast_exp2(m_run - mn);
                        m_run = mn;
                        l_run *= alpha;
                    }
                    const float nref = m_run == -INFINITY ? 0.f : -m_run;
                    uint32_t pw[HN / 2];
                    float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
                    for (int c = 0; c < HN; c += 2) {
                        tc::fma2(sc[c], sc[c + 1], sc[c], sc[c + 1], p.scale_log2, nref);
                        sc[c] = fast_exp2(sc[c]);
                        sc[c + 1] = fast_exp2(sc[c + 1]);
                        tc::add2(ps0, ps1, sc[c], sc[c + 1]);
                        pw[c / 2] = Ops::pack(sc[c], sc[c + 1]);
                    }
                    l_run += ps0 + ps1;
                    // O_X may be rescaled once P.V of the half before is done
                    if ((j > 0 || h > 0) && __any_sync(0xffffffffu, need)) {
                        wait_bar(bar_o + (X * 2 + (h ^ 1)) * 8, (h ? J : J - 1) & 1);
                        tc::tc_fence_after();
#pragma unroll
                        for (int c0 = 0; c0 < DP; c0 += 32) {
                            uint32_t o[32];
                            tc::tmem_ld32(o_addr + c0, o);
                            tc::tmem_ld_wait();
#pragma unroll
                            for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
                            tc::tmem_st32(o_addr + c0, o);
                        }
                    }
                    if constexpr (HN == 64) tc::tmem_st32(s_addr + h * HN, pw);
                    else tc::tmem_st16(s_addr + h * HN, pw);
                    tc::tmem_st_wait();
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(bar_p + (X * 2 + h) * 8);
                }
            }

            // ---- the piece's rows: to `out` when it is the whole sequence, else as a partial ----
            wait_bar(bar_o + (X * 2 + 1) * 8, (J0 + n - 1) & 1);
            tc::tc_fence_after();
            const unsigned long long seen_bad = bits & *reinterpret_cast<volatile unsigned long long*>(&s_bad[piece % kTreeBadRing]);
            const bool write = has_row && alive;
            const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
            const long long at = tree_part_row(p, 2 * run_no + (b == run.b ? 0 : 1), kvh, row);
            if (write && !whole) p.part_ml[at] = make_float2(m_run, l_run);
            T* dst = static_cast<T*>(p.out) + (((long long)b * p.tokens + tok) * p.q_heads + kvh * p.group + row - tok * p.group) * D;
#pragma unroll
            for (int c0 = 0; c0 < DP; c0 += 32) {
                uint32_t o[32];
                __syncwarp();
                tc::tmem_ld32(o_addr + c0, o);
                tc::tmem_ld_wait();
                if (!write || c0 >= D) continue;
                if (l_run == 0.f) {                              // saw nothing: O may hold 0 * infinity
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = 0u;
                }
                for (unsigned long long s = seen_bad; s; s &= s - 1ull) {
                    const int t = prefix + __ffsll((long long)s) - 1;
                    const T* vr = static_cast<const T*>(p.v) + tree_phys_row(p, table, t) * p.kv_heads * D + (long long)kvh * D + c0;
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        if (c0 + c >= D) continue;
                        const float val = to_f32<T>(vr[c]);
                        if ((__float_as_uint(val) & 0x7f800000u) == 0x7f800000u) o[c] = __float_as_uint(__uint_as_float(o[c]) + val);
                    }
                }
                if (whole) {
#pragma unroll
                    for (int c8 = 0; c8 < 4; ++c8) {
                        if (c0 + c8 * 8 >= D) continue;
                        uint4 v;
                        v.x = Ops::pack(__uint_as_float(o[c8 * 8 + 0]) * inv, __uint_as_float(o[c8 * 8 + 1]) * inv);
                        v.y = Ops::pack(__uint_as_float(o[c8 * 8 + 2]) * inv, __uint_as_float(o[c8 * 8 + 3]) * inv);
                        v.z = Ops::pack(__uint_as_float(o[c8 * 8 + 4]) * inv, __uint_as_float(o[c8 * 8 + 5]) * inv);
                        v.w = Ops::pack(__uint_as_float(o[c8 * 8 + 6]) * inv, __uint_as_float(o[c8 * 8 + 7]) * inv);
                        *reinterpret_cast<uint4*>(dst + c0 + c8 * 8) = v;
                    }
                } else {
                    uint4* acc = reinterpret_cast<uint4*>(p.part_acc + at * D + c0);
#pragma unroll
                    for (int c4 = 0; c4 < 8; ++c4)
                        if (c0 + c4 * 4 < D) acc[c4] = make_uint4(o[c4 * 4], o[c4 * 4 + 1], o[c4 * 4 + 2], o[c4 * 4 + 3]);
                }
            }
            __syncwarp();
            tc::tc_fence_before();                   // the loads of O_X are done before this warp's next arrival
        }
        J0 += n;
        ++piece;
    }
    if (is_load) cp_async_wait<0>();
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (warp == 0) tc::tmem_dealloc(tmem, kTreeTmemCols);
}

}  // namespace gqa_b200
