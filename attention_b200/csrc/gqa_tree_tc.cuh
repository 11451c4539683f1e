// Tree attention on the 5th-generation tensor cores: fp16 / bf16, rows of a multiple of 16 bytes.
// The kernel is the dense prefill kernel's pipeline (tcgen05.mma with scores, probabilities and
// accumulators in tensor memory) over the pages of a run of tiles (gqa_tree_common.cuh):
//
//   S_X(j,h)[128 x HN]  = Q_X[128 x D] . K(j)[HN keys of half h][D]^T    A, B from shared memory
//   O_X[128 x D]       += P_X(j,h)[128 x HN] . V(j)[HN keys][D]          A from tensor memory, B = V rows as they lie
//
// A query tile is up to 128 rows of one kv head (rows = drafted tokens x heads of the group; whole
// tokens, so that one TMA box fetches them).  K and V tiles have BN keys, worked on in two halves of
// HN = BN / 2.  A CTA runs one or two chains  scores -> softmax -> P.V , each with its own score and
// output columns, softmax warps and MMA warp:
//   MODE 0   one chain (D above 128: two outputs do not fit tensor memory)
//   MODE 1   one query tile, two chains that take the K/V tiles in turn; their sums are joined when a
//            piece is done.  A chain alone needs 2500 clocks per 128 keys, most of them one warp's
//            instructions (a few drafted tokens fill one warp of four): 141 us on the batch of 64 x 8
//            tokens against 104 of memory time.
//   MODE 2   two query tiles, a chain each, that share every K and V tile
//
// What bounds it.  A key of a kv head is 4 D bytes that R rows use for 4 R D flops: up to about
// 256 rows memory is the bound (6.55 TB/s over 148 SMs: 128 keys of D 128 arrive every 2850
// clocks).  Per 128 keys the tensor pipe needs 1024 clocks and the exponentials 1024 clocks for
// each tile of 128 rows, so one tile (R <= 128) hides behind memory and two just about do; with more
// rows the blocks of 256 run side by side and share the pages through L2.
// The rings (K and V, three tiles each with one query tile) keep up to 192 KB per SM in flight.
//
// How keys arrive.  By TMA, one box of a page's rows x 64 columns at a time (rows of one kv head,
// 128-byte swizzle, columns behind D as zeros), when pages hold a multiple of 8 rows that divides or
// is divided by the tile: a warp for K, a warp for Q and V (one warp for the boxes of both K and V
// would be the bound with 16-token pages: 100 clocks a box).  A warp of cp.async does not get enough
// bytes in flight: one warp each for K and V ran at 1.0 TB/s whatever the addresses, 190 clocks per
// 512 bytes.  Pages of other sizes are copied that way all the same, by four warps, a quarter of the
// rows each, in a single-chain CTA: 3.9 TB/s, the batch of 64 x 8 tokens with pages of 1 or 24 rows in
// 167 to 177 us, against 118 to 120 by TMA.
//
// Warp roles: four softmax warps per chain (one thread per query row: TMEM lane = row), the loaders,
// a warp per chain that issues its MMAs.  No CTA-wide barrier between the pieces of a run: mbarrier
// phases run on across them, the loaders run ahead into the next piece.
//   q_full / k_full[] / v_full[]     copies have landed                              -> MMA warps
//   (MODE 1: a set of k_full and v_full for each chain.  A wait knows a phase by its parity only, so it
//   must not miss one; with common barriers a chain that waits for tile J could take the end of tile
//   J - 6 for it while the other chain is still three tiles back.)
//   q_empty / k_empty[] / v_empty[]  tcgen05.commit of an MMA warp's last use        -> loaders
// and for chain X, half h of a tile:
//   bar_s[X][h]                      tcgen05.commit: S_X(j,h) is in TMEM             -> softmax X
//   bar_p[X][h]                      one arrival per live warp: P_X(j,h) is in TMEM  -> MMA warp X
//   bar_o[X][h]                      tcgen05.commit: P.V of (j,h) is done            -> softmax X
// Warps whose 32 rows lie behind the block's last row take no part (the arrival counts are of the
// live warps); their lanes of S, P and O hold anything and are never read.  Every wait is bounded;
// one that runs out raises the status word and the CTA walks its protocol to the end.
//
// Hidden values.  A drafted token is visible to some rows only, and P = 0 times an infinite V would
// be NaN, as would be what lies in a page behind the sequence's end.  So before they hand over P of a
// half with drafted tokens, the softmax warps look through its V rows from the first drafted token on:
// what is not finite becomes zero in shared memory and is remembered by token (a row that sees such a
// token adds the value to its sums when it stores them), rows behind the end become zero.
//
// Instruction fetch.  What runs once in a piece is straight-line code that the loop over tiles has pushed
// out of the instruction caches, and a miss behind the K and V tiles in flight costs 1000 clocks or
// more: the end of a piece took 8000 clocks and its way to the next piece's first scores 6000, whatever
// the rows.  So loops over columns stay rolled there, the rare additions of hidden values have a loop
// of their own, and a chain's two halves share one body (MODE 2, bound by that body, has two):
// 129 -> 117 us on the batch of 64 x 8 tokens (120 since the loaders' lanes agree on their waits), 45 -> 37 us on a
// ragged one of 32 x 16 tokens.
//
// Precision: scores and sums in fp32, O in fp32, P rounded to the element type for the products.  In bf16
// that is a relative error of half a step of each probability.  fp16 has that only down to 2^-14, and a key
// that is 2^-25 of the row's reference would be nothing: many such keys below one whose value is small are
// the result.  So the reference of fp16 rows is set tree_lift = 11 below the maximum and follows it more
// closely (kTreeSlack): P = 2^(s - reference) <= 2^15, half a step down to 2^-25 of the largest, below that an
// absolute error of up to 2^-36 of it a key.  P's sums are over the same reference, so it cancels in their
// quotient.  Scores beyond 2^20, which fp32 holds to an eighth of a unit and less, have a smaller lift: the
// maximum, the product behind it and the reference are each off by up to half a step (4 at 2^26).  (Batch of 64 sequences of
// 1 to 4 k keys, 16 tokens: no lift and a slack of 8, 128 us; 11 and 4, 130 to 135; 13 and 2, whose sums move
// much more often, 147.  D 256, 64 tokens, batch 16: 130, 131 and 156.)
#pragma once

#include <cuda.h>

#include <type_traits>

#include "gqa_decode_mma.cuh"
#include "gqa_tree_common.cuh"
#include "tcgen05_util.cuh"

namespace gqa_b200 {

// Status word: 0 ok, 2 (| barrier << 8 | warp << 16) = a bounded wait ran out, 3 = the dynamic shared
// memory base was not 1024-byte aligned.
static __device__ int g_tree_tc_status;

constexpr int kTreeBM = 128;            // rows of a query tile
constexpr int kTreeTmemCols = 512;

// How far (log2 units) a row's reference is set below its maximum `mx`, and how much higher the maximum may then
// rise before it is set again.
template <typename T> __device__ __forceinline__ float tree_lift(float mx) {
    if constexpr (std::is_same<T, __half>::value) return fabsf(mx) < 1048576.f ? 11.f : 7.f;
    else return 0.f;
}
template <typename T> constexpr float kTreeSlack = std::is_same<T, __half>::value ? 4.f : kRescaleSlack;

template <int DP, int MODE> struct TreeTcGeom {
    static constexpr int kChains = MODE == 0 ? 1 : 2;
    static constexpr int kNQ = MODE == 2 ? 2 : 1;                // query tiles
    static constexpr int kBN = DP == 256 ? 64 : 128;             // keys of an inner tile
    static constexpr int kHN = kBN / 2;
    static constexpr int kKB = DP / 64;                          // 128-byte blocks of a row
    static constexpr int kQBytes = kKB * kTreeBM * 128;          // [block][row][128 B]
    static constexpr int kTileBytes = kKB * kBN * 128;
    static constexpr int kStagesK = DP == 64 ? 5 : 3;
    static constexpr int kStagesV = DP == 64 ? 5 : (DP == 256 || kNQ == 2) ? 2 : 3;
    static constexpr int kOffK = kNQ * kQBytes;
    static constexpr int kOffV = kOffK + kStagesK * kTileBytes;
    static constexpr int kSmemBytes = kOffV + kStagesV * kTileBytes;
    static constexpr int kColS = 0;                              // kChains x BN
    static constexpr int kColO = kChains * kBN;                  // kChains x DP
    static_assert(kColO + kChains * DP <= kTreeTmemCols, "TMEM budget");
    static_assert(kSmemBytes > 116 * 1024 && kSmemBytes <= 229376, "one CTA per SM, and it fits");
    static_assert(kTreeTile % kBN == 0, "a tile of the cut is a whole number of inner tiles");
};
template <int MODE, bool TMA> constexpr int kTreeTcWarps = (MODE == 0 ? 5 : 10) + (TMA ? 2 : 4);   // softmax and MMA | loaders

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
__device__ __forceinline__ void tree_prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// Loads that start where they are written: the compiler moves a plain one down to where its value is used,
// and behind the K and V tiles in flight a read of HBM takes up to 7000 clocks.
__device__ __forceinline__ int tree_ask(const int32_t* at) {
    int x;
    asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(x) : "l"(at));
    return x;
}
__device__ __forceinline__ unsigned long long tree_ask(const unsigned long long* at) {
    unsigned long long x;
    asm volatile("ld.global.nc.b64 %0, [%1];" : "=l"(x) : "l"(at));
    return x;
}
// eight floats, a whole sector of memory, at once (a lane has a row, so a store of four fills half a sector
// in each of 32 places: 16 bytes a lane took 4000 clocks a piece of 112 rows); 32-byte aligned
__device__ __forceinline__ void tree_store8(float* at, const float* x) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(at), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]) : "memory");
}
// two lanes of packed fp32: d = a * b + c, d = a * b
__device__ __forceinline__ void tree_fma2(float& d0, float& d1, float a0, float a1, float b, float c0, float c1) {
    asm("{\n\t.reg .b64 ra, rb, rc;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %4};\n\tmov.b64 rc, {%5, %6};\n\t"
        "fma.rn.f32x2 ra, ra, rb, rc;\n\tmov.b64 {%0, %1}, ra;\n\t}"
        : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void tree_mul2(float& d0, float& d1, float a0, float a1, float b) {
    asm("{\n\t.reg .b64 ra, rb;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %4};\n\t"
        "mul.rn.f32x2 ra, ra, rb;\n\tmov.b64 {%0, %1}, ra;\n\t}"
        : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b));
}
// an arrival with the bytes that TMA copies will bring
__device__ __forceinline__ void mbar_arrive_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// Pieces whose not-finite drafted values are remembered at once.  The chains share the rings, so one is
// at most five tiles, and as many pieces, ahead of the other; a piece's word is cleared eight ahead.
constexpr int kTreeBadRing = 16;

template <typename T, int DP, int MODE, bool TMA>
__global__ void __launch_bounds__(kTreeTcWarps<MODE, TMA> * 32, 1)
gqa_tree_tc_kernel(const TreeParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v) {
    using G = TreeTcGeom<DP, MODE>;
    using Ops = MmaOps<T>;
    constexpr int BM = kTreeBM, BN = G::kBN, HN = G::kHN, NSK = G::kStagesK, NSV = G::kStagesV, KB = G::kKB;
    constexpr int NX = G::kChains, NQ = G::kNQ, NL = TMA ? 2 : 4, NT = kTreeTcWarps<MODE, TMA> * 32;
    constexpr int NF = MODE == 1 ? 2 : 1;            // sets of k_full and v_full
    constexpr int AB_TYPE = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    constexpr uint32_t EXP_MASK = AB_TYPE ? 0x7f807f80u : 0x7c007c00u;   // exponent bits of a pair of elements
    static_assert(NSK <= 5 && NSV <= NSK, "see kTreeBadRing");

    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ __align__(8) uint64_t s_bar[2 + (1 + NF) * (NSK + NSV) + 6 * NX];
    __shared__ long long s_scan[NT / 32 + 4];
    __shared__ unsigned long long s_bad[kTreeBadRing];
    __shared__ float2 s_ml[MODE == 1 ? 2 * BM : 1];  // MODE 1: the chains' (max, sum) of every row
    __shared__ uint32_t s_tmem;
    __shared__ int s_dead;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool is_softmax = warp < 4 * NX, is_load = warp >= 4 * NX && warp < 4 * NX + NL;
    const int X = is_softmax ? warp >> 2 : is_load ? 0 : warp - (4 * NX + NL);   // chain (softmax, MMA warps)
    const int quad = warp & 3;
    const int units = p.kv_heads * p.row_blocks;
    const int run_no = blockIdx.x / units, unit = blockIdx.x - run_no * units;
    const int kvh = unit / p.row_blocks, row0 = (unit - kvh * p.row_blocks) * (NQ * p.tile_rows);
    const int rows_here = min(p.rows - row0, NQ * p.tile_rows);  // >= 1
    const int tiles_live = rows_here > p.tile_rows ? 2 : 1;      // query tiles with a row (NQ 1: one)
    const int chains_live = MODE == 2 ? tiles_live : NX;
    const int warps_a = (min(rows_here, p.tile_rows) + 31) / 32; // live softmax warps of chain A, of B
    const int warps_b = MODE == 1 ? warps_a : tiles_live > 1 ? (rows_here - p.tile_rows + 31) / 32 : 0;
    const int D = p.head_dim;
    // Up to 32 rows fill one softmax warp per chain, and both would sit on one scheduler (a warp reaches the
    // tensor-memory lanes of its number mod 4 only).  So the rows lie in the query tile twice, at 0 and at
    // 64, and chain B takes its scores and sums from lanes 64 .. 95.  What the chains exchange at the end of
    // a piece then goes through shared memory: the query tile's rows 32 .. 63 and 96 .. 127, which nobody needs.
    const bool spread = MODE == 1 && TMA && rows_here <= 32;
    const int home = spread ? 2 * X : 0;             // first lane quadrant of this chain's rows

    const uint32_t s_base = tc::smem_u32(smem);
    if (s_base & 1023u) {                            // the swizzled tiles need a 1024-byte aligned base
        if (tid == 0) atomicExch(&g_tree_tc_status, 3);
        return;
    }
    const uint32_t sq = s_base, sk = s_base + G::kOffK, sv = s_base + G::kOffV;
    const uint32_t q_full = tc::smem_u32(&s_bar[0]);
    const uint32_t q_empty = tc::smem_u32(&s_bar[1]);
    const uint32_t k_full = tc::smem_u32(&s_bar[2]);
    const uint32_t k_empty = k_full + NF * NSK * 8;
    const uint32_t v_full = k_empty + NSK * 8;
    const uint32_t v_empty = v_full + NF * NSV * 8;
    const uint32_t bar_s = v_empty + NSV * 8;        // [2 NX]: chain x 2 + half
    const uint32_t bar_p = bar_s + NX * 16;
    const uint32_t bar_o = bar_p + NX * 16;

    if (warp == 0) { tc::tmem_alloc(tc::smem_u32(&s_tmem), kTreeTmemCols); tc::tmem_relinquish(); }
    if (tid == 0) {
        tc::mbar_init(q_full, TMA ? 1 : 128);
        tc::mbar_init(q_empty, chains_live);
#pragma unroll
        for (int i = 0; i < NF * NSK; ++i) tc::mbar_init(k_full + i * 8, TMA ? 1 : 128);
#pragma unroll
        for (int i = 0; i < NF * NSV; ++i) tc::mbar_init(v_full + i * 8, TMA ? 1 : 128);
#pragma unroll
        for (int i = 0; i < NSK; ++i) tc::mbar_init(k_empty + i * 8, MODE == 2 ? tiles_live : 1);
#pragma unroll
        for (int i = 0; i < NSV; ++i) tc::mbar_init(v_empty + i * 8, MODE == 2 ? tiles_live : 1);
#pragma unroll
        for (int x = 0; x < 2 * NX; ++x) {
            tc::mbar_init(bar_s + x * 8, 1);
            tc::mbar_init(bar_p + x * 8, x < 2 ? warps_a : (warps_b ? warps_b : 1));
            tc::mbar_init(bar_o + x * 8, 1);
        }
        tc::fence_mbar_init();
#pragma unroll
        for (int i = 0; i < kTreeBadRing; ++i) s_bad[i] = 0ull;
        s_dead = 0;
    }
    if (TMA && warp == 4 * NX && lane == 0) {        // the loader warp: the maps' first use is not to wait for them
        tree_prefetch_map(&map_q);
        tree_prefetch_map(&map_k);
        tree_prefetch_map(&map_v);
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = s_tmem;

    pdl_wait();
    const TreeRun run = tree_find_run<NT, kTreeTile>(p, run_no, s_scan);
    if (run.empties) tree_zero_empty<T>(p);
    if (unit == 0) tree_publish(p, run_no, run);
    // A wait that runs out ends this warp's work: it starts no copy or product any more (but keeps its
    // barriers with other warps), the others follow at their next wait.  The status word: 2, the
    // barrier's number, the warp.
    bool alive = true;
    auto wait_bar = [&](uint32_t bar, uint32_t parity) {
        if (tc::mbar_test(bar, parity)) return;
        const bool dead = *reinterpret_cast<volatile int*>(&s_dead) != 0;
        if (alive && !tc::mbar_wait(bar, parity, dead ? 1000ull : 1000000000ull)) {
            *reinterpret_cast<volatile int*>(&s_dead) = 1;
            alive = false;
            if (!dead) atomicCAS(&g_tree_tc_status, 0, 2 | (int)((bar - q_full) >> 3) << 8 | warp << 16);
        }
    };

    // The loaders' wait: their lanes work together (shuffles, __syncwarp), so all of them leave off or none.  (The MMA
    // warps' products hang on one lane, and the softmax warps go through their hand-offs either way.)
    auto wait_together = [&](uint32_t bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, tc::mbar_test(bar, parity))) return;
        wait_bar(bar, parity);
        alive = __all_sync(0xffffffffu, alive);
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
    const int lw = warp - 4 * NX;                                // loader warp
    const int page_shift = p.bs_shift;
    auto page_of = [&](int pos) { return page_shift >= 0 ? pos >> page_shift : pos / p.block_size; };
    auto clamp_page = [&](int id) { return id < 0 ? 0ll : ((long long)id >= p.num_blocks ? p.num_blocks - 1 : (long long)id); };
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
    // TMA: lanes of a warp issue the boxes of a tile, box i = (page i / KB of the tile, block i % KB)
    const int box_rows = p.block_size < BN ? p.block_size : BN;
    const int boxes = BN / (box_rows > 0 ? box_rows : 1) * KB;   // <= 32: pages of 8 rows at least

    int J0 = 0;                                      // running number of the piece's first inner tile
    int C0[2] = {0, 0};                              // the chains' running numbers of their tiles
    uint32_t k_par = 0, v_par = 0;                   // bit s: parity of the chain's next use of stage s
    int piece = 0;
    int left = (int)run.count;                       // (fits: the launcher checks it)
    int first = run.first;
    // what a piece needs of its sequence is asked for a piece ahead
    const int wq = quad - home;                                  // softmax warps: number among those of the chain
    const int row_l = wq * 32 + lane, row = row0 + (MODE == 2 ? X * p.tile_rows : 0) + row_l;
    const int tok = row / p.group;
    const bool has_row = row_l >= 0 && row_l < p.tile_rows && row < p.rows;   // (else a dead lane, or warp)
    // (as it was loaded: nothing is computed from it, and so waited for, before its piece begins)
    int len = 0, nd = 0, len_next = run.len, nd_next = run.drafts;
    unsigned long long word = 0ull, word_next = 0ull;
    auto ask_word = [&](int b) {
        if (is_softmax && p.mask && has_row) word_next = tree_ask(p.mask + (long long)b * p.tokens + tok);
    };
    auto ask_sequence = [&](int b) {
        if (b >= p.batch) return;
        len_next = tree_ask(p.lens + b);
        if (p.draft_lens) nd_next = tree_ask(p.draft_lens + b);
        ask_word(b);
    };
    if (left > 0) ask_word(run.b);
    for (int b = run.b; left > 0 && b < p.batch; ++b, first = 0) {
        len = tree_clamp(len_next, p.cap_tokens);
        nd = tree_clamp(nd_next, p.tokens);
        word = word_next;
        ask_sequence(b + 1);
        const int tiles = tree_tiles(len, kTreeTile);
        if (tiles == 0) continue;
        const int take = min(left, tiles - first);
        left -= take;
        const bool whole = take == tiles;
        const int t0 = first * kTreeTile, t1 = min(len, (first + take) * kTreeTile);
        const int n = (t1 - t0 + BN - 1) / BN;
        // the tiles of a chain: all, or every other one
        auto tiles_of = [&](int x) { return MODE == 1 ? (n - x + 1) / 2 : n; };
        auto tile_of = [&](int x, int i) { return MODE == 1 ? 2 * i + x : i; };
        const int32_t* table = p.table + (long long)b * p.max_pages;

        if (is_load) {
            // =============================== loaders ===============================
            if (TMA) {
                // ---- K (warp 0) or V, and Q behind its first tile (warp 1): lane i issues box i of a tile, its page id asked for a tile
                // ahead; pages behind the last used one are left out ----
                const CUtensorMap* const map = lw ? &map_v : &map_k;
                const uint32_t ring = lw ? sv : sk, full = lw ? v_full : k_full, empty = lw ? v_empty : k_empty;
                const int stages = lw ? NSV : NSK;
                const int last_page = page_of(t1 - 1);
                const int my_page = lane / KB, my_col = lane % KB;   // of the tile's pages, blocks of 64 columns
                const uint32_t my_off = my_col * (BN * 128) + my_page * (box_rows * 128);
                auto ask = [&](int t) {
                    const int pg = page_of(t) + my_page;
                    return lane < boxes && pg <= last_page ? tree_ask(table + pg) : 0;
                };
                int id = ask(t0);
                auto load_q = [&]() {
                    const int box_tok = min(p.tokens, p.tile_rows / p.group);
                    const int copies = spread ? 2 : tiles_live;
                    if (lane == 0) mbar_arrive_tx(q_full, (uint32_t)(copies * KB * box_tok * p.group * 128));
                    __syncwarp();
                    if (lane < copies * KB)
                        tree_tma_load_q(sq + lane / KB * (spread ? 64 * 128 : G::kQBytes) + lane % KB * (BM * 128), &map_q,
                                        lane % KB * 64, kvh,
                                        b * p.tokens + (row0 + (spread ? 0 : lane / KB * p.tile_rows)) / p.group, q_full);
                    __syncwarp();
                };
                if (lw == 1 && piece == 0) load_q();
                for (int j = 0; j < n; ++j) {
                    const int J = J0 + j, t = t0 + j * BN, use = J / stages, stage = J - use * stages;
                    const int pg = page_of(t);
                    const bool mine = lane < boxes && pg + my_page <= last_page;
                    // (the offset in the page is 0 unless pages are longer than the tile)
                    const int y = (int)(clamp_page(id) * p.block_size) + (t - pg * p.block_size);
                    const uint32_t bytes = (uint32_t)min(boxes, (last_page - pg + 1) * KB) * (uint32_t)(box_rows * 128);
                    if (use > 0) wait_together(empty + stage * 8, (use - 1) & 1);
                    if (!alive) break;
                    const uint32_t landed = full + ((MODE == 1 ? (j & 1) * stages : 0) + stage) * 8;
                    if (lane == 0) mbar_arrive_tx(landed, bytes);
                    __syncwarp();
                    if (mine) tree_tma_load(ring + stage * G::kTileBytes + my_off, map, my_col * 64, kvh, y, landed);
                    if (j + 1 < n) id = ask(t + BN);
                    __syncwarp();
                    if (lw == 1 && j == 0 && piece > 0) {
                        // (the rings have room for that tile whatever becomes of this piece's queries)
                        wait_together(q_empty, (piece - 1) & 1);
                        if (!alive) break;
                        load_q();
                    }
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
                    if (piece >= 1) wait_together(q_empty, (piece - 1) & 1);
                    if (!alive) return;
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
                    return pos < t1 && lane < WR ? tree_ask(table + page_of(pos)) : 0;
                };
                int id = ask(t0);
                for (int j = 0; j < n; ++j) {
                    const int J = J0 + j, t = t0 + j * BN;
                    const int stage_k = J % NSK, stage_v = J % NSV;
                    const uint32_t tile_k = sk + stage_k * G::kTileBytes, tile_v = sv + stage_v * G::kTileBytes;
                    const int pos = t + lw * WR + lane;
                    const uint32_t mine = (uint32_t)(clamp_page(id) * p.block_size + (pos - page_of(pos) * p.block_size));   // below 2^32: the launcher checks it
                    if (j + 1 < n) id = ask(t + BN);
                    if (J >= NSK) wait_together(k_empty + stage_k * 8, ((J / NSK) - 1) & 1);
                    if (!alive) break;
#pragma unroll 8
                    for (int i = 0; i < WR / RPI; ++i) {
                        const int r = i * RPI + ld_row0, row = lw * WR + r;
                        const uint64_t at = __shfl_sync(0xffffffffu, mine, r);
                        const bool valid = t + row < t1 && ld_col;
                        cp_async16<0>(chunk_addr(tile_k, row, BN), valid ? k0 + at * row_bytes : static_cast<const char*>(p.k),
                                      valid ? 16 : 0, 0);
                    }
                    tc::cp_async_arrive(k_full + stage_k * 8);
                    if (J >= NSV) wait_together(v_empty + stage_v * 8, ((J / NSV) - 1) & 1);
                    if (!alive) break;
#pragma unroll 8
                    for (int i = 0; i < WR / RPI; ++i) {
                        const int r = i * RPI + ld_row0, row = lw * WR + r;
                        const uint64_t at = __shfl_sync(0xffffffffu, mine, r);
                        const bool valid = t + row < t1 && ld_col;
                        cp_async16<0>(chunk_addr(tile_v, row, BN), valid ? v0 + at * row_bytes : static_cast<const char*>(p.v),
                                      valid ? 16 : 0, 0);
                    }
                    tc::cp_async_arrive(v_full + stage_v * 8);
                    if (piece > 0 && j == q_after) load_q();
                }
            }
        } else if (!is_softmax) {
            // =============================== MMA warp of chain X ===============================
            if (X < chains_live) {
                const uint32_t elected = tc::elect_one();
                const int nx = tiles_of(X);
                const int c0 = X ? C0[1] : C0[0];
                const uint32_t idesc_s = tc::idesc_f16(BM, HN, AB_TYPE);
                const uint32_t idesc_o = tc::idesc_f16(BM, DP, AB_TYPE) | tc::kIdescBMnMajor;
                const uint64_t dq = tc::smem_desc_sw128_kmajor(sq + (NQ == 2 ? X * G::kQBytes : 0));
                const uint64_t dk0 = tc::smem_desc_sw128_kmajor(sk);
                const uint64_t dv0 = tc::smem_desc_sw128_mnmajor(sv, BN * 128);
                const uint32_t s_col = tmem + G::kColS + X * BN;
                const uint32_t o_col = tmem + G::kColO + X * DP;
                auto scores_of = [&](int i, int h) {
                    const int J = J0 + tile_of(X, i), stage = J % NSK;
                    if (h == 0) {
                        wait_bar(k_full + (MODE == 1 ? X * NSK + stage : stage) * 8, k_par >> stage & 1);
                        k_par ^= 1u << stage;
                        tc::fence_async_smem();
                        tc::tc_fence_after();
                    }
                    if (!alive) return;
                    const uint64_t dk = dk0 + (uint64_t)((stage * G::kTileBytes + h * HN * 128) >> 4);
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tc::mma_f16_ss_w(elected, s_col + h * HN, dq + (uint64_t)((kb * (BM * 128) + k * 32) >> 4),
                                             dk + (uint64_t)((kb * (BN * 128) + k * 32) >> 4), idesc_s, (kb | k) ? 1u : 0u);
                    }
                    tc::mma_commit_w(elected, bar_s + (X * 2 + h) * 8);
                    if (h == 1) {
                        tc::mma_commit_w(elected, k_empty + stage * 8);
                        if (i == nx - 1) tc::mma_commit_w(elected, q_empty);
                    }
                };
                auto pv_of = [&](int i, int h) {
                    const int J = J0 + tile_of(X, i), stage = J % NSV;
                    wait_bar(bar_p + (X * 2 + h) * 8, (c0 + i) & 1);
                    if (h == 0) {
                        wait_bar(v_full + (MODE == 1 ? X * NSV + stage : stage) * 8, v_par >> stage & 1);
                        v_par ^= 1u << stage;
                        tc::fence_async_smem();
                    }
                    if (!alive) return;
                    tc::tc_fence_after();
                    const uint64_t dv = dv0 + (uint64_t)((stage * G::kTileBytes + h * (HN / 16) * 2048) >> 4);
#pragma unroll
                    for (int k = 0; k < HN / 16; ++k)
                        tc::mma_f16_ts_w(elected, o_col, s_col + h * HN + k * 8, dv + (uint64_t)((k * 2048) >> 4), idesc_o,
                                         (i | h | k) ? 1u : 0u);
                    tc::mma_commit_w(elected, bar_o + (X * 2 + h) * 8);
                    if (h == 1) tc::mma_commit_w(elected, v_empty + stage * 8);
                };
                // (waited for without a tile too: an arrival at q_empty counts for this piece only once its
                // queries are here)
                wait_bar(q_full, piece & 1);
                if (!alive) {
                } else if (nx == 0) {
                    if (elected) tc::mbar_arrive(q_empty);
                } else {
                    scores_of(0, 0);
                    scores_of(0, 1);
                }
                for (int i = 0; i < nx; ++i) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        // S(i+1, h) takes the columns of P(i, h): P.V(i, h) is queued ahead of it and the
                        // tensor pipe runs this warp's products in order
                        pv_of(i, h);
                        if (i + 1 < nx) scores_of(i + 1, h);
                    }
                }
            }
            __syncwarp();
        } else if (wq >= 0 && wq < (X ? warps_b : warps_a)) {
            // =============================== softmax warps of chain X ===============================
            const int prefix = len - nd;
            const bool live = has_row && tok < nd;
            const unsigned long long bits = live ? tree_bits_of(p, word, tok, nd) : 0ull;
            const uint32_t lane_sel = (uint32_t)(quad * 32) << 16;
            const uint32_t s_addr = tmem + G::kColS + X * BN + lane_sel;
            const uint32_t o_addr = tmem + G::kColO + X * DP + lane_sel;
            if (tid == 0) s_bad[(piece + 8) % kTreeBadRing] = 0ull;
            float m_run = -INFINITY, l_run = 0.f;
            const int nx = tiles_of(X), c0 = X ? C0[1] : C0[0];
            for (int i = 0; i < nx; ++i) {
                const int C = c0 + i;                            // running number: parity of the hand-offs
                const int stage = (J0 + tile_of(X, i)) % NSV;
                const uint32_t v_parity = v_par >> stage & 1;
                v_par ^= 1u << stage;
#pragma unroll (MODE == 2 ? 2 : 1)
                for (int h = 0; h < 2; ++h) {
                    wait_bar(bar_s + (X * 2 + h) * 8, C & 1);
                    __syncwarp();                                // the tensor-memory instructions want the whole warp
                    tc::tc_fence_after();
                    const int t_base = t0 + tile_of(X, i) * BN + h * HN;
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
                    // (t1 <= len: no key is missing before them.  A dead lane's scores of other halves may be
                    // anything: it leaves its sums out in the end.)
                    if (off < HN) {
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
                    const float lift = tree_lift<T>(mx);
                    const bool need = live && mx - m_run > lift + kTreeSlack<T>;
                    float alpha = 1.f;
                    if (need) {
                        const float mn = mx - lift;
                        alpha = m_run == -INFINITY ? 0.f : fast_exp2(m_run - mn);
                        m_run = mn;
                        l_run *= alpha;
                    }
                    const float nref = m_run == -INFINITY ? 0.f : -m_run;
#pragma unroll
                    for (int c = 0; c < HN; c += 2) tc::fma2(sc[c], sc[c + 1], sc[c], sc[c + 1], p.scale_log2, nref);
#pragma unroll
                    for (int c = 0; c < HN; ++c) sc[c] = fast_exp2(sc[c]);
                    uint32_t pw[HN / 2];
                    float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
                    for (int c = 0; c < HN; c += 2) {
                        tc::add2(ps0, ps1, sc[c], sc[c + 1]);
                        pw[c / 2] = Ops::pack(sc[c], sc[c + 1]);
                    }
                    l_run += ps0 + ps1;
                    // O_X may be rescaled once P.V of the half before is done
                    if ((i > 0 || h > 0) && __any_sync(0xffffffffu, need)) {
                        wait_bar(bar_o + (X * 2 + (h ^ 1)) * 8, (h ? C : C - 1) & 1);
                        __syncwarp();
                        tc::tc_fence_after();
#pragma unroll 1
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
                    if (off < HN) {                              // drafted tokens, or the end, in this half (warp-uniform)
                        wait_bar(v_full + (MODE == 1 ? X * NSV + stage : stage) * 8, v_parity);
                        const uint32_t tile = sv + stage * G::kTileBytes;
                        const int live_warps = X ? warps_b : warps_a;
                        const int from = max(0, off), end = min(HN, max(t1 - t_base, from)), by = live_warps * RPI;
#pragma unroll 4
                        for (int r = from + wq * RPI + ld_row0; r < end; r += by) {
                            const uint32_t at = chunk_addr(tile, h * HN + r, BN);
                            uint4 x;
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
                            if (clean(x)) {
                                atomicOr(&s_bad[piece % kTreeBadRing], 1ull << (t_base + r - prefix));
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w)
                                             : "memory");
                            }
                        }
#pragma unroll 4
                        for (int r = end + wq * RPI + ld_row0; r < HN; r += by)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(chunk_addr(tile, h * HN + r, BN)), "r"(0u)
                                         : "memory");
                        tc::fence_async_smem();
                        __syncwarp();
                    }
                    tc::tmem_st_wait();
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(bar_p + (X * 2 + h) * 8);
                }
            }

            if (!live) { m_run = -INFINITY; l_run = 0.f; }
            // ---- the piece's rows: to `out` when it is the whole sequence, else as a partial ----
            if (nx > 0) {
                wait_bar(bar_o + (X * 2 + 1) * 8, (c0 + nx - 1) & 1);
                tc::tc_fence_after();
            }
            // MODE 1: the two warps of these rows exchange (max, sum) and store half of the columns each.
            // A chain without a visible key (or a tile) has sum 0; its O may hold anything and is left out.
            float m_all = m_run, l_all = l_run, w_own = 1.f, w_other = 0.f;
            bool use_own = l_run != 0.f, use_other = false;
            constexpr int COLS = MODE == 1 ? DP / 2 : DP;        // columns this warp stores
            // spread: 4 KB for 32 columns of chain x, element (column, lane)
            auto exchange = [&](int x, int cc) {
                const int i = x * (COLS / 32) + cc / 32;
                return sq + (i >> 1) * (BM * 128) + 32 * 128 + (i & 1) * (64 * 128) + lane * 4;
            };
            if constexpr (MODE == 1) {
                s_ml[X * BM + row_l] = make_float2(m_run, l_run);
                __syncwarp();
                if (spread) {                                    // the columns that the other warp stores
#pragma unroll 1
                    for (int cc = 0; cc < COLS; cc += 32) {
                        uint32_t o[32];
                        tc::tmem_ld32(o_addr + (X ^ 1) * COLS + cc, o);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            asm volatile("st.shared.b32 [%0], %1;" ::"r"(exchange(X, cc) + c * 128), "r"(o[c]) : "memory");
                    }
                }
                tc::tc_fence_before();
                asm volatile("bar.sync %0, 64;" ::"r"(wq + 1) : "memory");
                tc::tc_fence_after();
                const float2 other = s_ml[(X ^ 1) * BM + row_l];
                use_other = other.y != 0.f;
                m_all = fmaxf(use_own ? m_run : -INFINITY, use_other ? other.x : -INFINITY);
                w_own = use_own ? fast_exp2(m_run - m_all) : 0.f;
                w_other = use_other ? fast_exp2(other.x - m_all) : 0.f;
                // (the two warps add in the same order: they must agree to the bit)
                const float own = use_own ? w_own * l_run : 0.f, oth = use_other ? w_other * other.y : 0.f;
                l_all = X ? oth + own : own + oth;
            }
            const unsigned long long seen_bad = bits & *reinterpret_cast<volatile unsigned long long*>(&s_bad[piece % kTreeBadRing]);
            const bool write = has_row && alive;
            const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
            if (whole) { w_own *= inv; w_other *= inv; }         // (a partial stays unnormalised)
            const bool plain = __all_sync(0xffffffffu, use_own && use_other);
            const long long at = tree_part_row(p, 2 * run_no + (b == run.b ? 0 : 1), kvh, row);
            if (write && !whole && (MODE != 1 || X == 0)) p.part_ml[at] = make_float2(m_all, l_all);
            T* dst = static_cast<T*>(p.out) + (((long long)b * p.tokens + tok) * p.q_heads + kvh * p.group + row - tok * p.group) * D;
#pragma unroll 1
            for (int cc = 0; cc < COLS; cc += 32) {
                const int c0 = cc + (MODE == 1 ? X * COLS : 0);
                uint32_t raw[32];
                float o[32];
                __syncwarp();
                tc::tmem_ld32(o_addr + c0, raw);
                if constexpr (MODE != 1) {
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 32; c += 2)
                        tree_mul2(o[c], o[c + 1], __uint_as_float(raw[c]), __uint_as_float(raw[c + 1]), w_own);
                    if (!use_own) {
#pragma unroll
                        for (int c = 0; c < 32; ++c) o[c] = 0.f;
                    }
                } else {
                    uint32_t raw2[32];
                    if (spread) {
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(raw2[c]) : "r"(exchange(X ^ 1, cc) + c * 128) : "memory");
                    } else {
                        tc::tmem_ld32(tmem + G::kColO + (X ^ 1) * DP + lane_sel + c0, raw2);
                    }
                    tc::tmem_ld_wait();
                    if (!plain) {                                // some row saw nothing in one of the chains
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            if (!use_own) raw[c] = 0u;
                            if (!use_other) raw2[c] = 0u;
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        tree_mul2(o[c], o[c + 1], __uint_as_float(raw[c]), __uint_as_float(raw[c + 1]), w_own);
                        tree_fma2(o[c], o[c + 1], __uint_as_float(raw2[c]), __uint_as_float(raw2[c + 1]), w_other, o[c], o[c + 1]);
                    }
                }
                if (!write || c0 >= D) continue;
                if (whole) {
#pragma unroll
                    for (int c8 = 0; c8 < 4; ++c8) {
                        if (c0 + c8 * 8 >= D) continue;
                        uint4 v;
                        v.x = Ops::pack(o[c8 * 8 + 0], o[c8 * 8 + 1]);
                        v.y = Ops::pack(o[c8 * 8 + 2], o[c8 * 8 + 3]);
                        v.z = Ops::pack(o[c8 * 8 + 4], o[c8 * 8 + 5]);
                        v.w = Ops::pack(o[c8 * 8 + 6], o[c8 * 8 + 7]);
                        *reinterpret_cast<uint4*>(dst + c0 + c8 * 8) = v;
                    }
                } else {
                    float* acc = p.part_acc + at * D + c0;       // (D is a multiple of 8)
#pragma unroll
                    for (int c8 = 0; c8 < 32; c8 += 8)
                        if (c0 + c8 < D) tree_store8(acc + c8, o + c8);
                }
            }
            // values that are not finite and that this row sees: added to what the thread has just stored
            if (write) {
                for (unsigned long long s = seen_bad; s; s &= s - 1ull) {
                    const int t = prefix + __ffsll((long long)s) - 1;
                    if (t < t0 || t >= t1) continue;             // (a drafted token of another piece)
                    const T* vr = static_cast<const T*>(p.v) + tree_phys_row(p, table, t) * p.kv_heads * D + (long long)kvh * D;
                    const int c1 = min(D, (MODE == 1 ? X * COLS : 0) + COLS);
#pragma unroll 1
                    for (int c = MODE == 1 ? X * COLS : 0; c < c1; ++c) {
                        const float val = to_f32<T>(vr[c]);
                        if ((__float_as_uint(val) & 0x7f800000u) != 0x7f800000u) continue;
                        if (whole) dst[c] = from_f32<T>(to_f32<T>(dst[c]) + val);
                        else p.part_acc[at * D + c] += val;
                    }
                }
            }
            __syncwarp();
            tc::tc_fence_before();                   // the loads of O are done before this warp's next arrival
            if constexpr (MODE == 1) asm volatile("bar.sync %0, 64;" ::"r"(wq + 1) : "memory");   // ... and the other warp's
        }
        C0[0] += tiles_of(0);
        C0[1] += tiles_of(1);
        J0 += n;
        ++piece;
    }
    // (not earlier: the merge kernel's CTAs, and behind them the next call's, would take their places on
    // the SMs in an order of chance; 138 against 127 us on the batch of 64 x 8 tokens, call after call)
    pdl_launch_dependents();
    if (is_load) cp_async_wait<0>();
    tc::tc_fence_before();
    __syncthreads();
    if (*reinterpret_cast<volatile int*>(&s_dead)) {  // copies and products may still be on their way
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        __syncthreads();
    }
    tc::tc_fence_after();
    if (warp == 0) tc::tmem_dealloc(tmem, kTreeTmemCols);
}

}  // namespace gqa_b200
