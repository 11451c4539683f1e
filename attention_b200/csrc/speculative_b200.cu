// Host side of the speculative-step entry points declared in include/gqa_decode_b200.h: norm and
// rotation (into pages), tree attention, compaction of an accepted path, page copies.  Argument
// checks, the cut of the work and the launches.  No allocation, no synchronisation.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <limits>
#include <mutex>

#include "../../include/gqa_decode_b200.h"
#include "gqa_tree_simt.cuh"
#include "gqa_tree_tc.cuh"
#include "kv_pages.cuh"
#include "qk_norm_rope.cuh"

namespace gqa_b200 {
namespace {

constexpr int kSms = 148;                    // the cut of the work is for a B200, whatever runs it
constexpr int kTreeSimtCtasPerSm = 3;
constexpr long long kIntMax = 0x7fffffffll;
constexpr long long kTreeMaxRows = 1 << 20;  // tokens x q_heads of a sequence: row numbers are int32

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int elem_size(int dtype) { return dtype == GQA_B200_F32 ? 4 : 2; }
inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }
inline bool known_dtype(int dtype) {
    return dtype == GQA_B200_F32 || dtype == GQA_B200_F16 || dtype == GQA_B200_BF16;
}

// A range of addresses, [lo, hi).
struct Span {
    uintptr_t lo, hi;
    bool meets(const Span& o) const { return lo < o.hi && o.lo < hi; }
};
inline Span span_of(const void* p, size_t bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    return Span{a, a + bytes};
}
// ... of `heads` rows of `dim` elements for each of batch * tokens tokens, strides in elements
Span span_of_rows(const void* p, int batch, int tokens, int heads, int dim, const int64_t* strides, int size) {
    int64_t lo = 0, hi = dim;
    const int n[3] = {batch, tokens, heads};
    for (int i = 0; i < 3; ++i) (strides[i] < 0 ? lo : hi) += (n[i] - 1) * strides[i];
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    return Span{a + lo * size, a + hi * size};
}

std::mutex g_mutex;                          // guards the per-device caches of this file

bool pdl_on() {
    static const bool on = [] {
        const char* e = std::getenv("GQA_B200_NO_PDL");
        return !(e && e[0] == '1');
    }();
    return on;
}

// Launch with programmatic stream serialization: the kernel may start while its predecessor in the
// stream drains; every kernel launched this way executes griddepcontrol.wait before its first
// global access.  GQA_B200_NO_PDL=1 in the environment turns it off.
template <typename... KArgs, typename... Args>
cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_on() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

// Raises a kernel's dynamic shared-memory limit once per device.
cudaError_t allow_smem(const void* kernel, size_t smem) {
    struct Entry { const void* kernel; int dev; };
    static Entry done[256];
    static int n_done = 0;
    if (smem <= 48 * 1024) return cudaSuccess;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(g_mutex);
    for (int i = 0; i < n_done; ++i)
        if (done[i].kernel == kernel && done[i].dev == dev) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess && n_done < 256) done[n_done++] = Entry{kernel, dev};
    return e;
}

// ---------------------------------------------------------------------------
// tree attention
// ---------------------------------------------------------------------------
// Number of runs the tiles are cut into for `units` CTAs per run on `slots` resident CTAs: as many
// as fill the GPU once, or up to four times if that leaves far fewer CTAs idle in the last round
// (80 units: one round uses 80 of 148 SMs, two use 240 of 296).  A round more has to give an eighth of
// the GPU: memory is busy with four fifths of the SMs at work already, and each round ends in pieces
// of its own.  About 80 000 keys x kv heads of D 128, 1 / 2 / 3 or 4 rounds: 20 kv heads (140, 140,
// 148 SMs of 148 at work) 127 / - / 147 us, 32 (128, 144) 126 / 130 / -, 40 (120, 140) 123 / 127 / -,
// 64 (128, 128, 144) 129 / - / 150.
int tree_run_count(long long units, long long slots, long long cap_tiles) {
    long long best = 1;
    double best_fill = 0.0;
    for (int rounds = 1; rounds <= 4; ++rounds) {
        const long long n = slots * rounds / units;
        if (n < 1) continue;
        const double fill = (double)(n * units) / (double)(slots * rounds);
        if (fill > best_fill + 0.12) { best_fill = fill; best = n; }
    }
    return (int)std::max(1ll, std::min(best, cap_tiles));
}

int tree_simt_rows(int rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : 32; }

struct TreePlan {
    int row_block, row_blocks, n_runs;
    long long units;
};
TreePlan tree_plan(int batch, int tokens, int q_heads, int kv_heads, long long cap_tokens, int row_block, int ctas_per_sm,
                   int tile) {
    TreePlan t;
    const long long rows = (long long)tokens * (q_heads / kv_heads);
    t.row_block = row_block;
    t.row_blocks = (int)((rows + row_block - 1) / row_block);
    t.units = (long long)kv_heads * t.row_blocks;
    const long long cap_tiles = (long long)batch * ((cap_tokens + tile - 1) / tile);
    t.n_runs = tree_run_count(t.units, (long long)kSms * ctas_per_sm, cap_tiles);
    // One sequence of a few tiles: a run that takes them all costs less than the merge (8 kv heads of D 128,
    // 8 drafted tokens, one run / a run a tile: 2 tiles 8.7 / 11.4 us, 4 10.5 / 12.1, 6 12.3 / 12.9, 8 14.2 / 13.6).
    // The host knows the table's width only: 400 keys take 11.3 us in a table of 25 pages, 13.3 in one of 256.
    if (batch == 1 && tile == kTreeTile && cap_tiles <= 6) t.n_runs = 1;
    return t;
}
TreePlan tree_plan_simt(int batch, int tokens, int q_heads, int kv_heads, long long cap_tokens) {
    return tree_plan(batch, tokens, q_heads, kv_heads, cap_tokens, tree_simt_rows(tokens * (q_heads / kv_heads)),
                     kTreeSimtCtasPerSm, kTreeSimtTile);
}

// Element types, sizes and alignments the tensor-core kernel takes: 16-bit, rows of whole 16-byte
// chunks, physical row numbers below 2^32.
bool tree_tc_shape(int dtype, int head_dim, int64_t num_blocks, int block_size) {
    return dtype != GQA_B200_F32 && head_dim % 8 == 0 && num_blocks * block_size < (1ll << 32);
}
int tree_tc_keys(int head_dim) { return head_dim <= 128 ? 128 : 64; }      // of an inner tile
// Pages by TMA: a box of whole 8-row groups, a tile of whole boxes or a page of whole tiles, row numbers
// that are int32 coordinates, and query tiles of whole tokens.
bool tree_tma_shape(int group, int head_dim, int64_t num_blocks, int block_size, long long query_tokens) {
    const int bn = tree_tc_keys(head_dim);
    return block_size % 8 == 0 && (bn % block_size == 0 || block_size % bn == 0) && num_blocks * block_size <= kIntMax &&
           group <= kTreeBM && query_tokens <= kIntMax;
}
// Rows of a query tile: as many whole tokens as 128 rows hold (a group of more than 128 heads is cut).
int tree_tile_rows(int group) { return group <= kTreeBM ? kTreeBM / group * group : kTreeBM; }
// Two query tiles per CTA share every K and V tile when one does not hold all rows (if the keys come by
// TMA, and two accumulators fit tensor memory).
TreePlan tree_plan_tc(int batch, int tokens, int q_heads, int kv_heads, int head_dim, long long cap_tokens, bool tma) {
    const int group = q_heads / kv_heads, tile = tree_tile_rows(group);
    const int tiles = tma && head_dim <= 128 && tokens * group > tile ? 2 : 1;
    return tree_plan(batch, tokens, q_heads, kv_heads, cap_tokens, tile * tiles, 1, kTreeTile);
}

struct TreeScratch {
    size_t info, ml, acc, total;
};
TreeScratch tree_scratch(const TreePlan& t, int tokens, int q_heads, int head_dim) {
    TreeScratch s;
    const size_t rows = t.n_runs > 1 ? 2 * (size_t)t.n_runs * tokens * q_heads : 0;
    s.info = 0;
    s.ml = align_up((size_t)(t.n_runs + 1) * sizeof(int4), 256);
    s.acc = s.ml + align_up(rows * sizeof(float2), 256);
    s.total = s.acc + align_up(rows * head_dim * sizeof(float), 256);
    return s;
}

inline long long cap_tokens_of(int max_pages, int block_size) {
    return std::min((long long)max_pages * block_size, kIntMax - kTreeTile);
}

template <typename T, int RB, int DC>
cudaError_t launch_tree_simt(const TreeParams& p, const TreePlan& t, int piece, cudaStream_t stream) {
    constexpr size_t smem = TreeSimtGeom<RB, DC>::kSmemBytes;
    auto kernel = gqa_tree_simt_kernel<T, RB, DC>;
    const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kernel), smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3((unsigned)(t.n_runs * t.units)), kTreeSimtThreads, smem, stream, p, piece);
}
template <typename T, int RB>
cudaError_t launch_tree_simt_dim(const TreeParams& p, const TreePlan& t, int piece, cudaStream_t stream) {
    if (p.head_dim <= 64) return launch_tree_simt<T, RB, 64>(p, t, piece, stream);
    if (p.head_dim <= 128) return launch_tree_simt<T, RB, 128>(p, t, piece, stream);
    return launch_tree_simt<T, RB, 256>(p, t, piece, stream);
}
// cuTensorMapEncodeTiled, looked up through the runtime so that the library needs no link to the driver.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}

// A cache as [physical row][kv head][D]; a box is 64 columns of one head x `rows` rows, swizzled as
// the shared-memory operands are, zeros behind column D.
bool cache_map(CUtensorMap* map, const void* cache, bool bf16, const TreeParams& p, int rows) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)p.head_dim, (cuuint64_t)p.kv_heads, (cuuint64_t)p.num_blocks * p.block_size};
    const cuuint64_t strides[2] = {(cuuint64_t)p.head_dim * 2, (cuuint64_t)p.kv_heads * p.head_dim * 2};
    const cuuint32_t box[3] = {64, 1, (cuuint32_t)rows}, ones[3] = {1, 1, 1};
    return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(cache),
                  dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Queries as [batch * token][kv head][head of the group][D]; a box is 64 columns of a kv head's group x
// `box_tokens` tokens.  (Tokens behind a sequence's last belong to rows that nobody reads.)
bool query_map(CUtensorMap* map, bool bf16, const TreeParams& p, int box_tokens) {
    const EncodeTiled encode = encode_tiled();
    if (!encode) return false;
    const cuuint64_t row = (cuuint64_t)p.head_dim * 2;
    const cuuint64_t dims[4] = {(cuuint64_t)p.head_dim, (cuuint64_t)p.group, (cuuint64_t)p.kv_heads, (cuuint64_t)p.batch * p.tokens};
    const cuuint64_t strides[3] = {row, row * p.group, row * p.q_heads};
    const cuuint32_t box[4] = {64, (cuuint32_t)p.group, 1, (cuuint32_t)box_tokens}, ones[4] = {1, 1, 1, 1};
    return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(p.q), dims,
                  strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct TreeMaps {
    CUtensorMap q, k, v;
};
bool tree_maps(TreeMaps* m, bool bf16, const TreeParams& p) {
    const int rows = std::min(p.block_size, tree_tc_keys(p.head_dim));
    return cache_map(&m->k, p.k, bf16, p, rows) && cache_map(&m->v, p.v, bf16, p, rows) &&
           query_map(&m->q, bf16, p, std::min(p.tokens, p.tile_rows / p.group));
}

template <typename T, int DP, int MODE, bool TMA>
cudaError_t launch_tree_tc(const TreeParams& p, const TreePlan& t, const TreeMaps& maps, cudaStream_t stream) {
    using G = TreeTcGeom<DP, MODE>;
    static_assert(G::kBN == (DP <= 128 ? 128 : 64), "tree_tc_keys");
    auto kernel = gqa_tree_tc_kernel<T, DP, MODE, TMA>;
    const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kernel), G::kSmemBytes);
    if (e != cudaSuccess) return e;
    return launch_pdl(kernel, dim3((unsigned)(t.n_runs * t.units)), kTreeTcWarps<MODE, TMA> * 32, G::kSmemBytes, stream, p,
                      maps.q, maps.k, maps.v);
}
template <typename T>
cudaError_t launch_tree_tc_dim(const TreeParams& p, const TreePlan& t, const TreeMaps* maps, cudaStream_t stream) {
    const int d = p.head_dim;
    if (!maps) {
        const TreeMaps none{};
        if (d <= 64) return launch_tree_tc<T, 64, 0, false>(p, t, none, stream);
        if (d <= 128) return launch_tree_tc<T, 128, 0, false>(p, t, none, stream);
        return launch_tree_tc<T, 256, 0, false>(p, t, none, stream);
    }
    const bool two = t.row_block > p.tile_rows;
    if (d <= 64) return two ? launch_tree_tc<T, 64, 2, true>(p, t, *maps, stream) : launch_tree_tc<T, 64, 1, true>(p, t, *maps, stream);
    if (d <= 128) return two ? launch_tree_tc<T, 128, 2, true>(p, t, *maps, stream) : launch_tree_tc<T, 128, 1, true>(p, t, *maps, stream);
    return launch_tree_tc<T, 256, 0, true>(p, t, *maps, stream);
}
template <typename T>
cudaError_t launch_tree(const TreeParams& p, const TreePlan& t, bool tc, const TreeMaps* maps, int piece, cudaStream_t stream) {
    cudaError_t e = cudaErrorInvalidValue;
    if (tc) {
        if constexpr (sizeof(T) == 2) e = launch_tree_tc_dim<T>(p, t, maps, stream);
    } else {
        switch (t.row_block) {
            case 8:  e = launch_tree_simt_dim<T, 8>(p, t, piece, stream); break;
            case 16: e = launch_tree_simt_dim<T, 16>(p, t, piece, stream); break;
            default: e = launch_tree_simt_dim<T, 32>(p, t, piece, stream); break;
        }
    }
    if (e != cudaSuccess || t.n_runs == 1) return e;
    const int rows = p.rows * p.kv_heads;
    const int per_cta = kTreeMergeWarps * kTreeMergeRows;
    const int by = std::min((rows + per_cta - 1) / per_cta, 65535);
    auto merge = p.head_dim % 4 != 0 ? gqa_tree_merge_kernel<T, 0>
                 : p.head_dim <= 128 ? gqa_tree_merge_kernel<T, 1>
                                     : gqa_tree_merge_kernel<T, 2>;
    return launch_pdl(merge, dim3((unsigned)(t.n_runs - 1), (unsigned)by), kTreeMergeWarps * 32, 0, stream, p);
}

// ---------------------------------------------------------------------------
// norm and rotation (these return a status of the C interface)
// ---------------------------------------------------------------------------
template <typename T, int L, int HB>
int launch_rope_vec(const RopeParams& p, cudaStream_t stream) {
    RopeBlocks blocks;
    blocks.q = (unsigned)((p.q_heads + HB - 1) / HB);
    blocks.k = (unsigned)((p.kv_heads + HB - 1) / HB);
    blocks.all = blocks.q + blocks.k * (p.append ? 2 : 1);
    const long long units = p.n_tokens * blocks.all, groups = kRopeThreads / L;
    if (units > kIntMax) return GQA_B200_ERR_INT32_RANGE;
    auto kernel = p.interleaved ? qk_norm_rope_vec_kernel<T, L, HB, true> : qk_norm_rope_vec_kernel<T, L, HB, false>;
    kernel<<<(unsigned)((units + groups - 1) / groups), kRopeThreads, 0, stream>>>(p, blocks, (unsigned)units);
    return (int)cudaGetLastError();
}
template <typename T, int L>
int launch_rope_heads(const RopeParams& p, int heads, cudaStream_t stream) {
    // Several heads per group once that still gives every SM its fill of threads: the 32 bytes of angles
    // that a lane reads from the first-level cache then serve as many 16-byte pieces of rows.
    // (Dense 16384 tokens x 72 heads of 128 bf16: 854 us with a warp per row, 154 with two heads per group,
    // 116 with four, 151 with eight, whose registers leave fewer warps.)
    constexpr int HB = 4;
    return p.n_tokens * heads * L >= (long long)HB * kSms * 1024 ? launch_rope_vec<T, L, HB>(p, stream)
                                                                 : launch_rope_vec<T, L, 1>(p, stream);
}

// The vector kernel takes rows of whole eight-element chunks, 16-byte aligned throughout, with the
// rotation's halves (or pairs) in whole chunks.
bool rope_vec_ok(const RopeParams& p, int size) {
    const long long strides[9] = {p.q_sb, p.q_st, p.q_sh, p.k_sb, p.k_st, p.k_sh, p.v_sb, p.v_st, p.v_sh};
    for (int i = 0; i < (p.append ? 9 : 6); ++i)
        if (strides[i] * size % 16 != 0) return false;
    const void* ptrs[10] = {p.q, p.k, p.v, p.q_weight, p.k_weight, p.cos_sin, p.q_out, p.k_out, p.k_cache, p.v_cache};
    for (const void* x : ptrs)
        if (!aligned16(x)) return false;
    return p.head_dim % 8 == 0 && p.rot_dim % 8 == 0;
}

template <typename T>
int launch_rope(const RopeParams& p, cudaStream_t stream) {
    const int heads = p.q_heads + p.kv_heads * (p.append ? 2 : 1);
    if (rope_vec_ok(p, (int)sizeof(T))) {
        if (p.head_dim <= 64) return launch_rope_heads<T, 8>(p, heads, stream);
        if (p.head_dim <= 128) return launch_rope_heads<T, 16>(p, heads, stream);
        return launch_rope_heads<T, 32>(p, heads, stream);
    }
    const long long rows = p.n_tokens * heads;
    const long long grid = (rows + kRopeWarps - 1) / kRopeWarps;
    if (grid > kIntMax) return GQA_B200_ERR_INT32_RANGE;
    qk_norm_rope_any_kernel<T><<<(unsigned)grid, kRopeWarps * 32, 0, stream>>>(p);
    return (int)cudaGetLastError();
}

}  // namespace
}  // namespace gqa_b200

using namespace gqa_b200;

extern "C" {

int gqa_b200_qk_norm_rope(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight,
                          const float* cos_sin, const int32_t* positions, void* q_out, void* k_out, void* k_cache,
                          void* v_cache, const int32_t* block_table, const int32_t* slots, int dtype, int weight_dtype,
                          int batch, int tokens, int q_heads, int kv_heads, int head_dim, int rot_dim,
                          int64_t max_position, const int64_t* strides, float eps, int interleaved, int64_t num_blocks,
                          int block_size, int max_pages, void* stream) {
    if (!known_dtype(dtype) || (weight_dtype != dtype && weight_dtype != GQA_B200_F32)) return GQA_B200_ERR_DTYPE;
    if (batch < 0 || tokens < 0) return GQA_B200_ERR_BATCH;
    if (q_heads <= 0 || kv_heads <= 0) return GQA_B200_ERR_HEADS;
    if (head_dim <= 0 || head_dim > 256) return GQA_B200_ERR_HEAD_DIM;
    if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 2 != 0 || max_position < 0 || max_position > kIntMax)
        return GQA_B200_ERR_ROTATION;
    if (!(std::isfinite(eps) && eps >= 0.f)) return GQA_B200_ERR_SCALE;
    if (!strides || (!q_weight) != (!k_weight)) return GQA_B200_ERR_NULL_POINTER;
    if (batch == 0 || tokens == 0) return GQA_B200_OK;
    const bool append = k_cache != nullptr;
    if (!q || !k || !q_out || !positions || (rot_dim > 0 && max_position > 0 && !cos_sin)) return GQA_B200_ERR_NULL_POINTER;
    if (append) {
        if (num_blocks <= 0 || block_size <= 0) return GQA_B200_ERR_CACHE_SHAPE;
        if (max_pages <= 0) return GQA_B200_ERR_MAX_PAGES;
        if (num_blocks > kIntMax) return GQA_B200_ERR_INT32_RANGE;
        if (!v || !v_cache || !block_table || !slots) return GQA_B200_ERR_NULL_POINTER;
        // a row that is still to be read must not be another token's place in the cache
        const size_t size = elem_size(dtype), cache = (size_t)num_blocks * block_size * kv_heads * head_dim * size;
        const Span caches[2] = {span_of(k_cache, cache), span_of(v_cache, cache)};
        for (const Span& c : caches)
            if (c.meets(span_of_rows(q, batch, tokens, q_heads, head_dim, strides, (int)size)) ||
                c.meets(span_of_rows(k, batch, tokens, kv_heads, head_dim, strides + 3, (int)size)) ||
                c.meets(span_of_rows(v, batch, tokens, kv_heads, head_dim, strides + 6, (int)size)))
                return GQA_B200_ERR_OVERLAP;
    } else if (!k_out) {
        return GQA_B200_ERR_NULL_POINTER;
    }
    RopeParams p{};
    p.q = q; p.k = k; p.v = v; p.q_weight = q_weight; p.k_weight = k_weight; p.cos_sin = cos_sin;
    p.positions = positions; p.slots = slots; p.table = block_table;
    p.q_out = q_out; p.k_out = k_out; p.k_cache = k_cache; p.v_cache = v_cache;
    p.q_sb = strides[0]; p.q_st = strides[1]; p.q_sh = strides[2];
    p.k_sb = strides[3]; p.k_st = strides[4]; p.k_sh = strides[5];
    p.v_sb = strides[6]; p.v_st = strides[7]; p.v_sh = strides[8];
    p.num_blocks = num_blocks;
    p.cap_tokens = append ? std::min((long long)max_pages * block_size, kIntMax) : 0;
    p.n_tokens = (long long)batch * tokens;
    p.tokens = tokens; p.q_heads = q_heads; p.kv_heads = kv_heads; p.head_dim = head_dim; p.rot_dim = rot_dim;
    p.max_position = (int)max_position; p.block_size = block_size; p.max_pages = max_pages;
    p.append = append ? 1 : 0; p.interleaved = interleaved ? 1 : 0; p.weight_f32 = weight_dtype == GQA_B200_F32;
    p.eps = eps;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case GQA_B200_F32: return launch_rope<float>(p, s);
        case GQA_B200_F16: return launch_rope<__half>(p, s);
        default:           return launch_rope<__nv_bfloat16>(p, s);
    }
}

size_t gqa_b200_tree_workspace_bytes(int batch, int tokens, int q_heads, int kv_heads, int head_dim, int block_size,
                                     int max_pages) {
    if (batch <= 0 || tokens <= 0 || tokens > kTreeMaxTokens || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads ||
        head_dim <= 0 || head_dim > 256 || block_size <= 0 || max_pages <= 0 || (long long)tokens * q_heads > kTreeMaxRows)
        return 0;
    const long long cap = cap_tokens_of(max_pages, block_size);
    // any of the kernels may run: which one depends on types, addresses and the size of the pool
    const TreePlan plans[3] = {tree_plan_simt(batch, tokens, q_heads, kv_heads, cap),
                               tree_plan_tc(batch, tokens, q_heads, kv_heads, head_dim, cap, false),
                               tree_plan_tc(batch, tokens, q_heads, kv_heads, head_dim, cap, true)};
    size_t need = 0;
    for (const TreePlan& t : plans) need = std::max(need, tree_scratch(t, tokens, q_heads, head_dim).total);
    return need;
}

int gqa_b200_tree_decode(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                         const int32_t* context_lens, const int32_t* draft_lens, const int64_t* tree_mask, void* out,
                         int dtype, int batch, int tokens, int q_heads, int kv_heads, int head_dim, int64_t num_blocks,
                         int block_size, int max_pages, float scale, int kernel, void* workspace,
                         size_t workspace_bytes, void* stream) {
    if (!known_dtype(dtype)) return GQA_B200_ERR_DTYPE;
    if (batch < 0) return GQA_B200_ERR_BATCH;
    if (tokens < 1 || tokens > kTreeMaxTokens) return GQA_B200_ERR_TREE_TOKENS;
    if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0) return GQA_B200_ERR_HEADS;
    if (head_dim <= 0 || head_dim > 256) return GQA_B200_ERR_HEAD_DIM;
    if (num_blocks <= 0 || block_size <= 0) return GQA_B200_ERR_CACHE_SHAPE;
    if (max_pages <= 0) return GQA_B200_ERR_MAX_PAGES;
    if (!(std::isfinite(scale) && scale > 0.f)) return GQA_B200_ERR_SCALE;
    if (num_blocks > kIntMax || (long long)tokens * q_heads > kTreeMaxRows) return GQA_B200_ERR_INT32_RANGE;
    if (kernel != GQA_B200_KERNEL_AUTO && kernel != GQA_B200_KERNEL_SIMT && kernel != GQA_B200_KERNEL_TCGEN05)
        return GQA_B200_ERR_KERNEL;
    if (batch == 0) return GQA_B200_OK;
    if (!q || !k_cache || !v_cache || !block_table || !context_lens || !out) return GQA_B200_ERR_NULL_POINTER;

    const long long cap = cap_tokens_of(max_pages, block_size);
    const bool tc = kernel != GQA_B200_KERNEL_SIMT && tree_tc_shape(dtype, head_dim, num_blocks, block_size) &&
                    aligned16(q) && aligned16(k_cache) && aligned16(v_cache) && aligned16(out);
    if (kernel == GQA_B200_KERNEL_TCGEN05 && !tc) return GQA_B200_ERR_KERNEL;
    TreeParams p{};
    p.q = q; p.k = k_cache; p.v = v_cache; p.out = out;
    p.table = block_table; p.lens = context_lens; p.draft_lens = draft_lens;
    p.mask = reinterpret_cast<const unsigned long long*>(tree_mask);
    p.batch = batch; p.tokens = tokens; p.q_heads = q_heads; p.kv_heads = kv_heads; p.group = q_heads / kv_heads;
    p.head_dim = head_dim; p.rows = tokens * p.group; p.tile_rows = tree_tile_rows(p.group);
    p.block_size = block_size; p.max_pages = max_pages; p.num_blocks = num_blocks;
    p.bs_shift = -1;
    for (int s = 0; s < 31; ++s)
        if (block_size == 1 << s) p.bs_shift = s;
    p.cap_tokens = (int)cap;
    p.scale_log2 = scale * kLog2e;
    // bytes that rows are read by: what divides a row and the three addresses
    const uintptr_t all = (uintptr_t)head_dim * elem_size(dtype) | reinterpret_cast<uintptr_t>(q) |
                          reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache);
    const int piece = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : elem_size(dtype);
    TreeMaps maps{};
    const bool tma = tc && tree_tma_shape(p.group, head_dim, num_blocks, block_size, (long long)batch * tokens) &&
                     tree_maps(&maps, dtype == GQA_B200_BF16, p);
    const TreePlan plan = tc ? tree_plan_tc(batch, tokens, q_heads, kv_heads, head_dim, cap, tma)
                             : tree_plan_simt(batch, tokens, q_heads, kv_heads, cap);
    const long long cap_tiles = (long long)batch * ((cap + kTreeSimtTile - 1) / kTreeSimtTile);
    if (plan.n_runs * plan.units > kIntMax || cap_tiles / plan.n_runs >= kIntMax / 2) return GQA_B200_ERR_INT32_RANGE;
    const TreeScratch lay = tree_scratch(plan, tokens, q_heads, head_dim);
    // (the published size, whichever kernel runs)
    const size_t need = gqa_b200_tree_workspace_bytes(batch, tokens, q_heads, kv_heads, head_dim, block_size, max_pages);
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < need) return GQA_B200_ERR_WORKSPACE;
    // scratch and result are written while the inputs are read, and scratch is read after the first results are written
    const size_t size = elem_size(dtype), rows = (size_t)batch * tokens * q_heads * head_dim * size;
    const size_t cache = (size_t)num_blocks * block_size * kv_heads * head_dim * size;
    const Span scratch = span_of(workspace, need), result = span_of(out, rows);
    const Span inputs[7] = {span_of(q, rows), span_of(k_cache, cache), span_of(v_cache, cache),
                            span_of(block_table, (size_t)batch * max_pages * sizeof(int32_t)),
                            span_of(context_lens, batch * sizeof(int32_t)),
                            span_of(draft_lens, draft_lens ? batch * sizeof(int32_t) : 0),
                            span_of(tree_mask, tree_mask ? (size_t)batch * tokens * sizeof(int64_t) : 0)};
    if (scratch.meets(result)) return GQA_B200_ERR_OVERLAP;
    for (const Span& x : inputs)
        if (scratch.meets(x) || result.meets(x)) return GQA_B200_ERR_OVERLAP;
    char* ws = static_cast<char*>(workspace);
    p.info = reinterpret_cast<int4*>(ws + lay.info);
    p.part_ml = reinterpret_cast<float2*>(ws + lay.ml);
    p.part_acc = reinterpret_cast<float*>(ws + lay.acc);
    p.n_ranges = plan.n_runs;
    p.row_blocks = plan.row_blocks;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case GQA_B200_F32: return (int)launch_tree<float>(p, plan, tc, tma ? &maps : nullptr, piece, s);
        case GQA_B200_F16: return (int)launch_tree<__half>(p, plan, tc, tma ? &maps : nullptr, piece, s);
        default:           return (int)launch_tree<__nv_bfloat16>(p, plan, tc, tma ? &maps : nullptr, piece, s);
    }
}

int gqa_b200_tree_tc_status(int reset) {
    int host = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&host, g_tree_tc_status, sizeof(int));
    if (e != cudaSuccess) return -(int)e;
    if (reset) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_tree_tc_status, &zero, sizeof(int));
        if (e != cudaSuccess) return -(int)e;
    }
    return host;
}

int gqa_b200_kv_compact(void* k_cache, void* v_cache, const int32_t* block_table, const int32_t* src_positions,
                        const int32_t* dst_positions, int dtype, int batch, int n, int kv_heads, int head_dim,
                        int64_t num_blocks, int block_size, int max_pages, void* stream) {
    if (!known_dtype(dtype)) return GQA_B200_ERR_DTYPE;
    if (batch < 0 || n < 0) return GQA_B200_ERR_BATCH;
    if (n > kCompactMaxRows) return GQA_B200_ERR_COMPACT_ROWS;
    if (kv_heads <= 0) return GQA_B200_ERR_HEADS;
    if (head_dim <= 0) return GQA_B200_ERR_HEAD_DIM;
    if (num_blocks <= 0 || block_size <= 0) return GQA_B200_ERR_CACHE_SHAPE;
    if (max_pages <= 0) return GQA_B200_ERR_MAX_PAGES;
    if (num_blocks > kIntMax) return GQA_B200_ERR_INT32_RANGE;
    if (batch == 0 || n == 0) return GQA_B200_OK;
    if (!k_cache || !v_cache || !block_table || !src_positions || !dst_positions) return GQA_B200_ERR_NULL_POINTER;
    CompactParams p{};
    p.k_cache = k_cache; p.v_cache = v_cache; p.table = block_table; p.src = src_positions; p.dst = dst_positions;
    p.row_bytes = (long long)kv_heads * head_dim * elem_size(dtype);
    p.num_blocks = num_blocks; p.cap_tokens = std::min((long long)max_pages * block_size, kIntMax);
    p.n = n; p.block_size = block_size; p.max_pages = max_pages;
    const int unit = p.row_bytes % 16 == 0 && aligned16(k_cache) && aligned16(v_cache) ? 16 : elem_size(dtype);
    const long long units = p.row_bytes / unit;
    const long long fit = (long long)kCompactThreads * kCompactItems / n;      // >= 1
    p.slice = (int)std::min(units, fit);
    const long long slices = (units + p.slice - 1) / p.slice;
    if (slices > 65535) return GQA_B200_ERR_INT32_RANGE;
    const dim3 grid((unsigned)batch, (unsigned)slices, 2);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (unit == 16) kv_compact_kernel<uint4><<<grid, kCompactThreads, 0, s>>>(p);
    else if (unit == 4) kv_compact_kernel<uint32_t><<<grid, kCompactThreads, 0, s>>>(p);
    else kv_compact_kernel<uint16_t><<<grid, kCompactThreads, 0, s>>>(p);
    return (int)cudaGetLastError();
}

int gqa_b200_kv_copy_pages(void* k_cache, void* v_cache, const int32_t* src_pages, const int32_t* dst_pages, int dtype,
                           int n, int kv_heads, int head_dim, int64_t num_blocks, int block_size, void* stream) {
    if (!known_dtype(dtype)) return GQA_B200_ERR_DTYPE;
    if (n < 0) return GQA_B200_ERR_BATCH;
    if (kv_heads <= 0) return GQA_B200_ERR_HEADS;
    if (head_dim <= 0) return GQA_B200_ERR_HEAD_DIM;
    if (num_blocks <= 0 || block_size <= 0) return GQA_B200_ERR_CACHE_SHAPE;
    if (num_blocks > kIntMax) return GQA_B200_ERR_INT32_RANGE;
    if (n == 0) return GQA_B200_OK;
    if (!k_cache || !v_cache || !src_pages || !dst_pages) return GQA_B200_ERR_NULL_POINTER;
    const long long bytes = (long long)block_size * kv_heads * head_dim * elem_size(dtype);
    const int unit = bytes % 16 == 0 && aligned16(k_cache) && aligned16(v_cache) ? 16 : elem_size(dtype);
    PageCopyParams p{};
    p.k_cache = k_cache; p.v_cache = v_cache; p.src = src_pages; p.dst = dst_pages;
    p.page_units = bytes / unit;
    p.num_blocks = num_blocks;
    p.parts = (p.page_units + kPageCopyThreads * kPageCopyItems - 1) / (kPageCopyThreads * kPageCopyItems);
    if (p.parts * n > kIntMax) return GQA_B200_ERR_INT32_RANGE;
    const dim3 grid((unsigned)(p.parts * n), 2);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (unit == 16) kv_copy_pages_kernel<uint4><<<grid, kPageCopyThreads, 0, s>>>(p);
    else if (unit == 4) kv_copy_pages_kernel<uint32_t><<<grid, kPageCopyThreads, 0, s>>>(p);
    else kv_copy_pages_kernel<uint16_t><<<grid, kPageCopyThreads, 0, s>>>(p);
    return (int)cudaGetLastError();
}

}  // extern "C"
