// Per-head RMS norm of queries and keys, their position rotation, and (append form) the write of
// keys and values into their cache pages, in one pass over the data.
//
//   y = x * rsqrt(mean(x^2) + eps) * w          over the D elements of one head row, fp32
//   (a, b) -> (a cos - b sin, b cos + a sin)    over the first `rot_dim` elements; the pair is
//                                               (y[i], y[i + rot_dim/2]) or (y[2i], y[2i+1])
// and one rounding to the element type at the end.  Values are copied.
//
// A token whose position is outside [0, max_position) is padding: its query (and dense key) rows
// are written as zeros and nothing goes into the cache.  A cache slot outside the table or a page
// id outside the pool is skipped, as in kv_append.
#pragma once

#include <type_traits>

#include "gqa_common.cuh"

namespace gqa_b200 {

struct RopeParams {
    const void* q;
    const void* k;
    const void* v;                // append form only
    const void* q_weight;         // [D] or null: no norm
    const void* k_weight;
    const float* cos_sin;         // [max_position, rot_dim]: rot_dim/2 cosines, then the sines
    const int32_t* positions;     // [batch, tokens]
    const int32_t* slots;         // [batch, tokens], append form
    const int32_t* table;         // [batch, max_pages], append form
    void* q_out;                  // [batch, tokens, q_heads, D]
    void* k_out;                  // [batch, tokens, kv_heads, D], dense form
    void* k_cache;
    void* v_cache;
    long long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;   // strides in elements
    long long num_blocks, cap_tokens;
    long long n_tokens;           // batch * tokens
    int tokens, q_heads, kv_heads, head_dim, rot_dim, max_position;
    int block_size, max_pages;
    int append, interleaved, weight_f32;
    float eps;
};

// Element offset of a token's cache row (all kv heads), or -1: nothing to write.
__device__ __forceinline__ long long rope_cache_row(const RopeParams& p, long long token) {
    const int s = __ldg(p.slots + token);
    if (s < 0 || s >= p.cap_tokens) return -1;
    const int page = s / p.block_size;
    const long long phys = __ldg(p.table + (token / p.tokens) * p.max_pages + page);
    if (phys < 0 || phys >= p.num_blocks) return -1;
    return (phys * p.block_size + (s - page * p.block_size)) * p.kv_heads * p.head_dim;
}

struct RopeRow {
    long long src;   // element offset in q, k or v
    long long dst;   // element offset in the destination; -1: no destination
    int kind;        // 0 query, 1 key, 2 value
};

// Row `h` of a token, counted over query heads, key heads and (append form) value heads.
__device__ __forceinline__ RopeRow rope_row(const RopeParams& p, long long token, int h, long long cache_row) {
    const long long b = token / p.tokens, t = token - b * p.tokens;
    RopeRow r;
    if (h < p.q_heads) {
        r.kind = 0;
        r.src = b * p.q_sb + t * p.q_st + h * p.q_sh;
        r.dst = (token * p.q_heads + h) * p.head_dim;
        return r;
    }
    h -= p.q_heads;
    r.kind = 1;
    r.src = b * p.k_sb + t * p.k_st + h * p.k_sh;
    if (h >= p.kv_heads) {
        h -= p.kv_heads;
        r.kind = 2;
        r.src = b * p.v_sb + t * p.v_st + h * p.v_sh;
    }
    if (p.append) r.dst = cache_row < 0 ? -1 : cache_row + (long long)h * p.head_dim;
    else r.dst = (token * p.kv_heads + h) * p.head_dim;
    return r;
}

template <typename T> __device__ __forceinline__ const T* rope_src(const RopeParams& p, const RopeRow& r) {
    return static_cast<const T*>(r.kind == 0 ? p.q : r.kind == 1 ? p.k : p.v) + r.src;
}
template <typename T> __device__ __forceinline__ T* rope_dst(const RopeParams& p, const RopeRow& r) {
    T* base = static_cast<T*>(r.kind == 0 ? p.q_out : r.kind == 2 ? p.v_cache : p.append ? p.k_cache : p.k_out);
    return base + r.dst;
}
template <typename T> __device__ __forceinline__ float rope_weight(const RopeParams& p, int kind, int e) {
    const void* w = kind == 0 ? p.q_weight : p.k_weight;
    if (!w) return 1.f;
    return p.weight_f32 ? static_cast<const float*>(w)[e] : to_f32<T>(static_cast<const T*>(w)[e]);
}

// Every head_dim in [1, 256], every alignment and stride: one warp per head row, elements lane,
// lane + 32, ...  A lane also reads the partners of its elements (first-level cache hits), and
// every read of the row precedes its writes, so the output may be the input.
// Bound by issue, an element at a time: 16384 tokens x 72 heads of 100 16-bit elements take 840 us (0.57 TB/s),
// of 128 with 28 rotated 685, where the kernel below takes 117.
constexpr int kRopeWarps = 4;
template <typename T>
__global__ void __launch_bounds__(kRopeWarps * 32) qk_norm_rope_any_kernel(const RopeParams p) {
    constexpr int E = 8;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int heads = p.q_heads + p.kv_heads * (p.append ? 2 : 1);
    const long long row = (long long)blockIdx.x * kRopeWarps + warp;
    if (row >= p.n_tokens * heads) return;
    const long long token = row / heads;
    const int pos = __ldg(p.positions + token);
    const bool live = pos >= 0 && pos < p.max_position;
    const int D = p.head_dim, half = p.rot_dim / 2;
    const RopeRow r = rope_row(p, token, (int)(row - token * heads), p.append ? rope_cache_row(p, token) : 0);
    if (r.dst < 0) return;
    if (p.append && r.kind != 0 && !live) return;
    const T* src = rope_src<T>(p, r);
    T* dst = rope_dst<T>(p, r);
    float x[E], y[E];
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const int e = lane + 32 * j;
        int o = e;                                     // the other element of e's pair
        if (e < 2 * half) o = p.interleaved ? e ^ 1 : (e < half ? e + half : e - half);
        x[j] = e < D ? to_f32<T>(src[e]) : 0.f;
        y[j] = e < D ? to_f32<T>(src[o]) : 0.f;
        ss = fmaf(x[j], x[j], ss);
    }
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, s);
    const bool norm = p.q_weight != nullptr;
    const float rs = norm ? rsqrtf(ss / (float)D + p.eps) : 1.f;
    const float* cs = p.cos_sin + (long long)(live ? pos : 0) * p.rot_dim;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const int e = lane + 32 * j;
        if (e >= D) continue;
        if (r.kind == 2) { dst[e] = from_f32<T>(x[j]); continue; }
        if (!live) { dst[e] = from_f32<T>(0.f); continue; }   // (padding reads no angles: the table may be empty)
        float a = x[j] * rs * rope_weight<T>(p, r.kind, e);
        if (e < 2 * half) {
            const int o = p.interleaved ? e ^ 1 : (e < half ? e + half : e - half);
            const int i = p.interleaved ? e >> 1 : (e < half ? e : e - half);
            const bool first = p.interleaved ? !(e & 1) : e < half;
            const float b = y[j] * rs * rope_weight<T>(p, r.kind, o);
            a = a * __ldg(cs + i) + (first ? -b : b) * __ldg(cs + half + i);
        }
        dst[e] = from_f32<T>(a);
    }
}

// ---------------------------------------------------------------------------
// Aligned rows of whole eight-element chunks: a group of L lanes per head row, two chunks of four
// elements per lane, HB heads of a token one after the other.  The chunks are chosen so that both
// elements of a pair are in the lane: 4 l and rot_dim/2 + 4 l (halves), or 8 l and 8 l + 4 (interleaved,
// and behind rot_dim); a lane needs four cosines and four sines, and nothing crosses lanes but the sum.
// (With eight consecutive elements per lane the partner came by shuffle and a lane read 64 bytes of
// angles: 190 us for 16384 tokens of 72 heads of 128 16-bit elements.)  All loads of the HB rows are
// issued before the first is used, the angles are loaded once for all of them.
// Memory bound: 2 bytes read and 2 written per element of 16 bits (116 us for those tokens, 0.80 of the
// measured copy bandwidth; float32 1.0), and not far from the issue rate, hence the packed fp32 forms.
// ---------------------------------------------------------------------------
constexpr int kRopeThreads = 256;

template <typename T> struct RopeVec {                 // two chunks of four elements
    using Chunk = typename std::conditional<sizeof(T) == 2, uint2, uint4>::type;
    Chunk c[2];
    __device__ __forceinline__ void load(const T* p, int e0, int e1) {
        c[0] = *reinterpret_cast<const Chunk*>(p + e0);
        c[1] = *reinterpret_cast<const Chunk*>(p + e1);
    }
    __device__ __forceinline__ void store(T* p, int e0, int e1) const {
        *reinterpret_cast<Chunk*>(p + e0) = c[0];
        *reinterpret_cast<Chunk*>(p + e1) = c[1];
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const T* e = reinterpret_cast<const T*>(c);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(e[i]);
    }
    __device__ __forceinline__ void set(const float (&x)[8]) {
        T* e = reinterpret_cast<T*>(c);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
    }
};

// packed fp32 pairs: half the instructions of the scalar forms
__device__ __forceinline__ void rope_mul2(float* d, const float* a, const float* b) {
    asm("{\n\t.reg .b64 ra, rb;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
        "mul.rn.f32x2 ra, ra, rb;\n\tmov.b64 {%0, %1}, ra;\n\t}"
        : "=f"(d[0]), "=f"(d[1]) : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]));
}
__device__ __forceinline__ void rope_fma2(float* d, const float* a, const float* b, const float* c) {
    asm("{\n\t.reg .b64 ra, rb, rc;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
        "fma.rn.f32x2 ra, ra, rb, rc;\n\tmov.b64 {%0, %1}, ra;\n\t}"
        : "=f"(d[0]), "=f"(d[1]) : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]), "f"(c[0]), "f"(c[1]));
}

// A token has blocks of HB query heads, then of key heads, then (append form) of value heads.
struct RopeBlocks {
    unsigned q, k, all;
};

template <typename T, int L, int HB, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads, 4)
qk_norm_rope_vec_kernel(const RopeParams p, const RopeBlocks blocks, const unsigned units) {
    constexpr unsigned GROUPS = kRopeThreads / L;
    const int lane = threadIdx.x % L;
    const unsigned unit = blockIdx.x * GROUPS + threadIdx.x / L;
    const bool work = unit < units;                    // (no early return: the shuffles name whole warps)
    const unsigned token = work ? unit / blocks.all : 0, block = work ? unit - token * blocks.all : 0;
    const int pos = __ldg(p.positions + token);
    const bool live = pos >= 0 && pos < p.max_position;
    const unsigned b = token / (unsigned)p.tokens, t = token - b * (unsigned)p.tokens;
    const int D = p.head_dim, half = p.rot_dim / 2;
    const bool mine = work && lane * 8 < D, turned = lane * 8 < p.rot_dim;
    const bool halves = !INTERLEAVED && turned;        // this lane's pairs are (first chunk, second chunk)
    const int e0 = halves ? lane * 4 : lane * 8, e1 = halves ? half + lane * 4 : lane * 8 + 4;

    // the block's kind, its heads, where they lie and go
    const T* src;
    T* dst;
    long long step;
    const void* weight = nullptr;
    int count;
    bool goes = true, value = false;
    if (block < blocks.q) {
        const int h0 = block * HB;
        count = p.q_heads - h0;
        step = p.q_sh;
        src = static_cast<const T*>(p.q) + b * p.q_sb + t * p.q_st + h0 * step;
        dst = static_cast<T*>(p.q_out) + ((long long)token * p.q_heads + h0) * D;
        weight = p.q_weight;
    } else {
        value = block >= blocks.q + blocks.k;
        const int h0 = (block - blocks.q - (value ? blocks.k : 0)) * HB;
        count = p.kv_heads - h0;
        step = value ? p.v_sh : p.k_sh;
        src = value ? static_cast<const T*>(p.v) + b * p.v_sb + t * p.v_st : static_cast<const T*>(p.k) + b * p.k_sb + t * p.k_st;
        src += h0 * step;
        weight = value ? nullptr : p.k_weight;
        if (p.append) {
            const long long row = live ? rope_cache_row(p, token) : -1;
            goes = row >= 0;
            dst = static_cast<T*>(value ? p.v_cache : p.k_cache) + row + (long long)h0 * D;
        } else {
            dst = static_cast<T*>(p.k_out) + ((long long)token * p.kv_heads + h0) * D;
        }
    }
    RopeVec<T> x[HB];
#pragma unroll
    for (int j = 0; j < HB; ++j)
        if (mine && j < count) x[j].load(src + j * step, e0, e1);
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.f;
    if (weight && mine) {
        if (p.weight_f32) {
            RopeVec<float> f;
            f.load(static_cast<const float*>(weight), e0, e1);
            f.get(w);
        } else {
            RopeVec<T> f;
            f.load(static_cast<const T*>(weight), e0, e1);
            f.get(w);
        }
    }
    // the angles of this lane's four pairs
    float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mine && turned && live && !value) {
        const float* at = p.cos_sin + (long long)pos * p.rot_dim + lane * 4;
        cs = __ldg(reinterpret_cast<const float4*>(at));
        sn = __ldg(reinterpret_cast<const float4*>(at + half));
    }
    const float ca[4] = {cs.x, cs.y, cs.z, cs.w}, sa[4] = {sn.x, sn.y, sn.z, sn.w};
    const float ms[4] = {-sn.x, -sn.y, -sn.z, -sn.w};
#pragma unroll
    for (int j = 0; j < HB; ++j) {
        // (the groups of a warp may have blocks of different kinds: all take part in the shuffles)
        float v[8];
        if (mine && j < count) {
            x[j].get(v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
        }
        float rs = 1.f;
        if (p.q_weight) {
            float s2[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 8; i += 2) rope_fma2(s2, v + i, v + i, s2);
            float ss = s2[0] + s2[1];
#pragma unroll
            for (int z = L / 2; z >= 1; z >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, z, L);
            rs = rsqrtf(ss / (float)D + p.eps);
        }
        if (!mine || j >= count || !goes) continue;
        if (!value) {
            const float r2[2] = {rs, rs};
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                rope_mul2(y + i, w + i, r2);
                rope_mul2(v + i, v + i, y + i);
            }
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    y[2 * i] = v[2 * i] * ca[i] - v[2 * i + 1] * sa[i];
                    y[2 * i + 1] = v[2 * i + 1] * ca[i] + v[2 * i] * sa[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    rope_mul2(y + i, v + i + 4, ms + i);
                    rope_fma2(y + i, v + i, ca + i, y + i);
                    rope_mul2(y + i + 4, v + i, sa + i);
                    rope_fma2(y + i + 4, v + i + 4, ca + i, y + i + 4);
                }
            }
            if (!live) {                               // padding: query (and dense key) rows of zeros
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = 0.f;
            }
            x[j].set(y);
        }
        x[j].store(dst + j * D, e0, e1);
    }
}

}  // namespace gqa_b200
