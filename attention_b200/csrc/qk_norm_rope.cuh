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
        float a = x[j] * rs * rope_weight<T>(p, r.kind, e);
        if (e < 2 * half) {
            const int o = p.interleaved ? e ^ 1 : (e < half ? e + half : e - half);
            const int i = p.interleaved ? e >> 1 : (e < half ? e : e - half);
            const bool first = p.interleaved ? !(e & 1) : e < half;
            const float b = y[j] * rs * rope_weight<T>(p, r.kind, o);
            a = a * __ldg(cs + i) + (first ? -b : b) * __ldg(cs + half + i);
        }
        dst[e] = from_f32<T>(live ? a : 0.f);
    }
}

// ---------------------------------------------------------------------------
// Rows of whole 16-byte chunks, aligned: a group of L lanes per head row, eight consecutive elements
// per lane, HB heads of a token one after the other.  All loads of the HB rows are issued before the
// first is used.  The token's cosines and sines are loaded once for the HB heads (for eight 16-bit
// elements they are as many as 64 bytes against 16: one head per group is bound by the first-level
// cache, see the launcher).  The partner of an element is in the same lane (interleaved) or rot_dim/2
// elements away, rot_dim/16 lanes, so a shuffle fetches it after the scaling.
// Memory bound: 2 bytes read and 2 written per element of 16 bits.
// ---------------------------------------------------------------------------
constexpr int kRopeThreads = 256;

template <typename T> struct RopeVec {                 // eight elements of a lane
    uint4 raw[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = raw[i];
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(e[i]);
    }
    __device__ __forceinline__ void set(const float (&x)[8]) {
        T* e = reinterpret_cast<T*>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
    }
};

template <typename T, int L, int HB, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_vec_kernel(const RopeParams p, const int blocks_per_token) {
    constexpr int GROUPS = kRopeThreads / L;
    const int lane = threadIdx.x % L;
    const long long unit = (long long)blockIdx.x * GROUPS + threadIdx.x / L;
    const long long units = p.n_tokens * blocks_per_token;
    const bool work = unit < units;                    // (no early return: the shuffles name whole warps)
    const long long token = work ? unit / blocks_per_token : 0;
    const int h0 = work ? (int)(unit - token * blocks_per_token) * HB : 0;
    const int heads = p.q_heads + p.kv_heads * (p.append ? 2 : 1);
    const int D = p.head_dim, e0 = lane * 8;
    const bool mine = work && e0 < D;
    const int pos = __ldg(p.positions + token);
    const bool live = pos >= 0 && pos < p.max_position;
    const long long cache_row = p.append && h0 + HB > p.q_heads ? rope_cache_row(p, token) : -1;

    RopeVec<T> x[HB];
    RopeRow r[HB];
#pragma unroll
    for (int j = 0; j < HB; ++j) {
        r[j].dst = -1;
        if (mine && h0 + j < heads) {
            r[j] = rope_row(p, token, h0 + j, cache_row);
            if (p.append && r[j].kind != 0 && !live) r[j].dst = -1;
            x[j].load(rope_src<T>(p, r[j]) + e0);
        }
    }
    // angles of this lane's elements; beyond rot_dim (and for padding) cosine 1, sine 0
    const int half = p.rot_dim / 2;
    const bool turned = mine && e0 < p.rot_dim;
    float c[8], s[8];
    if (h0 < p.q_heads + p.kv_heads) {
        const float* cs = p.cos_sin + (long long)(live ? pos : 0) * p.rot_dim;
        if constexpr (INTERLEAVED) {
            float4 a = make_float4(1.f, 1.f, 1.f, 1.f), b = make_float4(0.f, 0.f, 0.f, 0.f);
            if (turned && live) {
                a = __ldg(reinterpret_cast<const float4*>(cs + e0 / 2));
                b = __ldg(reinterpret_cast<const float4*>(cs + half + e0 / 2));
            }
            c[0] = c[1] = a.x; c[2] = c[3] = a.y; c[4] = c[5] = a.z; c[6] = c[7] = a.w;
            s[1] = b.x; s[3] = b.y; s[5] = b.z; s[7] = b.w;
            s[0] = -b.x; s[2] = -b.y; s[4] = -b.z; s[6] = -b.w;
        } else {
            const int i0 = e0 < half ? e0 : e0 - half;
            float4 a[2] = {make_float4(1.f, 1.f, 1.f, 1.f), make_float4(1.f, 1.f, 1.f, 1.f)};
            float4 b[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
            if (turned && live) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    a[i] = __ldg(reinterpret_cast<const float4*>(cs + i0) + i);
                    b[i] = __ldg(reinterpret_cast<const float4*>(cs + half + i0) + i);
                }
            }
            const float sign = e0 < half ? -1.f : 1.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                c[4 * i] = a[i].x; c[4 * i + 1] = a[i].y; c[4 * i + 2] = a[i].z; c[4 * i + 3] = a[i].w;
                s[4 * i] = sign * b[i].x; s[4 * i + 1] = sign * b[i].y; s[4 * i + 2] = sign * b[i].z; s[4 * i + 3] = sign * b[i].w;
            }
        }
    }
    const bool norm = p.q_weight != nullptr;
    const int partner = turned ? (e0 < half ? lane + half / 8 : lane - half / 8) : lane;
#pragma unroll
    for (int j = 0; j < HB; ++j) {
        const int kind = h0 + j < p.q_heads ? 0 : h0 + j < p.q_heads + p.kv_heads ? 1 : 2;
        // (the heads of a warp's groups may differ in kind: every lane takes part in the shuffles)
        float v[8], ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
        const bool row = mine && h0 + j < heads;
        if (row) x[j].get(v);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
#pragma unroll
        for (int z = L / 2; z >= 1; z >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, z, L);
        const float rs = norm ? rsqrtf(ss / (float)D + p.eps) : 1.f;
        if (row && norm && kind != 2) {
            const void* w = kind == 0 ? p.q_weight : p.k_weight;
            float wf[8];
            if (p.weight_f32) {
                RopeVec<float> t;
                t.load(static_cast<const float*>(w) + e0);
                t.get(wf);
            } else {
                RopeVec<T> t;
                t.load(static_cast<const T*>(w) + e0);
                t.get(wf);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= rs * wf[i];
        }
        float o[8];
        if constexpr (INTERLEAVED) {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = v[i ^ 1];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xffffffffu, v[i], partner, L);
        }
        if (row && r[j].dst >= 0) {
            if (kind != 2) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = live ? fmaf(v[i], c[i], o[i] * s[i]) : 0.f;
                x[j].set(v);
            }
            x[j].store(rope_dst<T>(p, r[j]) + e0);
        }
    }
}

}  // namespace gqa_b200
