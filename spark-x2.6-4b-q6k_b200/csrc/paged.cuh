// paged.cuh — what the paged 8-bit cache's kernels share (paged_append.cu, paged_attn.cu).
//
// The cache holds e4m3 bytes under one f32 scale per (block of 16 tokens, KV head), keys and
// values apart. A page is page_tokens (a multiple of 16) tokens of every KV head; per (page, head):
//   keys    [page_tokens / 8][hd / 16][8 tokens][16 dims]
//   values  [page_tokens / 16][hd][16 tokens], byte b of a dim's 16 holding token order(b)
// Both are what the tensor cores read with no re-lay: 8-row x 16-byte core matrices (K-major, keys
// of stride 8 hd, values of stride 128), and 4 bytes that are one thread's share of an m16n8k16
// A operand; a block's keys (16 hd bytes) and its values lie contiguous, one bulk copy each.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "spk.h"

namespace spk {
namespace paged {

constexpr int BLOCK = 16;                 // tokens that share a scale
constexpr float E4M3_MAX = 448.0f;
constexpr float SCALE_MIN = 0x1p-100f;    // so that no scale is 0 and its log2 stays finite
constexpr int MAX_SEQ = 1024;             // sequences per call

enum : int { T_F32 = 0, T_F16 = 1, T_BF16 = 2 };

struct Pool {
    uint8_t *k, *v;
    float *ks, *vs;
    int pages, page_tokens, kv_heads, hd;
};
struct Batch {
    int nseq, rows;
    const int *row0, *kv_len, *table;
    int max_pages;
};

// Value bytes: token order(b) at byte b, byte place(i) for token i.
__host__ __device__ constexpr int order(int b) { return 2 * (b >> 2) + (b & 1) + 8 * ((b >> 1) & 1); }
__host__ __device__ constexpr int place(int i) { return 4 * ((i & 7) >> 1) + (i & 1) + 2 * (i >> 3); }

// Block `blk` of a page: its place among the blocks of the pool for one KV head.
__device__ __forceinline__ size_t block_index(const Pool &p, int page, int head, int blk) {
    return ((size_t)page * p.kv_heads + head) * (p.page_tokens / BLOCK) + blk;
}

// 4 consecutive values as f32; vec: the 4 values' address is a multiple of their size.
template <typename T>
__device__ __forceinline__ float4 load4(const T *p, bool vec);
template <>
__device__ __forceinline__ float4 load4<float>(const float *p, bool vec) {
    if (vec) return __ldg(reinterpret_cast<const float4 *>(p));
    return make_float4(p[0], p[1], p[2], p[3]);
}
template <>
__device__ __forceinline__ float4 load4<__half>(const __half *p, bool vec) {
    if (!vec) return make_float4(__half2float(p[0]), __half2float(p[1]), __half2float(p[2]), __half2float(p[3]));
    const uint2 w = __ldg(reinterpret_cast<const uint2 *>(p));
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16 *p, bool vec) {
    if (!vec)
        return make_float4(__bfloat162float(p[0]), __bfloat162float(p[1]), __bfloat162float(p[2]),
                           __bfloat162float(p[3]));
    const uint2 w = __ldg(reinterpret_cast<const uint2 *>(p));
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
}

// A row of hd values is handled as hd / 8 units of two 4-value pieces, so that a rotated pair
// (i, i + pdim / 2) is in one thread: unit u < pdim / 8 holds dims 4u .. and pdim / 2 + 4u ..,
// the others 8 consecutive dims. The first dims of unit u's pieces:
__device__ __forceinline__ void unit_dims(int u, int pdim, int &d0, int &d1) {
    if (u < pdim / 8) {
        d0 = 4 * u;
        d1 = pdim / 2 + 4 * u;
    } else {
        d0 = 8 * u;
        d1 = d0 + 4;
    }
}

// Cosine and sine of the f32 product position * frequency (model.rs:431-439's angle). The whole turns
// are taken out in f64, where a turn count up to 2^24 still leaves 29 bits of the fraction, and the
// rest goes to sincospi: one path for every position, where sincosf branches at large angles.
__device__ __forceinline__ void angle(int pos, float freq, float &c, float &s) {
    const double turns = (double)__fmul_rn((float)pos, freq) * 0.15915494309189533577;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
}

template <typename T>
__device__ __forceinline__ void load_unit(const T *row, int u, int pdim, bool vec, float (&a)[4], float (&b)[4]) {
    int d0, d1;
    unit_dims(u, pdim, d0, d1);
    const float4 x = load4<T>(row + d0, vec), y = load4<T>(row + d1, vec);
    a[0] = x.x, a[1] = x.y, a[2] = x.z, a[3] = x.w;
    b[0] = y.x, b[1] = y.y, b[2] = y.z, b[3] = y.w;
}
// The rotation of a unit's 4 pairs, each product rounded (model.rs:431-439).
__device__ __forceinline__ void rotate_unit(float (&a)[4], float (&b)[4], const float (&c)[4], const float (&s)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float p = a[i], q = b[i];
        a[i] = __fsub_rn(__fmul_rn(p, c[i]), __fmul_rn(q, s[i]));
        b[i] = __fadd_rn(__fmul_rn(q, c[i]), __fmul_rn(p, s[i]));
    }
}

// Whether 4-value pieces of rows at p with stride ld (elements of `size` bytes) are aligned.
inline bool rows_aligned(const void *p, long long ld, int size) {
    return ((uintptr_t)p % (4 * size)) == 0 && (ld % 4) == 0;
}

int check_pool(const spk_kv_pool *p, const char *who);
int check_batch(const spk_kv_batch *b, const char *who);
inline Pool pool_of(const spk_kv_pool *p) {
    return Pool{(uint8_t *)p->k, (uint8_t *)p->v, p->k_scale, p->v_scale, p->pages, p->page_tokens, p->kv_heads,
                p->head_dim};
}
inline Batch batch_of(const spk_kv_batch *b) {
    return Batch{b->nseq, b->rows, b->row0, b->kv_len, b->table, b->max_pages};
}

}  // namespace paged
}  // namespace spk
