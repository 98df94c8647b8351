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

// Two f32 side by side, each operation rounded as its scalar form.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Cosine and sine of the f32 product position * frequency (model.rs:431-439's angle). The whole turns
// are taken out with 1 / 2 pi as the sum of two f32 and the product's own rounding error added, so a turn
// count up to 2^24 still leaves 24 bits of the fraction, and the rest goes to sincospi: one path for every
// position, where sincosf branches at large angles.
__device__ __forceinline__ void angle(int pos, float freq, float &c, float &s) {
    constexpr double INV = 0.15915494309189533577;
    constexpr float HI = (float)INV, LO = (float)(INV - (double)HI);
    const float p = __fmul_rn((float)pos, freq), t = __fmul_rn(p, HI);
    const float rest = __fmaf_rn(p, LO, __fmaf_rn(p, HI, -t));
    sincospif(2.0f * ((t - rintf(t)) + rest), &s, &c);
}

// 8 values of a row as they lie in memory: two pieces of 4 (dims d0 .. and d1 ..)
template <typename T>
struct Raw {
    uint32_t w[2 * sizeof(T)];
    __device__ __forceinline__ void load(const T *row, int d0, int d1, int vec) {
        if (sizeof(T) == 2 && vec == 2 && d1 == d0 + 4) {
            const uint4 a = __ldg(reinterpret_cast<const uint4 *>(row + d0));
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else if (vec) {
            if constexpr (sizeof(T) == 2) {
                const uint2 a = __ldg(reinterpret_cast<const uint2 *>(row + d0)), b = __ldg(reinterpret_cast<const uint2 *>(row + d1));
                w[0] = a.x, w[1] = a.y, w[2] = b.x, w[3] = b.y;
            } else {
                const uint4 a = __ldg(reinterpret_cast<const uint4 *>(row + d0)), b = __ldg(reinterpret_cast<const uint4 *>(row + d1));
                w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
                w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const T *p = row + (e < 4 ? d0 + e : d1 + e - 4);
                if constexpr (sizeof(T) == 4) w[e] = *reinterpret_cast<const uint32_t *>(p);
                else {
                    const uint32_t h = *reinterpret_cast<const uint16_t *>(p);
                    w[e >> 1] = e & 1 ? w[e >> 1] | (h << 16) : h;
                }
            }
        }
    }
    __device__ __forceinline__ void none() {
#pragma unroll
        for (int i = 0; i < (int)(2 * sizeof(T)); i++) w[i] = 0;
    }
    __device__ __forceinline__ void f32(float (&x)[8]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (__is_same(T, __half)) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                    x[2 * i] = f.x, x[2 * i + 1] = f.y;
                } else {
                    x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                }
            }
        }
    }
};

// The rotation of a unit's 4 pairs, each product rounded (model.rs:431-439).
__device__ __forceinline__ void rotate_unit(float (&a)[4], float (&b)[4], const float (&c)[4], const float (&s)[4]) {
    const f32x2 minus = pack2(-1.0f, -1.0f);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const f32x2 p = pack2(a[i], a[i + 1]), q = pack2(b[i], b[i + 1]), cc = pack2(c[i], c[i + 1]), ss = pack2(s[i], s[i + 1]);
        const float2 x = unpack2(fma2(mul2(q, ss), minus, mul2(p, cc))), y = unpack2(add2(mul2(q, cc), mul2(p, ss)));
        a[i] = x.x, a[i + 1] = x.y;
        b[i] = y.x, b[i + 1] = y.y;
    }
}

// Alignment of the pieces of rows at p with stride ld (elements of `size` bytes): 0 none, 1 four values,
// 2 eight, too.
inline int rows_aligned(const void *p, long long ld, int size) {
    if ((uintptr_t)p % (4 * size) || ld % 4) return 0;
    return (uintptr_t)p % (8 * size) == 0 && ld % 8 == 0 ? 2 : 1;
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
