// paged4.cuh — what the paged 4-bit cache's kernels share (paged4_append.cu, paged4_attn.cu, paged4_attn_wide.cu).
//
// A row of a KV head (head_dim values of one token) is kept as groups of 16 values: a code of 4 bits a value and a scale
// byte a group, keys and values apart, 4.5 bits a value. Code c stands for 0, .5, 1, 1.5, 2, 3, 4, 6 (c & 7) with the
// sign of bit 3 (e2m1); scale byte b for the f16 number of the bits b << 7, five of exponent and three of fraction. A value is
// code x scale: at most six bits of fraction, so f16 holds it exactly (2^-15 to 61440), and so do bf16 and f32: what the
// kernels multiply is what the cache stands for. Per (page, KV head):
//   codes   [page_tokens][head_dim / 2]    byte i of a row: dims 2 i (low half) and 2 i + 1
//   scales  [page_tokens][head_dim / 16]
// A row's codes and scales depend on that row alone, so a call never touches what an earlier one wrote. A group that held a
// NaN or an infinity has the scale byte 255 (f16 NaN) and reads as NaN. The largest scale is 10240; for the attention every byte above it says that the group
// is no number, whoever wrote it: a code of 6 under the next one is past f16's end, and an infinity among the values would reach the rows that do not see it.
#pragma once
#include "paged.cuh"

namespace spk {
namespace paged4 {

using paged::BLOCK;
using paged::Batch;
using paged::MAX_SEQ;
using paged::T_BF16;
using paged::T_F16;
using paged::T_F32;

constexpr int GROUP = 16;                       // values that share a scale
constexpr float SCALE_MIN = 0x1p-14f, SCALE_MAX = 10240.0f;   // 6 x 10240 is the largest six-bit number under f16's end
constexpr uint32_t POISON = 0xe3;               // scale bytes from here on, above SCALE_MAX, are no numbers

struct Pool {
    uint8_t *k, *v, *ks, *vs;
    int pages, page_tokens, kv_heads, hd;
};
inline Pool pool_of(const spk_kv4_pool *p) {
    return Pool{(uint8_t *)p->k, (uint8_t *)p->v, (uint8_t *)p->k_scale, (uint8_t *)p->v_scale, p->pages, p->page_tokens, p->kv_heads, p->head_dim};
}
int check_pool(const spk_kv4_pool *p, const char *who);

// A token's row among the rows of a pool: (page, KV head, token of the page).
__device__ __forceinline__ size_t row_index(const Pool &p, int page, int head, int tok) {
    return ((size_t)page * p.kv_heads + head) * p.page_tokens + tok;
}

// The two values of a byte of codes, f16: the low half's in the low half.
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {   // a in the low half
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
// Whether one of four scale bytes is no number: the upper bit, and a carry into it from the others.
__device__ __forceinline__ uint32_t poisoned(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u * (0x100u - POISON)) & w & 0x80808080u; }

// The attention's arguments. A kernel takes the sequences whose rows per KV head (rows x group) are from `from` to `to`.
struct AttnParams {
    Pool pool;
    Batch b;
    const void *q, *gate;
    void *out;
    long long ldq, ldgate, ldout;
    int heads, group, window;
    float scale;                                        // softmax scale * log2(e)
    long long from, to;
    unsigned int *tickets;                              // [gridDim.x], zero at rest
    float *part;                                        // [gridDim.x][2][part_floats]
    int *err;
    __device__ __forceinline__ bool takes(long long columns) const { return columns >= from && columns <= to; }
};
// Weights are f16 numbers 2^(s - m): a new reference m puts the row's largest at 2^W_TOP (the kernel for many rows: less), and it moves when
// one passes 2^W_MAX. A weight is kept down to 2^-24: 2^-36 of the largest (many rows: 2^-34 in f32, 2^-30 in the 16-bit types).
// f32 rows' weights are two f16 numbers, 22 bits. 16-bit rows' are one: off by half a step, 2^-11 of each weight, either way and so averaged over the keys, and what
// is divided by is the sum of the weights as they were rounded (bf16 many rows: before, which bf16's own half step of 2^-8 hides). Against 64 bits that is 1e-5 beside the
// 2e-4 of f16's output (24 x 8 rows), nothing beside bf16's; a second term would multiply the values twice.
constexpr float W_TOP = 12.0f, W_MAX = 15.0f;

// Floats of one CTA's part of a group of R query rows: O, then m, then l.
__host__ __device__ constexpr int part_floats(int R, int hd) { return R * (hd + 2); }
// the kernel for many rows: query rows of a group, its fixed cost in blocks (13 f32 prompts 125 us; 129 with 24, 130 with 64, 139 with 128)
constexpr int WIDE_R = 128, WIDE_COST = 40;
int attn_wide(const AttnParams &a, int type, cudaStream_t s, const char *who);   // paged4_attn_wide.cu

}  // namespace paged4
}  // namespace spk
