// paged4_append.cu — a projection's rows into the pages of the 4-bit cache, and cached rows back.
//
// append: row t of the call is q heads, keys and values of one token. Per head of queries and keys, where asked for,
//   x' = x r w,  r = 1 / sqrt(mean x^2 + eps);   then a rotation of pairs by the angle f32(position * freq[i]):
//   (a, b) -> (a cos - b sin, b cos + a sin), pairs (i, i + pdim / 2) or (2 i, 2 i + 1).
// Queries leave in their own type. Keys and values are rounded, per group of 16 values:
//   d = the number of 4 significant bits nearest to amax / 6 (ties to even), within [2^-14, 10240]
//   code = the e2m1 number nearest to x / d (ties to the even code, at most 6)
// Both are decided exactly: for d the f32 quotient's neighbour is checked against 6 (d + half a step), which f32 holds; the quotient
// x / d is corrected by its own residual, so that a tie is a tie, and moved off a border that it was only rounded to.
//
// What bounds append: the rows' bytes. A warp takes 256 values (256 / head_dim heads side by side), 8 consecutive ones a
// lane, which is one 16-byte load of 16-bit rows and one word of codes; a group is two lanes, a head's norm a shuffle tree, the other half of a
// rotated pair 8 shuffles. A CTA takes a tile of tokens, whose angles it computes once for all heads.
#include "paged4.cuh"

namespace spk {
namespace paged4 {

int check_pool(const spk_kv4_pool *p, const char *who) {
    if (!p || !p->k || !p->v || !p->k_scale || !p->v_scale) return set_error("%s: the pool has a null buffer", who);
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
        return set_error("%s: head_dim %d (64, 128 or 256)", who, p->head_dim);
    if (p->pages < 1 || p->kv_heads < 1 || p->page_tokens < BLOCK || p->page_tokens % BLOCK)
        return set_error("%s: %d pages of %d tokens (a multiple of 16), %d KV heads", who, p->pages, p->page_tokens, p->kv_heads);
    if (((uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->k_scale | (uintptr_t)p->v_scale) % 16)
        return set_error("%s: the pool is not 16-byte aligned", who);
    return 0;
}

namespace {

constexpr int AP_WARPS = 8, AP_THREADS = AP_WARPS * 32;
constexpr int MAX_TILE = 16;               // tokens of a tile

struct AppendArgs {
    Pool pool;
    Batch b;
    const void *q, *k, *v;
    void *q_out;
    long long ldq, ldqo, ldk, ldv;
    int vec;                               // 16-byte pieces: bit 0 q, 1 q_out, 2 k, 3 v
    const float *qw, *kw, *freq;
    int heads, pdim, interleaved, tile;    // q heads (0: none), rotated dims, tokens of a tile
    float eps;
    int *err;
};

template <typename T>
__device__ __forceinline__ void load8(const T *p, bool vec, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        if (vec) {
            const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = p[i];
        }
    } else {
        uint32_t w[4];
        if (vec) {
            const uint4 a = *reinterpret_cast<const uint4 *>(p);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                w[i] = reinterpret_cast<const uint16_t *>(p)[2 * i] | (uint32_t)reinterpret_cast<const uint16_t *>(p)[2 * i + 1] << 16;
        }
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
template <typename T>
__device__ __forceinline__ uint32_t two(float a, float b) {   // 16-bit types: a pair, a in the low half
    if constexpr (__is_same(T, __half)) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, bool vec, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        if (vec) {
            reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
            reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = x[i];
        }
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = two<T>(x[2 * i], x[2 * i + 1]);
        if (vec) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else {
#pragma unroll
            for (int i = 0; i < 8; i++) reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        }
    }
}

// The scale of a group whose largest magnitude is amax: its byte, and d.
__device__ __forceinline__ uint32_t scale_of(float amax, float &d) {
    if (!(amax < INFINITY)) {
        d = 0.f;
        return 0xffu;
    }
    const float t = fminf(fmaxf(__fdiv_rn(amax, 6.0f), SCALE_MIN), SCALE_MAX);
    uint32_t b = __float_as_uint(t) >> 20;                        // the 4 leading bits
    const float mid = __uint_as_float((b << 20) | 0x80000u);      // and the middle to the next
    const float six = 6.0f * mid;                                 // 8 bits: exact
    if (t < SCALE_MAX && (amax > six || (amax == six && (b & 1)))) b++;
    d = __uint_as_float(b << 20);
    return b - (112u << 3);                                       // f16's exponent bias
}

// x / d with the code decided: the corrected quotient, off a border that it does not truly meet. `wide`: x may have more bits
// than a border times d (f32 values, or ones computed here); 16-bit values are either on it or 2^-12 away.
__device__ __forceinline__ float ratio(float x, float d, float inv, bool wide) {
    float t = __fmul_rn(x, inv);
    t = __fmaf_rn(__fmaf_rn(-t, d, x), inv, t);
    if (wide) {
        const float rest = __fmaf_rn(-t, d, x);                   // exact: the true quotient lies on its side of t
        const uint32_t u = __float_as_uint(t);
        if (rest != 0.f && !(u & 1)) t = __uint_as_float((rest > 0.f) == (t > 0.f) ? u + 1 : u - 1);   // borders are even
    }
    return t;
}
__device__ __forceinline__ uint32_t codes2(float a, float b) {    // a in the low half
    uint32_t r;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tmov.b32 %0, {t, 0, 0, 0};\n\t}" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// max of |a|, |b| that keeps a NaN
__device__ __forceinline__ float max_abs(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}

// Where the rows of a call lie. Row t: the sequence whose rows hold it, or -1.
struct Rows {
    int row0[MAX_SEQ + 1], len[MAX_SEQ];
    __device__ __forceinline__ void load(const Batch &b, int tid, int threads) {
        for (int s = tid; s <= b.nseq; s += threads) {
            row0[s] = __ldg(b.row0 + s);
            if (s < b.nseq) len[s] = __ldg(b.kv_len + s);
        }
    }
    // the row's place in the pool for KV head 0 and its position; false: it belongs to nobody, or the batch does not fit
    __device__ __forceinline__ bool find(const Pool &p, const Batch &b, int t, size_t &at, int &pos, int *err) const {
        int lo = 0, hi = b.nseq;          // the last sequence that starts at or before t
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (row0[mid] <= t) lo = mid;
            else hi = mid;
        }
        const int r0 = row0[lo], r1 = row0[lo + 1];
        if (t < r0 || t >= r1) return false;
        pos = len[lo] - (r1 - t);
        int page = -1;
        if (r0 >= 0 && r1 <= b.rows && len[lo] >= r1 - r0 && pos / p.page_tokens < b.max_pages)
            page = __ldg(b.table + (size_t)lo * b.max_pages + pos / p.page_tokens);
        if (page < 0 || page >= p.pages) {
            if (err) atomicExch(err, DEV_BAD_INDEX);
            return false;
        }
        at = row_index(p, page, 0, pos % p.page_tokens);
        return true;
    }
};

template <typename T, int HD>
__global__ void __launch_bounds__(AP_THREADS) append_kernel(const AppendArgs a) {
    constexpr int LPR = HD / 8, GH = 256 / HD;                     // lanes of a head, heads of a warp
    __shared__ Rows rows;
    __shared__ size_t at_s[MAX_TILE];                              // a token's place, position (-1: none)
    __shared__ int pos_s[MAX_TILE];
    extern __shared__ __align__(16) float turn[];                  // [tile][pdim / 2] cosines, then sines
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane / LPR, u = lane % LPR;
    const int all = a.heads + 2 * a.pool.kv_heads, per = (all + GH - 1) / GH, half = a.pdim / 2, tile = a.tile;
    float *cs = turn, *sn = turn + tile * half;
    pdl_trigger();
    pdl_wait();
    rows.load(a.b, tid, AP_THREADS);
    __syncthreads();
    const int tiles = (a.b.rows + tile - 1) / tile;
    for (int tl = blockIdx.x; tl < tiles; tl += gridDim.x) {
        const int t0 = tl * tile, nt = min(tile, a.b.rows - t0);
        if (tid < nt) {
            size_t at = 0;
            int pos = 0;
            pos_s[tid] = rows.find(a.pool, a.b, t0 + tid, at, pos, a.err) ? pos : -1;
            at_s[tid] = at;
        }
        __syncthreads();
        for (int i = tid; i < nt * half; i += AP_THREADS) {
            const int r = i / half, j = i - r * half;
            paged::angle(pos_s[r], __ldg(a.freq + j), cs[i], sn[i]);
        }
        if (half) __syncthreads();
        for (int it = warp; it < nt * per; it += AP_WARPS) {
            const int r = it / per, head = (it - r * per) * GH + sub;
            const bool live = head < all && pos_s[r] >= 0;
            const int kind = head < a.heads ? 0 : head < a.heads + a.pool.kv_heads ? 1 : 2;   // q, k, v
            const int h = kind == 0 ? head : kind == 1 ? head - a.heads : head - a.heads - a.pool.kv_heads;
            const T *src = (const T *)(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                           (long long)(t0 + r) * (kind == 0 ? a.ldq : kind == 1 ? a.ldk : a.ldv) + (long long)h * HD + 8 * u;
            float x[8];
            if (live) load8<T>(src, a.vec >> (kind == 0 ? 0 : kind + 1) & 1, x);
            else {
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = 0.f;
            }
            const float *w = kind == 0 ? a.qw : kind == 1 ? a.kw : nullptr;
            if (__any_sync(0xffffffffu, w != nullptr)) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (w) {
                    const float rs = __frsqrt_rn(fmaf(ss, 1.0f / HD, a.eps));
                    const float4 w0 = __ldg(reinterpret_cast<const float4 *>(w + 8 * u)), w1 = __ldg(reinterpret_cast<const float4 *>(w + 8 * u) + 1);
                    const float ww[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = x[i] * rs * ww[i];
                }
            }
            if (half) {
                const bool turned = kind < 2 && 8 * u < a.pdim;
                const float *c = cs + r * half, *s = sn + r * half;
                if (a.interleaved) {
                    if (turned) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float cc = c[4 * u + i], ss = s[4 * u + i], p = x[2 * i], q = x[2 * i + 1];
                            x[2 * i] = p * cc - q * ss;
                            x[2 * i + 1] = q * cc + p * ss;
                        }
                    }
                } else {
                    const bool low = 8 * u < half;
                    const int other = lane + (low ? half / 8 : -(half / 8)), j = low ? 8 * u : 8 * u - half;
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) y[i] = __shfl_sync(0xffffffffu, x[i], turned ? other : lane);
                    if (turned) {
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float cc = c[j + i], ss = s[j + i];
                            x[i] = low ? x[i] * cc - y[i] * ss : x[i] * cc + y[i] * ss;
                        }
                    }
                }
            }
            if (live && kind == 0)
                store8<T>((T *)a.q_out + (long long)(t0 + r) * a.ldqo + (long long)h * HD + 8 * u, a.vec >> 1 & 1, x);
            if (__any_sync(0xffffffffu, kind > 0)) {
                float mx = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) mx = max_abs(mx, x[i]);
                mx = max_abs(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                float d;
                const uint32_t b = scale_of(mx, d);
                const float inv = d > 0.f ? __fdiv_rn(1.0f, d) : 0.f;
                const bool wide = sizeof(T) == 4 || (kind == 1 && (a.kw || half));
                uint32_t code = 0;
#pragma unroll
                for (int i = 0; i < 8; i += 2)
                    code |= codes2(ratio(x[i], d, inv, wide), ratio(x[i + 1], d, inv, wide)) << (4 * i);
                if (!(d > 0.f)) code = 0;
                if (live && kind > 0) {
                    const size_t at = at_s[r] + (size_t)h * a.pool.page_tokens;
                    reinterpret_cast<uint32_t *>((kind == 1 ? a.pool.k : a.pool.v) + at * (HD / 2))[u] = code;
                    if (!(u & 1)) ((kind == 1 ? a.pool.ks : a.pool.vs) + at * (HD / GROUP))[u >> 1] = (uint8_t)b;
                }
            }
        }
        __syncthreads();   // the tile's places and angles are free
    }
}

template <typename T>
cudaError_t launch(const AppendArgs &a, cudaStream_t s) {
    const int hd = a.pool.hd, per = (a.heads + 2 * a.pool.kv_heads + 256 / hd - 1) / (256 / hd);
    AppendArgs p = a;
    p.tile = min(MAX_TILE, max(1, 2 * AP_WARPS / per));
    const int tiles = (a.b.rows + p.tile - 1) / p.tile;
    const size_t smem = (size_t)p.tile * a.pdim * sizeof(float);
    auto k = hd == 256 ? append_kernel<T, 256> : hd == 128 ? append_kernel<T, 128> : append_kernel<T, 64>;
    return launch_pdl(k, dim3(min(tiles, 4 * sm_count())), dim3(AP_THREADS), smem, s, p);
}

// ------------------------------------------------------------------ cached rows back
struct ReadArgs {
    Pool pool;
    Batch b;
    void *out[2];                          // rows of values, or of codes
    void *sc[2];                           // scales of codes
    long long ld[2], lds[2];
    int vec;                               // 16-byte pieces: bit 0 k, 1 v
    int *err;
};
struct Codes {};                           // e4m3 codes and f16 scales, apart

constexpr int RD_THREADS = 256;

// e4m3 bytes of four codes
__device__ __forceinline__ uint32_t code_bytes(uint32_t four) {
    const uint32_t mag = __byte_perm(0x3c383000u, 0x4c484440u, four & 0x7777u);
    const uint32_t sign = (four & 0x8u) << 4 | (four & 0x80u) << 8 | (four & 0x800u) << 12 | (four & 0x8000u) << 16;
    return mag | sign;
}

template <typename T, int HD>
__global__ void __launch_bounds__(RD_THREADS) read_kernel(const ReadArgs a) {
    constexpr int WORDS = HD / 8;                                  // of 8 codes
    __shared__ Rows rows;
    pdl_trigger();
    pdl_wait();
    rows.load(a.b, threadIdx.x, RD_THREADS);
    __syncthreads();
    const int side = blockIdx.y, hw = a.pool.kv_heads * WORDS;
    const uint8_t *pool = side ? a.pool.v : a.pool.k, *scales = side ? a.pool.vs : a.pool.ks;
    if (!a.out[side]) return;
    for (long long i = (long long)blockIdx.x * RD_THREADS + threadIdx.x; i < (long long)a.b.rows * hw; i += (long long)gridDim.x * RD_THREADS) {
        const int t = (int)(i / hw), x = (int)(i - (long long)t * hw), h = x / WORDS, u = x % WORDS;
        size_t at;
        int pos;
        if (!rows.find(a.pool, a.b, t, at, pos, a.err)) continue;
        at += (size_t)h * a.pool.page_tokens;
        const uint32_t w = __ldg(reinterpret_cast<const uint32_t *>(pool + at * (HD / 2)) + u);
        const uint32_t sb = (uint32_t)__ldg(scales + at * (HD / GROUP) + (u >> 1)) << 7;
        const long long to = (long long)t * a.ld[side] + (long long)h * HD + 8 * u;
        if constexpr (__is_same(T, Codes)) {
            uint8_t *p = (uint8_t *)a.out[side] + to;
            const uint32_t lo = code_bytes(w & 0xffffu), hi = code_bytes(w >> 16);
            if (a.vec >> side & 1) *reinterpret_cast<uint2 *>(p) = make_uint2(lo, hi);
            else {
#pragma unroll
                for (int e = 0; e < 8; e++) p[e] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
            }
            if (!(u & 1)) ((uint16_t *)a.sc[side])[(long long)t * a.lds[side] + h * (HD / GROUP) + (u >> 1)] = (uint16_t)sb;
        } else {
            uint32_t c[4];
            codes_f16(w, c);
            const uint32_t ss = sb | sb << 16;
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 f = __half22float2(__hmul2(*reinterpret_cast<const __half2 *>(&c[e]), *reinterpret_cast<const __half2 *>(&ss)));
                v[2 * e] = f.x, v[2 * e + 1] = f.y;
            }
            store8<T>((T *)a.out[side] + to, a.vec >> side & 1, v);
        }
    }
}

template <typename T>
cudaError_t launch_read(const ReadArgs &a, cudaStream_t s) {
    const int hd = a.pool.hd;
    const long long items = (long long)a.b.rows * a.pool.kv_heads * (hd / 8);
    auto k = hd == 256 ? read_kernel<T, 256> : hd == 128 ? read_kernel<T, 128> : read_kernel<T, 64>;
    const long long ctas = (items + RD_THREADS - 1) / RD_THREADS;
    return launch_pdl(k, dim3((unsigned)min(ctas, 8ll * sm_count()), 2), dim3(RD_THREADS), 0, s, a);
}

}  // namespace
}  // namespace paged4
}  // namespace spk

extern "C" {

int spk_paged4_append(const spk_kv4_pool *pool, const spk_kv_batch *batch, const spk_paged4_append_args *p, void *stream) {
    using namespace spk;
    using namespace spk::paged4;
    const char *who = "spk_paged4_append";
    if (check_pool(pool, who) || paged::check_batch(batch, who)) return -1;
    if (!p) return set_error("%s: null arguments", who);
    if (p->type < T_F32 || p->type > T_BF16) return set_error("%s: type %d (0 f32, 1 f16, 2 bf16)", who, p->type);
    if (p->heads < 0 || p->heads > 65536 || pool->kv_heads > 65536) return set_error("%s: %d heads, %d KV heads", who, p->heads, pool->kv_heads);
    if (p->pdim < 0 || p->pdim % 16 || p->pdim > pool->head_dim || (p->pdim > 0 && !p->freq) || (uintptr_t)p->freq % 4)
        return set_error("%s: pdim %d (a multiple of 16 up to head_dim, with its frequencies)", who, p->pdim);
    if ((uintptr_t)p->q_norm % 16 || (uintptr_t)p->k_norm % 16) return set_error("%s: norm weights are not 16-byte aligned", who);
    if ((p->q_norm || p->k_norm) && !(p->eps >= 0.f)) return set_error("%s: eps %g", who, p->eps);
    if (batch->rows == 0) return 0;
    if (!p->k || !p->v || (p->heads && (!p->q || !p->q_out))) return set_error("%s: null rows", who);
    const long long width = (long long)pool->kv_heads * pool->head_dim, qwidth = (long long)p->heads * pool->head_dim;
    if (batch->rows > 1 && (p->ldk < width || p->ldv < width || (p->heads && (p->ldq < qwidth || p->ldq_out < qwidth))))
        return set_error("%s: row strides %lld, %lld, %lld, %lld under %lld and %lld", who, p->ldq, p->ldq_out, p->ldk, p->ldv, qwidth, width);
    const int size = p->type == T_F32 ? 4 : 2;
    if (((uintptr_t)p->q | (uintptr_t)p->q_out | (uintptr_t)p->k | (uintptr_t)p->v) % size) return set_error("%s: unaligned rows", who);
    auto whole = [&](const void *at, long long ld) { return (uintptr_t)at % 16 == 0 && ld * size % 16 == 0 ? 1 : 0; };
    AppendArgs a{pool_of(pool), paged::batch_of(batch), p->q, p->k, p->v, p->q_out, p->ldq, p->ldq_out, p->ldk, p->ldv,
                 whole(p->q, p->ldq) | whole(p->q_out, p->ldq_out) << 1 | whole(p->k, p->ldk) << 2 | whole(p->v, p->ldv) << 3,
                 p->q_norm, p->k_norm, p->freq, p->heads, p->freq ? p->pdim : 0, p->interleaved ? 1 : 0, 1, p->eps, device_error_ptr()};
    const cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t e = p->type == T_F32 ? launch<float>(a, s) : p->type == T_F16 ? launch<__half>(a, s) : launch<__nv_bfloat16>(a, s);
    return e == cudaSuccess ? 0 : cuda_fail(who, e);
}

int spk_paged4_read(const spk_kv4_pool *pool, const spk_kv_batch *batch, const spk_paged4_read_args *p, void *stream) {
    using namespace spk;
    using namespace spk::paged4;
    const char *who = "spk_paged4_read";
    if (check_pool(pool, who) || paged::check_batch(batch, who)) return -1;
    if (!p) return set_error("%s: null arguments", who);
    const bool parts = p->type == SPK_PAGED4_PARTS;
    if (!parts && (p->type < T_F32 || p->type > T_BF16)) return set_error("%s: type %d (0 f32, 1 f16, 2 bf16, 3 codes and scales)", who, p->type);
    if (batch->rows == 0) return 0;
    if (!p->k && !p->v) return set_error("%s: null rows", who);
    const long long width = (long long)pool->kv_heads * pool->head_dim, swidth = width / GROUP;
    const int size = parts ? 1 : p->type == T_F32 ? 4 : 2;
    ReadArgs a{pool_of(pool), paged::batch_of(batch), {p->k, p->v}, {p->k_scale, p->v_scale}, {p->ldk, p->ldv}, {p->ldk_scale, p->ldv_scale}, 0, device_error_ptr()};
    for (int i = 0; i < 2; i++) {
        if (!a.out[i]) continue;
        if (parts && (!a.sc[i] || (uintptr_t)a.sc[i] % 2)) return set_error("%s: scales are null or unaligned", who);
        if (batch->rows > 1 && (a.ld[i] < width || (parts && a.lds[i] < swidth)))
            return set_error("%s: row strides %lld, %lld under %lld, %lld", who, a.ld[i], a.lds[i], width, swidth);
        if ((uintptr_t)a.out[i] % size) return set_error("%s: unaligned rows", who);
        const int piece = parts ? 8 : 16;
        if ((uintptr_t)a.out[i] % piece == 0 && a.ld[i] * size % piece == 0) a.vec |= 1 << i;
    }
    const cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t e = parts ? launch_read<Codes>(a, s) : p->type == T_F32 ? launch_read<float>(a, s) : p->type == T_F16 ? launch_read<__half>(a, s) : launch_read<__nv_bfloat16>(a, s);
    return e == cudaSuccess ? 0 : cuda_fail(who, e);
}

}  // extern "C"
