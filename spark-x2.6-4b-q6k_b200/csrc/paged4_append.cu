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
// What bounds append: at the rows' bytes' rate the issue slots are half used (50 M warp instructions for 16384 rows of 24 heads, 128 for 256 values) and
// a warp's chain (load, norm's tree of shuffles, rotation, scale, codes) waits for itself more often than for memory. A warp takes 256 values at a time (256 /
// head_dim heads side by side), 8 consecutive ones a lane, which is one 16-byte load of 16-bit rows and one word of codes; a group is two lanes, a head's norm
// a shuffle tree, the other half of a rotated pair 8 shuffles. A token's items (queries, keys, values) are one warp's where there are
// many tokens, so that it looks its place up and computes its angles once, and several warps' where there are few; the norms' weights stay in
// registers, four items' rows are loaded before the first one's work. No warp waits for another. One token takes as long as its launch.
#include <type_traits>

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

// Warps of an SM against registers a thread, and items whose loads go out and whose chains run together. 16384 bf16 rows (16 + 4 + 4 heads of
// 256, normalised, rotated over 64 dims) take 95 us, 3.7 TB/s of rows, queries and cache, 57 % of the measured copy rate. With the read of codes and
// scales behind it, 123 us now, these were chosen at 122: 128 with one CTA less, 123 with one more, 139 with two items together, 128 with twice the
// warps in a CTA; 13 f32 prompts of up to 1501 rows, 47 now, at 49: 59 with three CTAs, 57 with five. Rows through a ring of cp.async copies, more of them on their way, took 129 to 145
// and 67: what it adds per item, in f32 two passes over each sector, costs more than the wait that it hides.
constexpr int AP_WARPS = 4, AP_THREADS = AP_WARPS * 32;
template <typename T>
constexpr int AP_CTAS = sizeof(T) == 4 ? 4 : 5;                 // of an SM
template <typename T>
constexpr int AP_BATCH = 4;   // items

struct AppendArgs {
    Pool pool;
    Batch b;
    const void *q, *k, *v;
    void *q_out;
    long long ldq, ldqo, ldk, ldv;
    int vec;                               // 16-byte pieces: bit 0 q, 1 q_out, 2 k, 3 v
    const float *qw, *kw, *freq;
    int heads, pdim, interleaved;          // q heads (0: none), rotated dims
    float eps;
    int *err;
};

// 8 values of a row as they lie in memory
template <typename T>
struct Raw8 {
    uint32_t w[2 * sizeof(T)];
    __device__ __forceinline__ void load(const T *p, bool vec) {
        if (vec) {
            const uint4 a = *reinterpret_cast<const uint4 *>(p);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
            if constexpr (sizeof(T) == 4) {
                const uint4 b = *(reinterpret_cast<const uint4 *>(p) + 1);
                w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < (int)(2 * sizeof(T)); i++) {
                if constexpr (sizeof(T) == 4) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
                else w[i] = reinterpret_cast<const uint16_t *>(p)[2 * i] | (uint32_t)reinterpret_cast<const uint16_t *>(p)[2 * i + 1] << 16;
            }
        }
    }
    __device__ __forceinline__ void none() {
#pragma unroll
        for (int i = 0; i < (int)(2 * sizeof(T)); i++) w[i] = 0;
    }
    __device__ __forceinline__ void f32(paged::f32x2 (&x)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4) x[i] = paged::pack2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
            else if constexpr (__is_same(T, __half)) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                x[i] = paged::pack2(f.x, f.y);
            } else {
                x[i] = paged::pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            }
        }
    }
};
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
__device__ __forceinline__ void store8(T *p, bool vec, const paged::f32x2 (&v)[4]) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = paged::unpack2(v[i]);
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
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
    const float t = fminf(fmaxf(amax * (1.0f / 6.0f), SCALE_MIN), SCALE_MAX);
    uint32_t b = __float_as_uint(t) >> 20;                        // the 4 leading bits, or of the number a unit beside
    const float six = 6.0f * __uint_as_float((b << 20) | 0x80000u);   // six times the middle to the next: 8 bits, exact
    if (t < SCALE_MAX && (amax > six || (amax == six && (b & 1)))) b++;
    const bool number = amax < INFINITY;
    d = number ? __uint_as_float(b << 20) : 0.f;
    return number ? b - (112u << 3) : 0xffu;                      // f16's exponent bias
}

// The codes of 8 values under d (0: none). A corrected quotient is the nearest f32 to x / d: a tie is a tie. `wide`: x may have more bits
// than a border times d (f32 values, or ones computed here; 16-bit values are on a border or 2^-12 away), so a quotient that was rounded to
// a border (all of them have 21 zeros at the end) is moved off it, to the side that its residual, which is exact, says.
template <bool WIDE>
__device__ __forceinline__ uint32_t codes8(const paged::f32x2 (&x)[4], float d) {
    using namespace paged;
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(d));
    const f32x2 i2 = pack2(inv, inv), nd = pack2(-d, -d);
    float t[8];
    uint32_t low = ~0u;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const f32x2 q = mul2(x[e / 2], i2);
        const float2 r = unpack2(fma2(fma2(q, nd, x[e / 2]), i2, q));
        t[e] = r.x, t[e + 1] = r.y;
        if (WIDE) low = min(low, min(__float_as_uint(r.x) & 0x1fffffu, __float_as_uint(r.y) & 0x1fffffu));
    }
    if (WIDE && low == 0) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float2 xe = unpack2(x[e / 2]);
            const float rest = __fmaf_rn(-t[e], d, e & 1 ? xe.y : xe.x);
            const uint32_t u = __float_as_uint(t[e]);
            if (rest != 0.f && t[e] != 0.f && !(u & 0x1fffffu)) t[e] = __uint_as_float((rest > 0.f) == (t[e] > 0.f) ? u + 1 : u - 1);
        }
    }
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(t[0]), "f"(t[1]), "f"(t[2]), "f"(t[3]), "f"(t[4]), "f"(t[5]), "f"(t[6]), "f"(t[7]));
    return d > 0.f ? r : 0u;
}

// max of m, |a|, |b| that keeps a NaN
__device__ __forceinline__ float max_abs(float m, float a, float b) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(a), "f"(b));
    return r;
}

// A head's mean square and eps between these: no square that counts in it was lost, none was infinite. Where it is not (values beyond 2^60, or all under
// 2^-45 with as small an eps) the head is squared again on a power of two: up to 2^58 from 2^128, up from 2^-149 to 2^-49.
// The test between a sum and its root costs 3 % of a prompt's append (16384 bf16 rows with their reading back 122 us without it, 126 so; 129 with such heads done
// again behind a batch of items, 139 with one test for a batch); 123 since each kind of pairs has its own code.
constexpr float NORM_LOW = 0x1p-90f, NORM_HIGH = 0x1p120f, NORM_UP = 0x1p100f, NORM_DOWN = 0x1p-70f;

// Where the rows of a call lie: the sequences in shared memory.
struct Rows {
    int row0[MAX_SEQ + 1], len[MAX_SEQ];
    __device__ __forceinline__ void load(const Batch &b, int tid, int threads) {
        for (int s = tid; s <= b.nseq; s += threads) {
            row0[s] = __ldg(b.row0 + s);
            if (s < b.nseq) len[s] = __ldg(b.kv_len + s);
        }
        __syncthreads();
    }
    // row t's place in the pool for KV head 0, and its position; -1: it belongs to nobody, or the batch does not fit
    __device__ __forceinline__ long long find(const Pool &p, const Batch &b, int t, int &pos, int *err) const {
        int lo = 0, hi = b.nseq;          // the last sequence that starts at or before t
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (row0[mid] <= t) lo = mid;
            else hi = mid;
        }
        const int r0 = row0[lo], r1 = row0[lo + 1];
        if (t >= b.rows || t < r0 || t >= r1) return -1;
        pos = len[lo] - (r1 - t);
        int page = -1;
        if (r0 >= 0 && r1 <= b.rows && len[lo] >= r1 - r0 && pos / p.page_tokens < b.max_pages)
            page = __ldg(b.table + (size_t)lo * b.max_pages + pos / p.page_tokens);
        if (page < 0 || page >= p.pages) {
            if (err) atomicExch(err, DEV_BAD_INDEX);
            return -1;
        }
        return (long long)row_index(p, page, 0, pos % p.page_tokens);
    }
};

// The work of a call: a token's `per` items of 256 values belong to a team of `team` warps, which takes every `teams`-th token.
struct Share {
    int first, x0, team, teams;
    __device__ __forceinline__ Share(int rows, int per) {
        const long long warps = (long long)gridDim.x * (blockDim.x / 32), w = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
        team = (int)max(1ll, min((long long)per, warps / rows));
        teams = (int)(warps / team);
        first = w / team < teams ? (int)(w / team) : rows;
        x0 = (int)(w % team);
    }
};
// CTAs of a call
int ctas_of(long long rows, int per, int warps, int most) {
    return (int)max(1ll, min((long long)most, (rows * per + warps - 1) / warps));
}

__device__ __noinline__ float2 turn_of(int pos, float freq) {
    float2 t;
    paged::angle(pos, freq, t.x, t.y);
    return t;
}

template <typename T, int HD, bool VEC, bool SWAP>   // SWAP: pairs side by side
__global__ void __launch_bounds__(AP_THREADS, AP_CTAS<T>) append_kernel(const AppendArgs a) {
    using namespace paged;
    constexpr int LPR = HD / 8, GH = 256 / HD, BATCH = AP_BATCH<T>;   // lanes of a head, heads of a warp
    __shared__ Rows rows;
    const int lane = threadIdx.x & 31, sub = lane / LPR, u = lane % LPR;
    const int kv = a.pool.kv_heads, pq = (a.heads + GH - 1) / GH, pk = (kv + GH - 1) / GH, per = pq + 2 * pk;   // a token's items: queries, keys, values
    const int half = a.pdim / 2;
    const bool turned = 8 * u < a.pdim;
    // the lane that has the other halves of this one's pairs; the first of the 4 angles that this one works out
    const bool low = 8 * u < half;
    const int other = SWAP || !turned ? lane : low ? lane + half / 8 : lane - half / 8, angle0 = SWAP ? 4 * u : low ? 8 * u : 8 * u - half + 4;
    pdl_trigger();
    pdl_wait();
    rows.load(a.b, threadIdx.x, AP_THREADS);
    const Share sh(a.b.rows, per);

    auto weights = [&](const float *w, f32x2 (&to)[4]) {
        if (!w) return;
        const float4 w0 = __ldg(reinterpret_cast<const float4 *>(w + 8 * u)), w1 = __ldg(reinterpret_cast<const float4 *>(w + 8 * u) + 1);
        to[0] = pack2(w0.x, w0.y), to[1] = pack2(w0.z, w0.w), to[2] = pack2(w1.x, w1.y), to[3] = pack2(w1.z, w1.w);
    };
    f32x2 qw[4], kw[4];
    weights(a.qw, qw);
    weights(a.kw, kw);
    auto norm = [&](f32x2 (&x)[4], const f32x2 (&w)[4]) {
        auto mean = [&](float eps, uint32_t lanes) {
            f32x2 s2 = mul2(x[0], x[0]);
#pragma unroll
            for (int e = 1; e < 4; e++) s2 = fma2(x[e], x[e], s2);
            const float2 ab = unpack2(s2);
            float ss = ab.x + ab.y;
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(lanes, ss, o);
            return fmaf(ss, 1.0f / HD, eps);
        };
        float ms = mean(a.eps, 0xffffffffu);
        if (!__is_same(T, __half) && !(ms > NORM_LOW && ms < NORM_HIGH)) {   // f16's squares are from 2^-48 to 2^32
            const float k = ms <= NORM_LOW ? NORM_UP : NORM_DOWN;
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = mul2(x[e], pack2(k, k));
            ms = mean(a.eps * k * k, LPR == 32 ? 0xffffffffu : ((1u << (LPR & 31)) - 1) << (sub * LPR));   // the head's lanes, which are all here
        }
        const float rs = rsqrtf(ms);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = mul2(mul2(x[e], pack2(rs, rs)), w[e]);
    };
    // The token's factors of a dim and of its pair's other dim. Where nothing is rotated they are halves of the dim itself: x / 2 + x / 2 is x, an infinity and a
    // zero of either sign among them (f32 numbers under 2^-125 to 2^-149), where a factor of 0 made infinities no numbers. Chosen between behind the
    // sum, a prompt's append takes 127 us for 124.
    f32x2 cs[4], sn[4];
    auto angles = [&](int pos) {
        float c[4], s[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float2 t = turned ? turn_of(pos, __ldg(a.freq + angle0 + e)) : make_float2(0.5f, 0.5f);
            c[e] = t.x, s[e] = t.y;
        }
        if (SWAP) {
#pragma unroll
            for (int e = 0; e < 4; e++) cs[e] = pack2(c[e], c[e]), sn[e] = pack2(turned ? -s[e] : s[e], s[e]);
        } else {   // low lanes worked out the first 4 of their 8 angles, the others the last 4
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float oc0 = __shfl_sync(0xffffffffu, c[e], other), oc1 = __shfl_sync(0xffffffffu, c[e + 1], other);
                const float os0 = __shfl_sync(0xffffffffu, s[e], other), os1 = __shfl_sync(0xffffffffu, s[e + 1], other);
                cs[e / 2] = low ? pack2(c[e], c[e + 1]) : pack2(oc0, oc1);
                cs[2 + e / 2] = low ? pack2(oc0, oc1) : pack2(c[e], c[e + 1]);
                sn[e / 2] = low ? pack2(-s[e], -s[e + 1]) : pack2(os0, os1);
                sn[2 + e / 2] = low ? pack2(-os0, -os1) : pack2(s[e], s[e + 1]);
            }
        }
    };
    auto rotate = [&](f32x2 (&x)[4]) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float2 v = unpack2(x[e]);
            const f32x2 y = SWAP ? (turned ? pack2(v.y, v.x) : x[e]) : pack2(__shfl_sync(0xffffffffu, v.x, other), __shfl_sync(0xffffffffu, v.y, other));
            x[e] = fma2(y, sn[e], mul2(x[e], cs[e]));
        }
    };
    // A warp has every team-th of a token's items, queries, keys and values counted on. `items` of a row, `before` them
    // those of the others: heads of 256 values side by side, a batch's loads before its work.
    auto first_of = [&](int before) {
        const int x = (sh.x0 - before) % sh.team;
        return x < 0 ? x + sh.team : x;
    };
    auto row = [&](const T *src, int before, int items, int heads, auto &&work) {
        for (int x = first_of(before); x < items; x += BATCH * sh.team) {
            Raw8<T> raw[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const int xi = x + i * sh.team;
                if (xi < items && (GH == 1 || xi * GH + sub < heads)) raw[i].load(src + xi * 256, VEC);
                else raw[i].none();
            }
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const int xi = x + i * sh.team;
                if (xi >= items) break;
                f32x2 v[4];
                raw[i].f32(v);
                work(v, xi * GH + sub, GH == 1 || xi * GH + sub < heads);
            }
        }
    };

    long long places = -1;              // lane i: place and position of the team's i-th token from `count` & ~31 on
    int poses = 0, count = 0;
    for (int t = sh.first; t < a.b.rows; t += sh.teams, count++) {
        if (!(count & 31)) {
            const long long tt = (long long)t + (long long)lane * sh.teams;
            places = tt < a.b.rows ? rows.find(a.pool, a.b, (int)tt, poses, a.err) : -1;
        }
        const long long at = __shfl_sync(0xffffffffu, places, count & 31);
        const int pos = __shfl_sync(0xffffffffu, poses, count & 31);
        if (at < 0) continue;
        if (half) angles(pos);
        T *qo = (T *)a.q_out + (long long)t * a.ldqo + 8 * u;
        row((const T *)a.q + (long long)t * a.ldq + lane * 8, 0, pq, a.heads, [&](f32x2 (&v)[4], int h, bool live) {
            if (a.qw) norm(v, qw);
            if (half) rotate(v);
            if (live) store8<T>(qo + h * HD, VEC, v);
        });
        auto keep = [&](uint8_t *codes, uint8_t *scales, const f32x2 (&v)[4], int h, bool live, bool wide) {
            float mx = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 f = unpack2(v[e]);
                mx = max_abs(mx, f.x, f.y);
            }
            mx = max_abs(mx, __shfl_xor_sync(0xffffffffu, mx, 1), 0.f);
            float d;
            const uint32_t b = scale_of(mx, d), code = wide ? codes8<true>(v, d) : codes8<false>(v, d);
            if (live) {
                const size_t to = (size_t)at + (size_t)h * a.pool.page_tokens;
                reinterpret_cast<uint32_t *>(codes + to * (HD / 2))[u] = code;
                if (!(u & 1)) (scales + to * (HD / GROUP))[u >> 1] = (uint8_t)b;
            }
        };
        row((const T *)a.k + (long long)t * a.ldk + lane * 8, pq, pk, kv, [&](f32x2 (&v)[4], int h, bool live) {
            if (a.kw) norm(v, kw);
            if (half) rotate(v);
            keep(a.pool.k, a.pool.ks, v, h, live, sizeof(T) == 4 || a.kw || half);
        });
        row((const T *)a.v + (long long)t * a.ldv + lane * 8, pq + pk, pk, kv,
            [&](f32x2 (&v)[4], int h, bool live) { keep(a.pool.v, a.pool.vs, v, h, live, sizeof(T) == 4); });
    }
}

template <typename T>
cudaError_t launch(const AppendArgs &a, cudaStream_t s) {
    const int hd = a.pool.hd, gh = 256 / hd, per = (a.heads + gh - 1) / gh + 2 * ((a.pool.kv_heads + gh - 1) / gh);
    auto of = [&](auto vec, auto swap) {
        constexpr bool V = decltype(vec)::value, S = decltype(swap)::value;
        return hd == 256 ? append_kernel<T, 256, V, S> : hd == 128 ? append_kernel<T, 128, V, S> : append_kernel<T, 64, V, S>;
    };
    using Yes = std::true_type;
    using No = std::false_type;
    auto k = a.vec == 15 ? (a.interleaved ? of(Yes(), Yes()) : of(Yes(), No())) : (a.interleaved ? of(No(), Yes()) : of(No(), No()));
    return launch_pdl(k, dim3(ctas_of(a.b.rows, per, AP_WARPS, AP_CTAS<T> * sm_count())), dim3(AP_THREADS), 0, s, a);
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
template <typename T>
struct Out {
    using type = T;
};
template <>
struct Out<Codes> {
    using type = uint8_t;
};

// Read is bound by issue slots (70 % used; a lane's 8 values take some 35 instructions) and needs warps to hide the lookups of places. 40 MB of
// bf16 rows from 11 MB of cache take 16.7 us with 12 CTAs of an SM and two items' loads together, 48 % of the measured copy rate; 17.4 with four
// items, 17.6 with 16 CTAs, 20.0 with 8. Codes and scales apart take fewer instructions: append and read of 13 f32 prompts 47.4 us with 16
// CTAs, 49.6 with 12.
constexpr int RD_THREADS = 128;
template <typename T>
constexpr int RD_CTAS = __is_same(T, Codes) ? 16 : 12;       // of an SM

// e4m3 bytes of four codes
__device__ __forceinline__ uint32_t code_bytes(uint32_t four) {
    const uint32_t mag = __byte_perm(0x3c383000u, 0x4c484440u, four & 0x7777u);
    const uint32_t sign = (four & 0x8u) << 4 | (four & 0x80u) << 8 | (four & 0x800u) << 12 | (four & 0x8000u) << 16;
    return mag | sign;
}

template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(RD_THREADS, RD_CTAS<T>) read_kernel(const ReadArgs a) {
    constexpr int LPR = HD / 8, GH = 256 / HD, BATCH = 2;          // lanes of a head, heads of a warp, items whose loads go out together
    constexpr bool APART = __is_same(T, Codes);
    using O = typename Out<T>::type;
    __shared__ Rows rows;
    const int lane = threadIdx.x & 31, sub = lane / LPR, u = lane % LPR;
    const int kv = a.pool.kv_heads, parts = (kv + GH - 1) / GH, per = 2 * parts;   // a token's items: keys, values
    const size_t step = (size_t)GH * a.pool.page_tokens, mine = (size_t)sub * a.pool.page_tokens;   // rows of the pool from item to item
    pdl_trigger();
    pdl_wait();
    rows.load(a.b, threadIdx.x, RD_THREADS);
    const Share sh(a.b.rows, per);
    long long places = -1;              // lane i: place of the team's i-th token from `count` & ~31 on
    int count = 0;
    for (int t = sh.first; t < a.b.rows; t += sh.teams, count++) {
        if (!(count & 31)) {
            const long long tt = (long long)t + (long long)lane * sh.teams;
            int pos;
            places = tt < a.b.rows ? rows.find(a.pool, a.b, (int)tt, pos, a.err) : -1;
        }
        const long long at = __shfl_sync(0xffffffffu, places, count & 31);
        if (at < 0) continue;
        const size_t row = (size_t)at + mine;
        const uint8_t *kc = a.pool.k + row * (HD / 2) + 4 * u, *vc = a.pool.v + row * (HD / 2) + 4 * u;
        const uint8_t *ks = a.pool.ks + row * (HD / GROUP) + (u >> 1), *vs = a.pool.vs + row * (HD / GROUP) + (u >> 1);
        O *ko = (O *)a.out[0] + (long long)t * a.ld[0] + lane * 8, *vo = (O *)a.out[1] + (long long)t * a.ld[1] + lane * 8;
        for (int x = sh.x0; x < per; x += BATCH * sh.team) {
            uint32_t w[BATCH], sb[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const int xi = x + i * sh.team, side = xi >= parts, it = side ? xi - parts : xi;
                w[i] = sb[i] = 0;
                if (xi < per && (GH == 1 || it * GH + sub < kv) && a.out[side]) {
                    w[i] = __ldg(reinterpret_cast<const uint32_t *>((side ? vc : kc) + it * step * (HD / 2)));
                    sb[i] = __ldg((side ? vs : ks) + it * step * (HD / GROUP));
                }
            }
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const int xi = x + i * sh.team, side = xi >= parts, it = side ? xi - parts : xi;
                if (xi >= per) break;
                if ((GH > 1 && it * GH + sub >= kv) || !a.out[side]) continue;
                O *to = (side ? vo : ko) + it * 256;
                if constexpr (APART) {
                    const uint32_t lo = code_bytes(w[i] & 0xffffu), hi = code_bytes(w[i] >> 16);
                    if (VEC) *reinterpret_cast<uint2 *>(to) = make_uint2(lo, hi);
                    else {
#pragma unroll
                        for (int e = 0; e < 8; e++) to[e] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
                    }
                    if (!(u & 1)) ((uint16_t *)a.sc[side])[(long long)t * a.lds[side] + (it * GH + sub) * (HD / GROUP) + (u >> 1)] = (uint16_t)(sb[i] << 7);
                } else {
                    uint32_t c[4];
                    codes_f16(w[i], c);
                    const uint32_t ss = sb[i] * 0x00800080u;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const __half2 h = __hmul2(*reinterpret_cast<const __half2 *>(&c[e]), *reinterpret_cast<const __half2 *>(&ss));
                        c[e] = *reinterpret_cast<const uint32_t *>(&h);
                    }
                    if constexpr (__is_same(T, __half)) {
                        if (VEC) *reinterpret_cast<uint4 *>(to) = make_uint4(c[0], c[1], c[2], c[3]);
                        else {
#pragma unroll
                            for (int e = 0; e < 8; e++) reinterpret_cast<uint16_t *>(to)[e] = (uint16_t)(c[e >> 1] >> (16 * (e & 1)));
                        }
                    } else {
                        paged::f32x2 v[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&c[e]));
                            v[e] = paged::pack2(f.x, f.y);
                        }
                        store8<T>(to, VEC, v);
                    }
                }
            }
        }
    }
}

template <typename T>
cudaError_t launch_read(const ReadArgs &a, cudaStream_t s) {
    const int hd = a.pool.hd, per = 2 * ((a.pool.kv_heads + 256 / hd - 1) / (256 / hd));
    auto k = a.vec == 3 ? (hd == 256 ? read_kernel<T, 256, true> : hd == 128 ? read_kernel<T, 128, true> : read_kernel<T, 64, true>)
                        : (hd == 256 ? read_kernel<T, 256, false> : hd == 128 ? read_kernel<T, 128, false> : read_kernel<T, 64, false>);
    return launch_pdl(k, dim3(ctas_of(a.b.rows, per, RD_THREADS / 32, RD_CTAS<T> * sm_count())), dim3(RD_THREADS), 0, s, a);
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
                 p->q_norm, p->k_norm, p->freq, p->heads, p->freq ? p->pdim : 0, p->interleaved ? 1 : 0, p->eps, device_error_ptr()};
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
        if (!a.out[i]) {
            a.vec |= 1 << i;
            continue;
        }
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
