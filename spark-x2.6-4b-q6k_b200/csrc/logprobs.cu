// logprobs.cu — what a row of logits says: the log probability of a given token, the entropy of the
// distribution and its best alternatives, in one read of the row.
//
//   m = max x,  S = sum e^(x - m),  A = sum (x - m) e^(x - m)
//   logp(i) = x_i - m - log S,   H = log S - A / S,   the top k by (x descending, index ascending)
//
// Every term of H is >= 0, so nothing cancels. -inf is a token that cannot come (0 to S and A); a
// row that holds a NaN or +inf, or only -inf, has no distribution: NaN for logp, H and the
// alternatives' values (their indices stay those of the order, a NaN ranking as -inf).
//
// What bounds it: the row's bytes, then the exponentials (16 a clock and SM: 30 us beside the 42 us that
// 1024 x 131072 bf16 values take to read; the unit is busy 56 % of the time, the issue slots 58 %). A CTA streams a range of a row, 16 bytes a load, four loads
// a thread in flight; each thread keeps its own (m, S, A) in base 2, pairs of values by one f32x2
// instruction, and moves m when a vector of values passes it. The best k (k <= 32) are a list over a
// warp's lanes, as 64-bit keys (order of the value, then of the index). A vector is looked at again only
// if its largest value reaches the best k-th value that the CTA has seen, which starts at the k-th
// largest of its lane maxima (one row of 131072, 20 alternatives: 8.7 us, and 13.2 when it starts at the
// best warp's k-th, which 20 of 32 lanes pass); lists join by half cleaners (5 exchanges). A row alone
// is cut over many CTAs (rows x splits fill the SMs); the last one to arrive, by a ticket that it
// resets, joins the parts.
//
// Measured: 1024 x 131072 bf16, 5 alternatives, 67 us (4.0 TB/s, 0.62 of a copy's rate; with 3 tokens left in each row 127,
// whole rows of the type's lowest value 175), f32 114 us; 61 x 50021 f16, 1 alternative, 8.9 us; 1 x 131072 f32, 20
// alternatives, 8.5 us, of which 1 us is the load, 3 the launch and the ticket, and the rest the lists: compare and
// exchange, one behind the other.
#include <cuda_bf16.h>

#include "common.cuh"
#include "spk.h"

namespace spk {
namespace {

constexpr int LP_TOP = 32;                 // the most alternatives
constexpr int LP_SPLITS = 64;              // the most CTAs of a row
constexpr int LP_PART = 4 + 2 * LP_TOP;    // floats of a part: m, S, A, then the keys
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float HUGE_M = 1e37f;            // references past it take the sums' slow form

struct LpArgs {
    const void *x;
    long long ld;
    int rows, vocab, top, splits;
    int chunk;                             // values of a split, a multiple of a tile
    const int *target;
    float *logp, *entropy;
    int *ids;
    float *best;
    unsigned int *tickets;                 // [rows that are split], zero at rest
    float *part;                           // [rows][splits][LP_PART]
    int *err;
};

__device__ __forceinline__ float ex2f_(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long pack2(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}

// (m, S, A) in base 2: t = (x - m) log2 e, S = sum 2^t, A = sum t 2^t
struct Stat {
    float m, s, a;
};
// moves st to the reference m (>= st.m, in the logits' unit)
__device__ __forceinline__ void move(Stat &st, float m) {
    if (st.m == m) return;   // both may be -inf
    const float d = (st.m - m) * LOG2E, f = ex2f_(d);
    st.a = f == 0.f ? 0.f : fmaf(d, st.s, st.a) * f;
    st.s *= f;
    st.m = m;
}
__device__ __forceinline__ Stat join(Stat p, Stat q) {
    const float m = fmaxf(p.m, q.m);
    move(p, m);
    move(q, m);
    return Stat{m, p.s + q.s, p.a + q.a};
}
__device__ __forceinline__ Stat warp_join(Stat st) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        st = join(st, Stat{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                           __shfl_xor_sync(0xffffffffu, st.a, o)});
    return st;
}

// Keys: larger is better; 0 is no token. The value's bits in order, then the index from the end.
typedef unsigned long long Key;
__device__ __forceinline__ uint32_t order_of(float x) {   // -0 as 0, NaN as -inf
    const uint32_t b = __float_as_uint(fmaxf(x, -INFINITY) + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(Key k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ Key key_of(float x, int i) { return ((Key)order_of(x) << 32) | (0xffffffffu - (uint32_t)i); }
__device__ __forceinline__ int index_of(Key k) { return (int)(0xffffffffu - (uint32_t)k); }

__device__ __forceinline__ Key exchange(Key k, int o, bool large) {
    const Key p = __shfl_xor_sync(0xffffffffu, k, o);
    return (k > p) == large ? k : p;
}
__device__ __forceinline__ Key clean(Key k, int lane) {   // a bitonic sequence, descending
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) k = exchange(k, o, !(lane & o));
    return k;
}
__device__ __forceinline__ float exchange(float k, int o, bool large) {
    const float p = __shfl_xor_sync(0xffffffffu, k, o);
    return large ? fmaxf(k, p) : fminf(k, p);
}
template <typename K>
__device__ __forceinline__ K sort32(K k, int lane) {   // descending
#pragma unroll
    for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
        for (int o = n >> 1; o > 0; o >>= 1) k = exchange(k, o, !(lane & o) == !(lane & n));
    return k;
}
// the best 32 of two descending lists; `rev`: the other one's key of lane 31 - lane
__device__ __forceinline__ Key merge(Key k, Key rev, int lane) { return clean(k > rev ? k : rev, lane); }

// Offers each lane's candidate (0: none) to the warp's list; kth: its last place that counts.
__device__ __forceinline__ void offer(Key &list, Key cand, int kth, int lane) {
    Key last = __shfl_sync(0xffffffffu, list, kth);
    unsigned left = __ballot_sync(0xffffffffu, cand > last);
    if (__popc(left) > 3) {
        cand = sort32(cand, lane);
        list = merge(list, __shfl_sync(0xffffffffu, cand, 31 - lane), lane);
        return;
    }
    while (left) {
        const Key c = __shfl_sync(0xffffffffu, cand, __ffs(left) - 1);
        const bool mine = c > list;
        const Key up = __shfl_up_sync(0xffffffffu, list, 1);
        const bool shift = lane > 0 && c > up;
        if (mine) list = shift ? up : c;
        left &= left - 1;
    }
}

template <typename T>
struct Vec {   // 16 bytes of T
    static constexpr int N = 16 / sizeof(T);
    // sums take the fast form for references above this: -inf ends as FLOOR, far below all of them
    static constexpr float LOW_M = __is_same(T, __half) ? -3e4f : -HUGE_M;
    static __device__ __forceinline__ float one(const T *p) {
        if constexpr (sizeof(T) == 4) return (float)*p;
        else if constexpr (__is_same(T, __half)) return __half2float(*p);
        else return __bfloat162float(*p);
    }
    static __device__ __forceinline__ float2 two(uint32_t u) {   // of 16-bit types
        if constexpr (__is_same(T, __half)) return __half22float2(*reinterpret_cast<const __half2 *>(&u));
        else return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t max_(uint32_t a, uint32_t b) {   // of a pair (or of one f32), NaN is less
        uint32_t r;
        if constexpr (sizeof(T) == 4) r = __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
        else if constexpr (__is_same(T, __half)) asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        else asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t floor_(uint32_t a) {   // -inf becomes a finite value, a NaN stays
        uint32_t r;
        if constexpr (sizeof(T) == 4) asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0xff167699u));   // -2e38
        else if constexpr (__is_same(T, __half)) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0xfbfffbffu));
        else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0xff16ff16u));
        return r;
    }
    static constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : __is_same(T, __half) ? 0xfc00fc00u : 0xff80ff80u;
};

template <typename T, int LP_THREADS>
__global__ void __launch_bounds__(LP_THREADS, 768 / LP_THREADS) logprobs_kernel(const LpArgs a) {
    using V = Vec<T>;
    constexpr int N = V::N, UN = 4, LP_WARPS = LP_THREADS / 32;
    __shared__ Stat ws[LP_WARPS];
    __shared__ Key wk[LP_WARPS][32];
    __shared__ uint32_t bar_s;                 // order of the best k-th value seen
    __shared__ int last_in;
    __shared__ float tops[32];
    __shared__ __align__(16) uint32_t look_s[LP_WARPS][UN * 4];   // one lane's values, for the whole warp to look at
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.y, split = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T *x = (const T *)a.x + (size_t)row * a.ld;
    // vector v covers values v N - mis .. of the row: 16-byte aligned, cut at the row's ends
    const int mis = (int)(((uintptr_t)x % 16) / sizeof(T));
    const int c0 = split * a.chunk, c1 = min(a.vocab, c0 + a.chunk);
    const int v0 = (c0 + mis) / N, v1 = (c1 + mis + N - 1) / N;
    // the vectors that lie whole in the range, and those of them that fill whole tiles
    const int w0 = (c0 + mis + N - 1) / N, w1 = max(w0, (c1 + mis) / N);
    constexpr int STRIDE = LP_THREADS * UN;
    const int full = w0 + (w1 - w0) / STRIDE * STRIDE;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x - mis);
    if (threadIdx.x == 0) bar_s = 0;
    __syncthreads();
    // the target's logit, on its way from the start
    int target = -1;
    float tx = 0.f;
    if (threadIdx.x == 0 && a.logp) {
        target = a.target[row];
        if (target >= 0 && target < a.vocab) tx = V::one(x + target);
    }
    Stat st{-INFINITY, 0.f, 0.f};
    unsigned long long s2 = 0, a2 = 0;         // S and A as pairs; st's own are 0 meanwhile
    Key list = 0;
    const int kth = max(a.top, 1) - 1;
    float tv = a.top ? -INFINITY : NAN;        // what a value has to reach; nothing reaches a NaN
    bool barred = false;
    // UN vectors of this thread, the first at value i0, the others STEP values apart; edge: those
    // before c0 and from `stop` on are not this call's (they are -inf) and are not offered
    auto eat = [&](const uint32_t (&w)[UN][4], int i0, int used, bool edge, int stop) {
        constexpr int STEP = LP_THREADS * N;
        uint32_t q = V::max_(V::max_(w[0][0], w[0][1]), V::max_(w[0][2], w[0][3]));
#pragma unroll
        for (int u = 1; u < UN; u++) q = V::max_(q, V::max_(V::max_(w[u][0], w[u][1]), V::max_(w[u][2], w[u][3])));
        float mx;
        if constexpr (sizeof(T) == 4) mx = __uint_as_float(q);
        else {
            const float2 f = V::two(q);
            mx = fmaxf(f.x, f.y);
        }
        mx = fmaxf(mx, -INFINITY);   // nothing but NaN ranks as -inf
        if (mx > st.m) {
            const float2 s = unpack2(s2), t = unpack2(a2);
            st.s = s.x + s.y;
            st.a = t.x + t.y;
            move(st, mx);
            s2 = pack2(st.s, 0.f);
            a2 = pack2(st.a, 0.f);
        }
        if (st.m > V::LOW_M && st.m < HUGE_M) {
            // x - m first: it is exact near the maximum, where a rounded m log2 e would shift every exponent
            const unsigned long long nm2 = pack2(-st.m, -st.m), l2 = pack2(LOG2E, LOG2E);
#pragma unroll
            for (int u = 0; u < UN; u++) {
                if (u >= used) break;   // the same for the CTA
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    float2 f;
                    if constexpr (sizeof(T) == 4)
                        f = make_float2(__uint_as_float(V::floor_(w[u][e])), __uint_as_float(V::floor_(w[u][e + 1])));
                    else f = V::two(V::floor_(w[u][e >> 1]));
                    const unsigned long long t = mul2(add2(pack2(f.x, f.y), nm2), l2);
                    const float2 tt = unpack2(t);
                    const unsigned long long p = pack2(ex2f_(tt.x), ex2f_(tt.y));
                    s2 = add2(s2, p);
                    a2 = fma2(p, t, a2);
                }
            }
        } else {   // nothing but -inf so far, or a row at its type's edge (masked whole by the lowest value)
            float2 s = unpack2(s2), t2 = unpack2(a2);
#pragma unroll
            for (int u = 0; u < UN; u++)
#pragma unroll 1
                for (int e = 0; e < 4; e++) {
                    const uint32_t word = e == 0 ? w[u][0] : e == 1 ? w[u][1] : e == 2 ? w[u][2] : w[u][3];
                    float f[2] = {__uint_as_float(word), -INFINITY};
                    if constexpr (sizeof(T) == 2) {
                        const float2 g = V::two(word);
                        f[0] = g.x, f[1] = g.y;
                    }
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        if (f[y] == -INFINITY) continue;
                        const float t = f[y] - st.m, p = t < -1e4f ? 0.f : ex2f_(t * LOG2E);
                        s.x += p;
                        if (!(p == 0.f)) t2.x = fmaf(p, t * LOG2E, t2.x);
                    }
                }
            s2 = pack2(s.x, s.y);
            a2 = pack2(t2.x, t2.y);
        }
        if (!a.top) return;
        if (!barred) {
            // a first bar: the k-th largest of a warp's lane maxima, the best warp's, or the k-th largest of 32
            // of the CTA's, the same number of each warp's largest, if that is more
            barred = true;
            constexpr int EACH = 32 / LP_WARPS;
            float k = sort32(mx, lane);
            if (lane == kth) atomicMax(&bar_s, order_of(k));
            if (lane < EACH) tops[warp * EACH + lane] = k;
            __syncthreads();
            k = sort32(tops[lane], lane);
            tv = __shfl_sync(0xffffffffu, k, kth);
        }
        const float seen = value_of((Key) * (volatile uint32_t *)&bar_s << 32);
        tv = fmaxf(tv, seen);
        if (!__any_sync(0xffffffffu, mx >= tv)) return;
        // the lanes with a value that may count: the warp looks at one lane's values together. The best that a lane may
        // have is its largest at its first place: equal values behind a full list are passed over
        const Key best = key_of(mx, max(i0, c0));
        Key last = __shfl_sync(0xffffffffu, list, kth);
        unsigned left = __ballot_sync(0xffffffffu, mx >= tv && best > last);
        while (left) {
            const int src = __ffs(left) - 1;
            left &= left - 1;
            if (lane == src)
#pragma unroll
                for (int u = 0; u < UN; u++)
                    *reinterpret_cast<uint4 *>(&look_s[warp][4 * u]) = make_uint4(w[u][0], w[u][1], w[u][2], w[u][3]);
            const int base = __shfl_sync(0xffffffffu, i0, src);
            __syncwarp();
#pragma unroll
            for (int h = 0; h < UN * N; h += 32) {   // 16 or 32 values
                const int v = h + lane, i = base + (v / N) * STEP + v % N;
                Key k = 0;
                if (v < UN * N && (!edge || (i >= c0 && i < stop))) {
                    const float f = fmaxf(V::one(reinterpret_cast<const T *>(look_s[warp]) + v), -INFINITY);
                    if (f >= tv) k = key_of(f, i);
                }
                offer(list, k, kth, lane);
            }
            __syncwarp();
            last = __shfl_sync(0xffffffffu, list, kth);
            left &= __ballot_sync(0xffffffffu, best > last);
        }
        if (last) {
            tv = fmaxf(tv, value_of(last));
            if (lane == 0 && value_of(last) > seen) atomicMax(&bar_s, (uint32_t)(last >> 32));
        }
    };
    auto fetch = [&](uint32_t (&w)[UN][4], int b) {
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const uint4 q = __ldcs(xv + b + u * LP_THREADS + threadIdx.x);
            w[u][0] = q.x, w[u][1] = q.y, w[u][2] = q.z, w[u][3] = q.w;
        }
    };
    {
        uint32_t w[UN][4];
        if (w0 < full) fetch(w, w0);
        for (int b = w0; b < full; b += STRIDE) {   // the next tile comes while this one is worked on
            uint32_t n[UN][4];
            const bool more = b + STRIDE < full;
            if (more) fetch(n, b + STRIDE);
            eat(w, (b + (int)threadIdx.x) * N - mis, UN, false, 0);
            if (more)
#pragma unroll
                for (int u = 0; u < UN; u++)
#pragma unroll
                    for (int e = 0; e < 4; e++) w[u][e] = n[u][e];
        }
        // what is left behind the whole tiles, then a cut vector before them
#pragma unroll 1
        for (int r = full < v1 ? 0 : 1; r < (v0 < w0 ? 2 : 1); r++) {
            const int b = r == 0 ? full : v0, end = r == 0 ? v1 : w0;
#pragma unroll
            for (int u = 0; u < UN; u++) {
                const int v = b + u * LP_THREADS + threadIdx.x, i0 = v * N - mis;
#pragma unroll
                for (int e = 0; e < 4; e++) w[u][e] = V::NONE;
                if (v >= w0 && v < w1 && v < end) {
                    const uint4 q = __ldcs(xv + v);
                    w[u][0] = q.x, w[u][1] = q.y, w[u][2] = q.z, w[u][3] = q.w;
                } else if (v < end) {
#pragma unroll
                    for (int e = 0; e < N; e++)
                        if (i0 + e >= c0 && i0 + e < c1) {
                            if constexpr (sizeof(T) == 4) w[u][e] = reinterpret_cast<const uint32_t *>(x)[i0 + e];
                            else {
                                const uint32_t h = reinterpret_cast<const uint16_t *>(x)[i0 + e];
                                w[u][e >> 1] = e & 1 ? (w[u][e >> 1] & 0xffffu) | (h << 16) : (w[u][e >> 1] & 0xffff0000u) | h;
                            }
                        }
                }
            }
            eat(w, (b + (int)threadIdx.x) * N - mis, (end - b + LP_THREADS - 1) / LP_THREADS, true,
                min(c1, end * N - mis));
        }
    }
    const float2 s = unpack2(s2), t = unpack2(a2);
    st.s = s.x + s.y;
    st.a = t.x + t.y;
    st = warp_join(st);
    // the CTA's (m, S, A) and list: a tree over the warps
    auto cta = [&]() {
        if (lane == 0) ws[warp] = st;
        wk[warp][lane] = list;
        __syncthreads();
        if (a.top)
#pragma unroll 1
            for (int h = LP_WARPS / 2; h > 0; h >>= 1) {
                if (warp < h) wk[warp][lane] = list = merge(list, wk[warp + h][31 - lane], lane);
                __syncthreads();
            }
        if (warp == 0) st = warp_join(lane < LP_WARPS ? ws[lane] : Stat{-INFINITY, 0.f, 0.f});
    };
    cta();
    if (a.splits > 1) {
        float *p = a.part + ((size_t)row * a.splits + split) * LP_PART;
        if (warp == 0) {
            if (lane == 0) {
                p[0] = st.m;
                p[1] = st.s;
                p[2] = st.a;
            }
            reinterpret_cast<Key *>(p + 4)[lane] = list;
            __syncwarp();
            if (lane == 0) {
                __threadfence();
                last_in = atomicAdd(a.tickets + row, 1u) == (unsigned)(a.splits - 1);
                __threadfence();
            }
        }
        __syncthreads();
        if (!last_in) return;
        if (threadIdx.x == 0) a.tickets[row] = 0u;
        p = a.part + (size_t)row * a.splits * LP_PART;
        st = Stat{-INFINITY, 0.f, 0.f};
        list = 0;
        for (int c0 = warp; c0 < a.splits; c0 += 4 * LP_WARPS) {   // 4 parts a warp in flight
            Key k[4];
            Stat q[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float *pc = p + (size_t)min(c0 + i * LP_WARPS, a.splits - 1) * LP_PART;
                const bool in = c0 + i * LP_WARPS < a.splits;
                q[i] = in ? Stat{__ldcg(pc), __ldcg(pc + 1), __ldcg(pc + 2)} : Stat{-INFINITY, 0.f, 0.f};
                k[i] = in ? __ldcg(reinterpret_cast<const Key *>(pc + 4) + (i & 1 ? 31 - lane : lane)) : 0;
            }
            if (lane == 0) st = join(st, join(join(q[0], q[1]), join(q[2], q[3])));
            if (a.top) {
                k[0] = merge(k[0], k[1], lane);
                k[2] = merge(k[2], k[3], lane);
                list = merge(list, __shfl_sync(0xffffffffu, merge(k[0], __shfl_sync(0xffffffffu, k[2], 31 - lane), lane),
                                               31 - lane), lane);
            }
        }
        cta();
    }
    if (warp != 0) return;
    // no distribution: a NaN in the sums, +inf (whose reference makes them NaN) or nothing but -inf
    const float ls = log2f(st.s) * LN2;
    const bool sound = st.s > 0.f;
    if (lane == 0) {
        if (a.logp) {
            a.logp[row] = target < 0 ? 0.f : target < a.vocab && sound ? (tx - st.m) - ls : NAN;
            if (target >= a.vocab && a.err) atomicExch(a.err, DEV_BAD_INDEX);
        }
        if (a.entropy) a.entropy[row] = sound ? fmaxf(ls - st.a / st.s * LN2, 0.f) : NAN;
    }
    if (lane < a.top) {
        a.ids[(size_t)row * a.top + lane] = index_of(list);
        a.best[(size_t)row * a.top + lane] = sound ? (value_of(list) - st.m) - ls : NAN;
    }
}

// The CTAs of a row and their threads. Few rows, whose tiles of 4 vectors a thread (32 KB) are no more
// than the SMs: CTAs of 512 threads, one an SM, one tile each; their 16 warps look at a tile's best and
// join the parts' lists faster (12 x 131072 bf16, 8 alternatives: 8.0 us, and 11.3 with 128 threads;
// 64 x 10000: 5.0 and 9.1), and smaller tiles would only make more parts (12 x 10000: 4.9, and 9.1 as 3
// parts of a vector a thread). Else an SM holds 6 CTAs of 128 threads, so that about as many rows (or parts of
// rows) as the SMs hold run side by side and share the memory until the end (24 x 131072: 9.8 us, and
// 13.2 with 512), and so for rows that 128 threads read at once (12 x 1000: 5.5 us, and 6.8 with 512).
int plan(const LpArgs &a, int size, int *chunk, int *threads) {
    const int slots = 6 * sm_count(), n = 16 / size;
    const long long tiles = ((long long)a.vocab + 4 * 512 * n - 1) / (4 * 512 * n);
    *threads = a.vocab > 128 * n && a.rows * tiles <= sm_count() ? 512 : 128;
    const int tile = *threads * n;
    long long s = *threads == 512 ? tiles : slots / a.rows;
    const long long most = ((long long)a.vocab + tile - 1) / tile;   // a vector a thread at least
    if (s > most) s = most;
    if (s > LP_SPLITS) s = LP_SPLITS;
    if (s < 1) s = 1;
    const long long per = ((a.vocab + s - 1) / s + tile - 1) / tile * tile;
    *chunk = (int)(per < a.vocab ? per : a.vocab);
    return (int)((a.vocab + (long long)*chunk - 1) / *chunk);
}

template <typename T>
cudaError_t launch(LpArgs &a, cudaStream_t s) {
    int threads;
    a.splits = plan(a, sizeof(T), &a.chunk, &threads);
    const dim3 grid(a.splits, a.rows);
    return threads == 512 ? launch_pdl(logprobs_kernel<T, 512>, grid, dim3(512), 0, s, a)
                          : launch_pdl(logprobs_kernel<T, 128>, grid, dim3(128), 0, s, a);
}

// Rows that are split, and their parts: no more than the CTAs side by side (plan()). The tickets lie at the same
// place for every number of rows, so that a workspace may serve calls of fewer rows, too.
int most_parts() { return 6 * sm_count(); }
size_t ticket_bytes() { return ((size_t)most_parts() * 4 + 255) / 256 * 256; }

}  // namespace
}  // namespace spk

extern "C" {

size_t spk_logprobs_workspace_bytes(int rows, int vocab) {
    using namespace spk;
    if (rows < 1 || vocab < 1) return 0;
    const long long parts = (long long)rows * LP_SPLITS;
    return ticket_bytes() + (size_t)(parts < most_parts() ? parts : most_parts()) * LP_PART * sizeof(float);
}
int spk_logprobs(const void *logits, int type, int rows, int vocab, long long ld, const int *target, float *logp,
                 float *entropy, int top, int *top_ids, float *top_logp, void *workspace, void *stream) {
    using namespace spk;
    const char *who = "spk_logprobs";
    if (type < 0 || type > 2) return set_error("%s: type %d (0 f32, 1 f16, 2 bf16)", who, type);
    if (rows < 0 || rows > 65535 || vocab < 1 || vocab > (1 << 30)) return set_error("%s: %d rows of %d", who, rows, vocab);
    if (top < 0 || top > LP_TOP || top > vocab) return set_error("%s: %d alternatives (0 to %d, at most vocab)", who, top, LP_TOP);
    if (rows == 0) return 0;
    const int size = type == 0 ? 4 : 2;
    if ((uintptr_t)workspace % 16) return set_error("%s: the workspace is not 16-byte aligned", who);
    if (!logits || !workspace || (logp && !target) || (top && (!top_ids || !top_logp)))
        return set_error("%s: null buffer", who);
    if ((uintptr_t)logits % size) return set_error("%s: unaligned logits", who);
    if (rows > 1 && ld < vocab) return set_error("%s: row stride %lld under %d", who, ld, vocab);
    LpArgs a{};
    a.x = logits;
    a.ld = ld;
    a.rows = rows;
    a.vocab = vocab;
    a.top = top;
    a.target = target;
    a.logp = logp;
    a.entropy = entropy;
    a.ids = top_ids;
    a.best = top_logp;
    a.tickets = (unsigned int *)workspace;
    a.part = (float *)((uint8_t *)workspace + ticket_bytes());
    a.err = device_error_ptr();
    const cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t e = type == 0 ? launch<float>(a, s) : type == 1 ? launch<__half>(a, s) : launch<__nv_bfloat16>(a, s);
    return e == cudaSuccess ? 0 : cuda_fail(who, e);
}

}  // extern "C"
