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
// What bounds it: the row's bytes. A CTA streams a range of a row, 16 bytes a load, four loads a
// thread in flight; each thread keeps its own (m, S, A) in f32 in base 2 and moves m when a vector
// of values passes it. The best k (k <= 32) are a list sorted over a warp's lanes; a vector is
// looked at again only if its largest value reaches the list's last, which few do. A row alone is cut
// over many CTAs (rows x splits fill the SMs); the last one to arrive, by a ticket that it resets,
// joins the parts in order.
#include <cuda_bf16.h>

#include "common.cuh"
#include "spk.h"

namespace spk {
namespace {

constexpr int LP_THREADS = 512, LP_WARPS = LP_THREADS / 32;
constexpr int LP_TOP = 32;                 // the most alternatives
constexpr int LP_SPLITS = 64;              // the most CTAs of a row
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float FAR = -1e4f;               // 2^FAR is 0 and FAR * 0 too: where -inf ends in the sums
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
    unsigned int *tickets;                 // [rows], zero at rest
    float *part;                           // [rows][splits][4 + 2 * LP_TOP]
    int *err;
};

__device__ __forceinline__ float ex2f_(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max_nan_(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// (m, S, A) with values in base 2: t = (x - m) log2 e, S = sum 2^t, A = sum t 2^t
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

// lane i of the warp holds the i-th best (value, index); a candidate goes to its place
__device__ __forceinline__ bool before(float x, int i, float y, int j) { return x > y || (x == y && i < j); }
__device__ __forceinline__ void insert(float &lv, int &li, float v, int i, int lane) {
    const bool mine = before(v, i, lv, li);
    const float uv = __shfl_up_sync(0xffffffffu, lv, 1);
    const int ui = __shfl_up_sync(0xffffffffu, li, 1);
    const bool up = __shfl_up_sync(0xffffffffu, (int)mine, 1) && lane > 0;
    if (mine) {
        lv = up ? uv : v;
        li = up ? ui : i;
    }
}
// offers each lane's candidate (ok) to the list; kth: the list's last place that counts
__device__ __forceinline__ void offer(float &lv, int &li, float v, int i, bool ok, int kth, int lane) {
    float tv = __shfl_sync(0xffffffffu, lv, kth);
    int ti = __shfl_sync(0xffffffffu, li, kth);
    unsigned left = __ballot_sync(0xffffffffu, ok && before(v, i, tv, ti));
    while (left) {
        const int src = __ffs(left) - 1;
        insert(lv, li, __shfl_sync(0xffffffffu, v, src), __shfl_sync(0xffffffffu, i, src), lane);
        tv = __shfl_sync(0xffffffffu, lv, kth);
        ti = __shfl_sync(0xffffffffu, li, kth);
        left &= left - 1;
        left &= __ballot_sync(0xffffffffu, ok && before(v, i, tv, ti));
    }
}

template <typename T>
struct Vec {   // 16 bytes of T as f32
    static constexpr int N = 16 / sizeof(T);
    static __device__ __forceinline__ void f32(uint4 w, float (&v)[N]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(u[i]);
            } else if constexpr (sizeof(T) == 2) {
                if constexpr (__is_same(T, __half)) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
                    v[2 * i] = f.x;
                    v[2 * i + 1] = f.y;
                } else {
                    v[2 * i] = __uint_as_float(u[i] << 16);
                    v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
                }
            }
        }
    }
    static __device__ __forceinline__ float one(const T *p) {
        if constexpr (sizeof(T) == 4) return (float)*p;
        else if constexpr (__is_same(T, __half)) return __half2float(*p);
        else return __bfloat162float(*p);
    }
};

template <typename T>
__global__ void __launch_bounds__(LP_THREADS, 2) logprobs_kernel(const LpArgs a) {
    using V = Vec<T>;
    constexpr int N = V::N, UN = 4;
    __shared__ float ws[LP_WARPS][3];
    __shared__ float wv[LP_WARPS][LP_TOP];
    __shared__ int wi[LP_WARPS][LP_TOP];
    __shared__ int last_in;
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.y, split = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T *x = (const T *)a.x + (size_t)row * a.ld;
    // vector v covers values v N - mis .. of the row: 16-byte aligned, cut at the row's ends
    const int mis = (int)(((uintptr_t)x % 16) / sizeof(T));
    const int c0 = split * a.chunk, c1 = min(a.vocab, c0 + a.chunk);
    const int v0 = (c0 + mis) / N, v1 = (c1 + mis + N - 1) / N;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x - mis);
    Stat st{-INFINITY, 0.f, 0.f};
    float lv = -INFINITY;
    int li = 0x7fffffff;
    const int kth = max(a.top, 1) - 1;
    float tv = a.top ? -INFINITY : INFINITY;
    for (int b = v0; b < v1; b += LP_THREADS * UN) {
        float f[UN][N];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const int v = b + u * LP_THREADS + threadIdx.x, i0 = v * N - mis;
            if (v < v1 && i0 >= c0 && i0 + N <= c1) {
                V::f32(__ldcs(xv + v), f[u]);
            } else {
#pragma unroll
                for (int e = 0; e < N; e++)
                    f[u][e] = v < v1 && i0 + e >= c0 && i0 + e < c1 ? V::one(x + i0 + e) : -INFINITY;
            }
        }
        bool some[UN];
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < UN; u++) {
            float w = f[u][0];
#pragma unroll
            for (int e = 1; e < N; e++) w = fmaxf(w, f[u][e]);
            some[u] = w >= tv;
            mx = fmaxf(mx, w);
        }
        if (mx > st.m) move(st, mx);
        if (fabsf(st.m) < HUGE_M) {
            const float nm = -st.m * LOG2E;
#pragma unroll
            for (int u = 0; u < UN; u++)
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const float t = max_nan_(fmaf(f[u][e], LOG2E, nm), FAR), p = ex2f_(t);
                    st.s += p;
                    st.a = fmaf(p, t, st.a);
                }
        } else {   // nothing but -inf so far, or a row at the edge of f32 (masked whole by the lowest value)
#pragma unroll
            for (int u = 0; u < UN; u++)
#pragma unroll
                for (int e = 0; e < N; e++) {
                    if (f[u][e] == -INFINITY) continue;
                    const float t = max_nan_((f[u][e] - st.m) * LOG2E, FAR), p = ex2f_(t);
                    st.s += p;
                    st.a = fmaf(p, t, st.a);
                }
        }
        bool any = false;
#pragma unroll
        for (int u = 0; u < UN; u++) any |= some[u];
        if (a.top && __any_sync(0xffffffffu, any)) {
#pragma unroll
            for (int u = 0; u < UN; u++) {
                if (!__any_sync(0xffffffffu, some[u])) continue;
                const int i0 = (b + u * LP_THREADS + threadIdx.x) * N - mis;
#pragma unroll
                for (int e = 0; e < N; e++)
                    offer(lv, li, fmaxf(f[u][e], -INFINITY), i0 + e, i0 + e >= c0 && i0 + e < c1, kth, lane);
            }
            tv = __shfl_sync(0xffffffffu, lv, kth);
        }
    }
    // the CTA's (m, S, A) and list
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Stat q{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                     __shfl_xor_sync(0xffffffffu, st.a, o)};
        st = join(st, q);
    }
    if (lane == 0) {
        ws[warp][0] = st.m;
        ws[warp][1] = st.s;
        ws[warp][2] = st.a;
    }
    wv[warp][lane] = lv;
    wi[warp][lane] = li;
    __syncthreads();
    if (warp != 0) return;
    st = Stat{ws[0][0], ws[0][1], ws[0][2]};
    for (int w = 1; w < LP_WARPS; w++) {
        st = join(st, Stat{ws[w][0], ws[w][1], ws[w][2]});
        if (a.top) offer(lv, li, wv[w][lane], wi[w][lane], lane < a.top, kth, lane);
    }
    if (a.splits > 1) {
        float *p = a.part + ((size_t)row * a.splits + split) * (4 + 2 * LP_TOP);
        if (lane == 0) {
            p[0] = st.m;
            p[1] = st.s;
            p[2] = st.a;
        }
        p[4 + lane] = lv;
        reinterpret_cast<int *>(p)[4 + LP_TOP + lane] = li;
        __threadfence();
        __syncwarp();
        if (lane == 0) last_in = atomicAdd(a.tickets + row, 1u) == (unsigned)(a.splits - 1);
        __syncwarp();
        if (!last_in) return;
        __threadfence();
        if (lane == 0) a.tickets[row] = 0u;
        p = a.part + (size_t)row * a.splits * (4 + 2 * LP_TOP);
        lv = -INFINITY;
        li = 0x7fffffff;
        st = Stat{-INFINITY, 0.f, 0.f};
        for (int c = 0; c < a.splits; c++, p += 4 + 2 * LP_TOP) {
            st = join(st, Stat{__ldcg(p), __ldcg(p + 1), __ldcg(p + 2)});
            if (a.top)
                offer(lv, li, __ldcg(p + 4 + lane), __ldcg(reinterpret_cast<const int *>(p) + 4 + LP_TOP + lane),
                      lane < a.top, kth, lane);
        }
    }
    // no distribution: a NaN in the sums, +inf (whose reference makes them NaN) or nothing but -inf
    const float ls2 = log2f(st.s);                     // log2 S
    const bool sound = st.s > 0.f;
    if (lane == 0) {
        if (a.logp && a.target) {
            const int i = a.target[row];
            float r = NAN;
            if (i >= 0 && i < a.vocab) {
                const float v = V::one(x + i);
                r = sound ? (v - st.m) - ls2 * LN2 : NAN;
            } else if (i < 0) {
                r = 0.f;
            } else if (a.err) {
                atomicExch(a.err, DEV_BAD_INDEX);
            }
            a.logp[row] = r;
        }
        if (a.entropy) a.entropy[row] = sound ? fmaxf((ls2 - st.a / st.s) * LN2, 0.f) : NAN;
    }
    if (lane < a.top) {
        a.ids[(size_t)row * a.top + lane] = li;
        a.best[(size_t)row * a.top + lane] = sound ? (lv - st.m) - ls2 * LN2 : NAN;
    }
}

// CTAs of a row: enough to give every SM two CTAs, each at least two tiles of values
int splits_of(int rows, int vocab, int size, int *chunk) {
    const int tile = LP_THREADS * (16 / size);
    long long s = (2ll * sm_count() + rows - 1) / rows;
    const long long most = (vocab + 2ll * tile - 1) / (2ll * tile);
    if (s > most) s = most;
    if (s > LP_SPLITS) s = LP_SPLITS;
    if (s < 1) s = 1;
    const long long per = ((vocab + s - 1) / s + tile - 1) / tile * tile;
    *chunk = (int)(per < vocab ? per : vocab);
    return (int)((vocab + (long long)*chunk - 1) / *chunk);
}

template <typename T>
cudaError_t launch(const LpArgs &a, cudaStream_t s) {
    return launch_pdl(logprobs_kernel<T>, dim3(a.splits, a.rows), dim3(LP_THREADS), 0, s, a);
}

size_t ticket_bytes(int rows) { return ((size_t)rows * 4 + 255) / 256 * 256; }

}  // namespace
}  // namespace spk

extern "C" {

size_t spk_logprobs_workspace_bytes(int rows, int vocab) {
    using namespace spk;
    if (rows < 1 || vocab < 1) return 0;
    return ticket_bytes(rows) + (size_t)rows * LP_SPLITS * (4 + 2 * LP_TOP) * sizeof(float);
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
    a.splits = splits_of(rows, vocab, size, &a.chunk);
    a.target = target;
    a.logp = logp;
    a.entropy = entropy;
    a.ids = top_ids;
    a.best = top_logp;
    a.tickets = (unsigned int *)workspace;
    a.part = (float *)((uint8_t *)workspace + ticket_bytes(rows));
    a.err = device_error_ptr();
    const cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t e = type == 0 ? launch<float>(a, s) : type == 1 ? launch<__half>(a, s) : launch<__nv_bfloat16>(a, s);
    return e == cudaSuccess ? 0 : cuda_fail(who, e);
}

}  // extern "C"
