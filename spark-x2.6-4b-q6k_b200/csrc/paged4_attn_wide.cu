// paged4_attn_wide.cu — causal grouped-query attention over the pages of the 4-bit cache for many rows (prompt chunks, verify
// batches), on the tcgen05 tensor cores. The definition is paged4_attn.cu's.
//
//   S[128 rows][64 tokens]  = Q K^T       A: the queries, f16, in tensor memory; B: keys, f16, in shared memory
//   O[128 rows][hd]        += P V         A: the weights, f16, in tensor memory, where their scores were; B: values
// A row is a thread of the softmax warps and a lane of tensor memory, so a row's maximum and sum need no exchange. Queries stand
// on a power of two of their row; f32 rows are two f16 terms (the second one's queries lie in shared memory), and so are their weights.
// The cached codes become f16 once per tile, exactly (paged4.cuh), by warps of their own, as 128-byte rows of 64 dims under
// the 128-byte swizzle: read along the dims that is the K-major B operand of the scores, read along the tokens the
// MN-major one of the outputs, so keys and values are laid alike.
//
// Work split: paged_line.cuh's line of groups of 128 rows, one CTA per SM. Warps: 0-3 queries, softmax and outputs,
// 4-11 codes to f16, 12 the MMAs. Each walks the CTA's groups by itself; they meet at mbarriers.
//
// What bounds it: 2048 bf16 rows of 16 heads of 256 behind 6144 cached tokens are 240 GFLOP in 309 us, 0.78 PFLOP/s, 47 % of the measured
// bf16 rate. A tile takes 1.6 us where its products take 0.76: the tensor pipe is busy 37 % of the time and 45 % of the issue slots are used; the
// softmax warps are the longest chain (scores out of the tensor memory, exponentials, weights back), the converting warps nearly as long. Eight softmax
// warps, two to 32 rows, would halve that chain, but 16 or 17 warps have 112 registers a thread or fewer: their loop spilled, 585 us and more (shares of
// their own by setmaxnreg, more for the softmax warps and fewer for the others, have not been tried). Outputs out of line (433 us for 368 then) and code of their own for keys,
// values and every second tile (1.5 times) were slower too: the loops have to stay in the instruction cache. 13 f32 prompts of
// up to 701 rows, 10 GFLOP counted once (f32 rows multiply twice), take 125 us: short groups of which several end in every CTA.
#include "paged4.cuh"
#include "paged_line.cuh"
#include "paged_tc.cuh"

namespace spk {
namespace paged4 {
namespace {

using namespace paged;

constexpr int N = 64, TB = N / BLOCK;                   // tokens of a tile, its blocks
constexpr int R = WIDE_R;
constexpr int QCH = R * 128;                            // 64 dims of the queries' second terms
constexpr int SM_WARPS = 4, DQ_WARPS = 8, MMA_WARP = SM_WARPS + DQ_WARPS, WARPS = MMA_WARP + 1, THREADS = WARPS * 32;
constexpr int COST = WIDE_COST;
constexpr int RUN = 16, MAX_CTAS = 512;                 // parts that are added together (a join takes 32); CTAs of a call

template <typename T_, int HD_>
struct Cfg {
    using T = T_;
    static constexpr int HD = HD_;
    static constexpr bool TWO = sizeof(T) == 4;
    // log2 of the largest weight at a new reference: the further under W_MAX, the fewer moves, each of which takes a warp's outputs
    // through its registers; a weight is kept down to 2^-24 under it.
    static constexpr float TOP = TWO ? 10.0f : 6.0f;
    // Tiles whose outputs one accumulator adds. The tensor cores cut their sums towards 0, 4e-8 of what is there at each of a tile's 4 steps
    // (f32: 8): 131072 keys of values of one sign ended up 6.6e-4 short. After a span f32 additions take the outputs over, in the workspace.
    static constexpr int SPAN = TWO ? 32 : 256;
    static constexpr int TILE = N * HD * 2;             // bytes of a tile's keys (or values) in f16
    static constexpr int CH = N * 128;                  // 64 dims of them
    static constexpr int V_OFF = 2 * TILE, Q_OFF = 4 * TILE;
    static constexpr int STG_OFF = Q_OFF + (TWO ? R * HD * 2 : 0);   // 4 KB a softmax warp: rows of 128 bytes between their owners and global memory
    static constexpr size_t SMEM = STG_OFF + SM_WARPS * 4096 + 1024;
    static constexpr int TOKENS = HD == 64 ? 1 : 2, HALVES = HD == 256 ? 2 : 1;   // a converting thread's tokens, 64-byte halves of their rows
    static constexpr int QC = HD, SC = HD + HD / 2;     // columns of tensor memory: outputs 0.., queries, scores
    static constexpr int TCOLS = SC + 2 * N <= 256 ? 256 : 512;
};

// Shared-memory operand under the 128-byte swizzle, 8 rows of 128 bytes 1024 bytes apart; lbo: 64 dims to the next 64 (MN-major).
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)((lbo >> 4) & 0x3fffu) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// f32 accumulators, f16 operands, M = 128; B K-major or MN-major
__device__ __forceinline__ constexpr uint32_t idesc(int n, bool mn) { return (1u << 4) | ((uint32_t)mn << 16) | ((uint32_t)(n / 8) << 17) | ((uint32_t)(128 / 16) << 24); }
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool acc) {   // A in tensor memory
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"((uint32_t)acc), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void tm_ld32(uint32_t addr, float *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
                   "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
                   "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
                   "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t addr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tm_wait_ld(float *v, int n) {   // the loads have landed; no use of them moves up
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < n; i++) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// What a softmax thread knows of its row
struct Row {
    float up;                                           // factor of its scores
    int pos, low;                                       // it sees the tokens (low, pos]
};

// The sum of n parts (32 at most) of the group that begins at CTA f0, `step` apart from part `at` on, by the softmax warps: to the outputs, or to the first
// one's place, which this CTA alone reads. wt: 16 KB.
template <typename C>
__device__ __noinline__ void join(const AttnParams &a, int f0, int rows, float *wt, const float *sig_s, const long long *out_s, int at, int step, int n, bool done, int ovec) {
    using T = typename C::T;
    constexpr int HD = C::HD;
    const int tid = threadIdx.x;
    auto part = [&](int p) { return a.part + ((size_t)(f0 + p) * 2 + (p == 0)) * part_floats(R, HD); };   // CTA f0: its second slot, the others: the first
    if (tid < rows) {   // the parts' weights, [n][R]
        float M = -INFINITY, L = 0.f;
#pragma unroll 4
        for (int p = 0; p < n; p++) {
            const float m = __ldcg(part(at + step * p) + R * HD + tid);
            wt[p * R + tid] = m;
            M = fmaxf(M, m);
        }
#pragma unroll 4
        for (int p = 0; p < n; p++) {
            const float m = wt[p * R + tid], l = __ldcg(part(at + step * p) + R * HD + R + tid), f = m == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : ex2(m - M);
            wt[p * R + tid] = f;
            L += m == -INFINITY ? l : l * f;
        }
        if (done) {
            const float fo = L == 0.f ? 0.f : sig_s[tid] / L;
            for (int p = 0; p < n; p++) wt[p * R + tid] = L == 0.f ? 0.f : wt[p * R + tid] * fo;
        } else {
            float *to = part(at) + R * HD;
            __stcg(to + tid, M);
            __stcg(to + R + tid, L);
        }
    }
    bar_sync(1, SM_WARPS * 32);
    const int items = rows * (HD / 4);                   // of 4 values; four of four parts on their way
    for (int x0 = tid; x0 < items; x0 += 4 * SM_WARPS * 32) {
        float4 o[4] = {};
        for (int p = 0; p < n; p += 4) {
            float4 v[4][4];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const float4 *src = reinterpret_cast<const float4 *>(part(at + step * min(p + q, n - 1)));
#pragma unroll
                for (int y = 0; y < 4; y++) v[q][y] = __ldcg(src + min(x0 + y * SM_WARPS * 32, items - 1));
            }
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const float f = p + q < n ? wt[(p + q) * R + min(x0 + y * SM_WARPS * 32, items - 1) / (HD / 4)] : 0.f;
                    if (f == 0.f) continue;              // nothing seen, or nothing to say
                    o[y].x = fmaf(v[q][y].x, f, o[y].x), o[y].y = fmaf(v[q][y].y, f, o[y].y), o[y].z = fmaf(v[q][y].z, f, o[y].z), o[y].w = fmaf(v[q][y].w, f, o[y].w);
                }
        }
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const int x = x0 + y * SM_WARPS * 32;
            if (x >= items) break;
            if (!done) __stcg(reinterpret_cast<float4 *>(part(at)) + x, o[y]);
            else {
                T *dst = (T *)a.out + out_s[x / (HD / 4)] + 4 * (x % (HD / 4));
                T t[4] = {from_f32<T>(o[y].x), from_f32<T>(o[y].y), from_f32<T>(o[y].z), from_f32<T>(o[y].w)};
                if (ovec) {
                    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(t);
                    else *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(t);
                } else {
#pragma unroll
                    for (int z = 0; z < 4; z++) dst[z] = t[z];
                }
            }
        }
    }
}

// A row's outputs and what `sums` has of it under another reference, f its factor (0: nothing yet): to there, or back to the tensor memory. A lane has its row
// in 16-byte pieces 512 bytes apart, so that a warp's lie side by side.
template <typename C, bool BACK>
__device__ __noinline__ void take_over(uint32_t mine, float4 *sums, float f) {
#pragma unroll 1
    for (int c = 0; c < C::HD / 32; c++) {
        float o[32];
        float4 v[8];
#pragma unroll
        for (int y = 0; y < 8; y++) v[y] = f == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : __ldcg(sums + (8 * c + y) * 32);
        tm_ld32(mine + 32 * c, o);
        tm_wait_ld(o, 32);
#pragma unroll
        for (int y = 0; y < 8; y++) {
            v[y].x = fmaf(v[y].x, f, o[4 * y]), v[y].y = fmaf(v[y].y, f, o[4 * y + 1]);
            v[y].z = fmaf(v[y].z, f, o[4 * y + 2]), v[y].w = fmaf(v[y].w, f, o[4 * y + 3]);
        }
        if constexpr (BACK) {
            uint32_t u[32];
#pragma unroll
            for (int y = 0; y < 8; y++) {
                u[4 * y] = __float_as_uint(v[y].x), u[4 * y + 1] = __float_as_uint(v[y].y);
                u[4 * y + 2] = __float_as_uint(v[y].z), u[4 * y + 3] = __float_as_uint(v[y].w);
            }
            tm_st32(mine + 32 * c, u);
        } else {
#pragma unroll
            for (int y = 0; y < 8; y++) __stcg(sums + (8 * c + y) * 32, v[y]);
        }
    }
    if constexpr (BACK) tm_wait_st();
    tc_before();
}

// A warp's queries, `rows` of 32 (src: where this thread's lies), to where the MMAs read them. Returns the factor of the row's scores. Not inlined: the
// loads on their way would cost the main loop its registers.
template <typename C, bool VEC>
__device__ __noinline__ float queries_in(const AttnParams &a, uint8_t *smem, uint8_t *stg, uint32_t mine, long long src, int rows, uint64_t *q_full) {
    using T = typename C::T;
    constexpr int HD = C::HD, LPR = HD / 8, GH = 32 / LPR, B = sizeof(T) == 4 ? 4 : 8;   // lanes of a row, rows of a load, loads on their way
    constexpr bool TWO = C::TWO;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    struct Eight {                                                    // values of a row, as they lie or (unaligned rows) as they are
        uint4 w[sizeof(T) == 4 || !VEC ? 2 : 1];
        __device__ __forceinline__ void load(const T *p) {
            if constexpr (VEC) {
                w[0] = __ldg(reinterpret_cast<const uint4 *>(p));
                if constexpr (sizeof(T) == 4) w[1] = __ldg(reinterpret_cast<const uint4 *>(p) + 1);
            } else {
                float *x = reinterpret_cast<float *>(w);
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = to_f32<T>(p[i]);
            }
        }
        __device__ __forceinline__ void f32(float (&x)[8]) const {
            const uint32_t v[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
            if constexpr (sizeof(T) == 4 || !VEC) {
                const uint32_t u[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = __uint_as_float(v[i]), x[4 + i] = __uint_as_float(u[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (__is_same(T, __half)) {
                        const float2 f = unpack_f16(v[i]);
                        x[2 * i] = f.x, x[2 * i + 1] = f.y;
                    } else {
                        x[2 * i] = __uint_as_float(v[i] << 16), x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
                    }
                }
            }
        }
    };
    float up = 0.f;
    if (rows > 0) {   // rows past the last one have its values, which nobody reads
        float mx = 0.f;
#pragma unroll 1
        for (int i0 = 0; i0 < LPR; i0 += B) {                         // the rows' largest
            Eight raw[B];
#pragma unroll
            for (int i = 0; i < B; i++) {
                const long long at = __shfl_sync(0xffffffffu, src, min((i0 + i) * GH + lane / LPR, rows - 1));
                raw[i].load((const T *)a.q + at + 8 * (lane % LPR));
            }
#pragma unroll
            for (int i = 0; i < B; i++) {
                float x[8], y = 0.f;
                raw[i].f32(x);
#pragma unroll
                for (int e = 0; e < 8; e++) y = fmaxf(y, fabsf(x[e]));
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, o));
                y = __shfl_sync(0xffffffffu, y, (lane % GH) * LPR);
                if (lane / GH == i0 + i) mx = y;
            }
        }
        const int e = mx > 0.f && mx < INFINITY ? min(14 - ilogbf(mx), 126) : 0;   // 2^e brings the largest into [2^14, 2^15)
        const float f = __int_as_float((e + 127) << 23);
        up = a.scale * __int_as_float((127 - e) << 23);
#pragma unroll 1
        for (int c = 0; c < HD / 64; c++) {                           // 64 dims
#pragma unroll 1
            for (int i0 = 0; i0 < 8; i0 += B) {
                Eight raw[B];
#pragma unroll
                for (int i = 0; i < B; i++) {
                    const long long at = __shfl_sync(0xffffffffu, src, min(4 * (i0 + i) + lane / 8, rows - 1));
                    raw[i].load((const T *)a.q + at + 64 * c + 8 * (lane % 8));
                }
#pragma unroll
                for (int i = 0; i < B; i++) {
                    const int rr = 4 * (i0 + i) + lane / 8, pc = lane % 8;
                    const float fr = __shfl_sync(0xffffffffu, f, min(rr, rows - 1));
                    float x[8];
                    raw[i].f32(x);
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int z = 0; z < 4; z++) {
                        const float p = x[2 * z] * fr, q = x[2 * z + 1] * fr;
                        hi[z] = pack_f16(p, q);
                        const float2 b = unpack_f16(hi[z]);
                        lo[z] = pack_f16(p - b.x, q - b.y);
                    }
                    const uint32_t to = rr * 128 + ((pc ^ (rr & 7)) << 4);
                    *reinterpret_cast<uint4 *>(stg + to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if constexpr (TWO) *reinterpret_cast<uint4 *>(smem + C::Q_OFF + c * QCH + warp * 4096 + to) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            }
            __syncwarp();
            uint32_t w[32];
#pragma unroll
            for (int y = 0; y < 8; y++) {
                const uint4 v = *reinterpret_cast<const uint4 *>(stg + lane * 128 + ((y ^ (lane & 7)) << 4));
                w[4 * y] = v.x, w[4 * y + 1] = v.y, w[4 * y + 2] = v.z, w[4 * y + 3] = v.w;
            }
            __syncwarp();
            tm_st32(mine + C::QC + 32 * c, w);
        }
        tm_wait_st();
        tc_before();
        if constexpr (TWO) fence_proxy_async();
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
    return up;
}

template <typename C>
__global__ void __launch_bounds__(THREADS, 1) attn_kernel(const AttnParams a, const int qvec, const int ovec) {
    using T = typename C::T;
    constexpr int HD = C::HD;
    constexpr bool TWO = C::TWO;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_k[2], empty_k[2], full_v[2], empty_v[2], s_full[2], p_full[2], pv_done[2], q_full, o_full, o_free;
    __shared__ uint32_t pre[MAX_SEQ + 1], wsum[WARPS];
    // Tokens of a tile with poisoned keys or values, and how many softmax warps have read that there are some: the last one clears them. No barrier may depend
    // on the flags: after a wait that ran out the warps may read different ones, and each still has to meet the others at every barrier.
    __shared__ uint32_t bad[4][2], bad_read[4];
    __shared__ Walk walk_s;
    __shared__ Seg seg_s;
    __shared__ int dead, last_s;
    __shared__ uint32_t tmem_s;
    uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(full_k + i, DQ_WARPS / 2);
            mbar_init(full_v + i, DQ_WARPS / 2);
            mbar_init(empty_k + i, 1);
            mbar_init(empty_v + i, 1);
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, SM_WARPS);
            mbar_init(pv_done + i, 1);
        }
        mbar_init(&q_full, SM_WARPS);
        mbar_init(&o_full, 1);
        mbar_init(&o_free, SM_WARPS);
        dead = 0;
        seg_s.k0 = -1;
        fence_mbar_init();
    }
    if (tid < 8) bad[tid >> 1][tid & 1] = bad_read[tid >> 1] = 0;
    if (warp == MMA_WARP) {   // this warp owns the tensor memory
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"((uint32_t)C::TCOLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    pdl_trigger();   // after the allocation: a dependent that took tensor memory first would wait on this kernel
    pdl_wait();
    const uint32_t tmem = tmem_s;

    // the line: an exclusive scan over the sequences
    uint32_t base = 0;
    for (int s0 = 0; s0 < a.b.nseq; s0 += THREADS) {
        const int s = s0 + tid;
        uint32_t n = 0;
        if (s < a.b.nseq) {
            const Seq q = seq_of(a, s, R);
            n = before(q, q.tiles, COST) * a.pool.kv_heads;
        }
        uint32_t x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) wsum[warp] = x;
        __syncthreads();
        uint32_t add = base, all = base;
        for (int w = 0; w < WARPS; w++) {
            if (w < warp) add += wsum[w];
            all += wsum[w];
        }
        if (s < a.b.nseq) pre[s] = add + x - n;
        base = all;
        __syncthreads();
    }
    if (tid == 0) pre[a.b.nseq] = base;
    __syncthreads();
    const uint32_t chunk = max((base + gridDim.x - 1) / gridDim.x, (uint32_t)TB), x0 = chunk * blockIdx.x;
    for (int s = tid; s < a.b.nseq; s += THREADS)
        if (pre[s] <= x0 && x0 < pre[s + 1]) {
            Walk w;
            w.chunk = chunk;
            w.x0 = x0;
            w.x1 = min(base, x0 + chunk);
            walk_at(a, pre, s, R, COST, w);
            Seg first;
            if (walk_next<TB>(a, pre, R, COST, w, first)) seg_s = first;
            walk_s = w;
        }
    __syncthreads();
    Seg sg = seg_s;
    Walk w;
    if (sg.k0 >= 0) w = walk_s;
    auto next = [&]() {   // by value: a group whose address is known would be read from memory again behind every barrier
        Seg g;
        if (!walk_next<TB>(a, pre, R, COST, w, g)) g.k0 = -1;
        return g;
    };
    auto tiles_of = [&](const Seg &g) { return g.k0 < 0 ? 0 : max(0, min(g.k1, (g.nblk + TB - 1) / TB) - g.k0); };

    if (sg.k0 < 0) {
        // nothing for this CTA
    } else if (warp == MMA_WARP) {
        const uint32_t kb = smem_u32(smem), vb = kb + C::V_OFF, qb = kb + C::Q_OFF;
        constexpr uint32_t id_s = idesc(N, false), id_o = idesc(HD, true);
        uint32_t kc = 0, vc = 0, groups = 0;            // tiles whose scores, outputs were issued; groups begun
        auto scores = [&]() {
            const uint32_t i = kc & 1;
            const bool ok = wait_for(full_k + i, (kc >> 1) & 1, &dead, a.err);
            tc_after();
            if (ok && elect_one()) {
                const uint32_t d = tmem + C::SC + i * N;
                // f32 queries' second terms first, while the sum that each step rounds is small: against 64 bits the 13 f32 prompts of
                // 20 to 700 rows are off by 1.1e-6 so, and by 1.5e-6 with the terms in turn; the time is the same
                if constexpr (TWO) {
#pragma unroll
                    for (int k = 0; k < HD / 16; k++)
                        mma_ss(d, desc(qb + (k / 4) * QCH + (k % 4) * 32, 0), desc(kb + i * C::TILE + (k / 4) * C::CH + (k % 4) * 32, 0), id_s, k > 0);
                }
#pragma unroll
                for (int k = 0; k < HD / 16; k++)
                    mma_ts(d, tmem + C::QC + 8 * k, desc(kb + i * C::TILE + (k / 4) * C::CH + (k % 4) * 32, 0), id_s, TWO || k > 0);
                mma_commit(empty_k + i);
                mma_commit(s_full + i);
            }
            __syncwarp();
            kc++;
        };
        for (; sg.k0 >= 0; sg = next()) {
            const int n = tiles_of(sg);
            if (n == 0) continue;
            wait_for(&q_full, groups & 1, &dead, a.err);
            tc_after();
            scores();
            for (int j = 0; j < n; j++) {
                if (j + 1 < n) scores();
                const uint32_t i = vc & 1, ph = (vc >> 1) & 1;
                bool ok = wait_for(full_v + i, ph, &dead, a.err);
                if (j == 0 && groups > 0) ok = wait_for(&o_free, (groups - 1) & 1, &dead, a.err) && ok;
                ok = wait_for(p_full + i, ph, &dead, a.err) && ok;
                tc_after();
                if (ok && elect_one()) {
#pragma unroll
                    for (int k = 0; k < N / 16; k++) {
                        const uint64_t b = desc(vb + i * C::TILE + k * 2048, C::CH);
                        mma_ts(tmem, tmem + C::SC + i * N + 8 * k, b, id_o, j % C::SPAN > 0 || k > 0);
                        if constexpr (TWO) mma_ts(tmem, tmem + C::SC + i * N + N / 2 + 8 * k, b, id_o, true);
                    }
                    mma_commit(empty_v + i);
                    mma_commit(pv_done + i);
                    if (j + 1 == n) mma_commit(&o_full);
                }
                __syncwarp();
                vc++;
            }
            groups++;
        }
    } else if (warp >= SM_WARPS) {
        // Codes to f16: keys by four warps, values by four. Eight neighbouring threads have the same 32 dims of eight tokens, so that their
        // stores meet all banks; a warp has 64 bytes of eight rows at a time (heads of 64: all 32 bytes of sixteen). The next tile's bytes are on
        // their way while one is converted, the pages of the one behind it.
        // One code for both: the kernel's loops have to fit the instruction cache together (with keys, values and every second tile by code
        // of their own, 2048-row chunks took 1.5 times as long).
        constexpr int G = C::TOKENS, H = C::HALVES, STEP = HD == 64 ? 64 : 32;   // tokens of a thread, 64-byte halves of their rows; tokens apart
        const bool keys = warp < SM_WARPS + DQ_WARPS / 2;
        const int w4 = warp & 3, x = HD == 64 ? lane >> 3 & 1 : lane >> 3, tok0 = HD == 64 ? w4 * 16 + (lane >> 4) * 8 + (lane & 7) : w4 * 8 + (lane & 7);
        const int per = a.pool.page_tokens / BLOCK, per_tile = TB / per, per_rest = TB % per;
        const uint8_t *pool = (keys ? a.pool.k : a.pool.v) + 16 * x, *scales = (keys ? a.pool.ks : a.pool.vs) + 2 * x, *vscales = a.pool.vs + 2 * x;
        uint64_t *full = keys ? full_k : full_v, *empty = keys ? empty_k : empty_v;
        uint32_t to[4];
#pragma unroll
        for (int y = 0; y < 4; y++) to[y] = (keys ? 0 : C::V_OFF) + (x >> 1) * C::CH + tok0 * 128 + ((((x & 1) * 4 + y) ^ (tok0 & 7)) << 4);
        uint32_t tc = 0;
        for (; sg.k0 >= 0; sg = next()) {
            const int n = tiles_of(sg);
            if (n == 0) continue;
            const int *table = a.b.table + (size_t)sg.s * a.b.max_pages;
            int at_j = 0, idx[G], rest[G], page[G], row[G];      // the next tile to be looked up: its blocks' pages of the table, blocks of those; a token's
                                                                 // page as the table has it, its token of the page (-1 where no row sees it)
#pragma unroll
            for (int u = 0; u < G; u++) {
                const int blk = sg.start / BLOCK + sg.k0 * TB + (tok0 + STEP * u) / BLOCK;
                idx[u] = blk / per;
                rest[u] = blk % per;
            }
            auto look_up = [&]() {
#pragma unroll
                for (int u = 0; u < G; u++) {
                    const int at = sg.start + (sg.k0 + at_j) * N + tok0 + STEP * u;
                    const bool seen = at_j < n && at >= sg.see0 && at <= sg.p_hi;
                    page[u] = __ldg(table + (seen ? idx[u] : 0));
                    row[u] = seen ? rest[u] * BLOCK + tok0 % BLOCK : -1;
                    idx[u] += per_tile;
                    rest[u] += per_rest;
                    if (rest[u] >= per) rest[u] -= per, idx[u]++;
                }
                at_j++;
            };
            uint4 c[G][H];
            uint32_t sc[G][H], vs[G][H];                         // vs: the tokens' scales of values, which are looked at for poison beside keys, too
            bool there[G];
            auto load = [&]() {
#pragma unroll
                for (int u = 0; u < G; u++) {
                    there[u] = row[u] >= 0 && (unsigned)page[u] < (unsigned)a.pool.pages;
                    if (!there[u] && row[u] >= 0 && a.err) atomicExch(a.err, DEV_BAD_INDEX);
                    // fewer than 2^32 rows of a pool fit the device; a token that none sees has row 0's bytes under scales of 0
                    const size_t at = there[u] ? ((uint32_t)page[u] * a.pool.kv_heads + sg.kvh) * a.pool.page_tokens + row[u] : 0;
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        c[u][h] = __ldg(reinterpret_cast<const uint4 *>(pool + at * (HD / 2) + 64 * h));
                        sc[u][h] = __ldg(reinterpret_cast<const uint16_t *>(scales + at * (HD / GROUP) + 8 * h));
                        vs[u][h] = __ldg(reinterpret_cast<const uint16_t *>(vscales + at * (HD / GROUP) + 8 * h));
                    }
                }
            };
            look_up();
            load();
            look_up();
#pragma unroll 1
            for (int j = 0; j < n; j++) {
                const uint32_t i = tc & 1;
                if (tc > 1) wait_for(empty + i, ((tc >> 1) - 1) & 1, &dead, a.err);
#pragma unroll
                for (int u = 0; u < G; u++)
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        const int tok = tok0 + STEP * u;
                        uint32_t s2 = there[u] ? sc[u][h] : 0;
                        // a key's own scales, too: byte 248 is an infinity, whose score may be -inf and its weight 0
                        if (there[u] && poisoned(vs[u][h] | sc[u][h] << 16)) {
                            if (keys) atomicOr(&bad[tc & 3][tok >> 5], 1u << (tok & 31));
                            else {   // poisoned values become 0: their tokens' weights say NaN where they are seen
                                if ((s2 & 0xff) >= POISON) s2 &= 0xff00;
                                if ((s2 >> 8) >= POISON) s2 &= 0x00ff;
                            }
                        }
                        const uint32_t wd[4] = {c[u][h].x, c[u][h].y, c[u][h].z, c[u][h].w}, s4[2] = {(s2 & 0xff) * 0x00800080u, (s2 >> 8) * 0x00800080u};
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            uint32_t f[4];
                            codes_f16(wd[y], f);
                            const uint4 v = make_uint4(hmul2(f[0], s4[y >> 1]), hmul2(f[1], s4[y >> 1]), hmul2(f[2], s4[y >> 1]), hmul2(f[3], s4[y >> 1]));
                            *reinterpret_cast<uint4 *>(smem + i * C::TILE + to[y] + u * STEP * 128 + h * 2 * C::CH) = v;
                        }
                    }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(full + i);
                tc++;
                load();
                look_up();
            }
        }
    } else {
        const int r = tid;
        const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);   // the warp's lanes of tensor memory
        // What a tile does not need lies in shared memory, so that the loop's registers hold what it does: the groups, and per row the
        // sigmoid of its gate and where its output lies (-1: no row), of this group and the next
        __shared__ Seg soft_s[2];
        __shared__ float sig_s[2][R];
        __shared__ long long out_s[2][R];
        uint32_t tc = 0, groups = 0;
        uint8_t *stg = smem + C::STG_OFF + warp * 4096;               // 32 rows of 128 bytes, 16-byte pieces spread as their row says
        const uint32_t own = lane * 128, cut = lane & 7;              // this thread's row of them
        // the row of a group that is this thread's, its queries to where the MMAs read them
        auto queries = [&](int side) {
            const Seg &g = soft_s[side];
            Row row{0.f, -1, -1};
            if (g.k0 < 0) return row;
            const int col = g.c0 + r, tok = col / a.group, h = g.kvh * a.group + col % a.group, rows = g.c1 - g.c0 + 1 - 32 * warp;   // of this warp
            const long long src = (long long)(g.r0 + tok) * a.ldq + (long long)h * HD;
            float sig = 1.f;
            long long out = -1;
            if (col <= g.c1) {
                row.pos = max(g.pos0 + tok, -1);                      // all before the first token alike
                row.low = a.window > 0 ? row.pos - a.window : -1;
                out = (long long)(g.r0 + tok) * a.ldout + (long long)h * HD;
                if (a.gate) sig = 1.0f / (1.0f + __expf(-to_f32<T>(((const T *)a.gate)[(long long)(g.r0 + tok) * a.ldgate + h])));
            }
            sig_s[side][r] = sig;
            out_s[side][r] = out;
            if (tiles_of(g) == 0) return row;
            row.up = qvec ? queries_in<C, true>(a, smem, stg, mine, src, rows, &q_full) : queries_in<C, false>(a, smem, stg, mine, src, rows, &q_full);
            return row;
        };
        auto group_is = [&](int side, const Seg &g) {
            if (tid == 0) soft_s[side] = g;
            bar_sync(1, SM_WARPS * 32);
        };
        group_is(0, sg);
        Row row = queries(0);
        for (int cur = 0; soft_s[cur].k0 >= 0; cur ^= 1) {
            const int n = tiles_of(soft_s[cur]), start = soft_s[cur].start + soft_s[cur].k0 * N;
            float m = -INFINITY, l0 = 0.f, l1 = 0.f;
            float stood = -INFINITY;                                   // the reference of what the workspace has
            // The CTA's place for a group's part: none but this group uses it until the group has left (whole groups come before one
            // that goes on in the next CTA).
            float *slot = a.part + ((size_t)blockIdx.x * 2 + (soft_s[cur].k0 == 0 ? 1 : 0)) * part_floats(R, HD);
            float4 *sums = reinterpret_cast<float4 *>(slot) + warp * (8 * HD) + lane;
            auto since = [&]() { return stood == -INFINITY ? 0.f : ex2(stood - m); };
            for (int j = 0; j < n;) {                                   // spans
                const int first = j, stop = min(n, j + C::SPAN);
                for (; j < stop; j++) {
                    const uint32_t i = tc & 1;
                    wait_for(s_full + i, (tc >> 1) & 1, &dead, a.err);
                    __syncwarp();
                    tc_after();
                    const int t0 = start + j * N;
                    const bool edge = __any_sync(0xffffffffu, t0 + N - 1 > row.pos || t0 <= row.low);
                    const uint32_t b0 = *(volatile uint32_t *)&bad[tc & 3][0], b1 = *(volatile uint32_t *)&bad[tc & 3][1];   // tokens with poisoned keys or values
                    // The weights under the reference as it stands, and the largest score. Where one is too large (and at a group's start) the
                    // reference moves, and they are taken again from the scores, which lie there until the weights are stored.
                    uint32_t hi[N / 32][16], lo[N / 32][16];
                    float d0, d1;
                    auto weigh = [&](float ref) {
                        float most = -INFINITY;
                        f32x2 sum = pack2(0.f, 0.f);
                        const f32x2 up2 = pack2(row.up, row.up), ref2 = pack2(-ref, -ref);
#pragma unroll
                        for (int c = 0; c < N / 32; c++) {
                            float s[32], m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                            tm_ld32(mine + C::SC + i * N + 32 * c, s);
                            tm_wait_ld(s, 32);
#pragma unroll
                            for (int x = 0; x < 32; x += 2) {
                                const float2 v = unpack2(mul2(pack2(s[x], s[x + 1]), up2));
                                s[x] = v.x, s[x + 1] = v.y;
                            }
                            if (edge || (b0 | b1)) {
                                const uint32_t flags = c ? b1 : b0;
#pragma unroll
                                for (int x = 0; x < 32; x++) {
                                    const int p = t0 + 32 * c + x;
                                    if (p > row.pos || p <= row.low) s[x] = -INFINITY;
                                    else if (flags >> x & 1) s[x] = NAN;
                                }
                            }
#pragma unroll
                            for (int x = 0; x < 32; x += 2) asm("max.f32 %0, %0, %1, %2;" : "+f"(m4[x / 2 & 3]) : "f"(s[x]), "f"(s[x + 1]));
#pragma unroll
                            for (int x = 0; x < 16; x++) {
                                const float2 w = unpack2(add2(pack2(s[2 * x], s[2 * x + 1]), ref2));   // the largest score's difference is exact, however large
                                const float p = ex2(w.x), q = ex2(w.y);
                                hi[c][x] = pack_f16(p, q);
                                if constexpr (__is_same(T, __nv_bfloat16)) sum = add2(sum, pack2(p, q));   // f16's rounding is beneath bf16's
                                else {
                                    const float2 b = unpack_f16(hi[c][x]);
                                    if constexpr (TWO) {
                                        lo[c][x] = pack_f16(p - b.x, q - b.y);
                                        sum = add2(sum, pack2(p, q));
                                    } else {
                                        sum = add2(sum, pack2(b.x, b.y));
                                    }
                                }
                            }
                            most = fmaxf(most, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
                        }
                        const float2 v = unpack2(sum);
                        d0 = v.x, d1 = v.y;
                        return most;
                    };
#pragma unroll 1
                    for (int again = 0;; again = 1) {
                        const float ref = m == -INFINITY ? 0.f : m, mx = weigh(ref);
                        const bool move = mx - ref > W_MAX || (m == -INFINITY && mx > -INFINITY);
                        if (again || !__any_sync(0xffffffffu, move)) break;
                        const float was = m;
                        if (move) m = mx - C::TOP;
                        const float f = was == -INFINITY ? 0.f : ex2(was - m);
                        l0 *= f, l1 *= f;
                        if (j > first) {   // what the outputs have so far, behind the products before
                            wait_for(pv_done + (i ^ 1), ((tc - 1) >> 1) & 1, &dead, a.err);
                            __syncwarp();
                            tc_after();
#pragma unroll 1
                            for (int c = 0; c < HD / 32; c++) {
                                float o[32];
                                tm_ld32(mine + 32 * c, o);
                                tm_wait_ld(o, 32);
                                uint32_t u[32];
#pragma unroll
                                for (int x = 0; x < 32; x++) u[x] = __float_as_uint(o[x] * f);
                                tm_st32(mine + 32 * c, u);
                            }
                            tm_wait_st();
                        }
                    }
                    l0 += d0, l1 += d1;
                    if constexpr (!TWO) {
#pragma unroll
                        for (int c = 0; c < N / 32; c++) tm_st16(mine + C::SC + i * N + 16 * c, hi[c]);
                    }
                    if constexpr (TWO) {
#pragma unroll
                        for (int c = 0; c < N / 32; c++) {
                            tm_st16(mine + C::SC + i * N + 16 * c, hi[c]);
                            tm_st16(mine + C::SC + i * N + N / 2 + 16 * c, lo[c]);
                        }
                    }
                    if (b0 | b1) {
                        __syncwarp();
                        if (lane == 0 && atomicAdd(&bad_read[tc & 3], 1) == SM_WARPS - 1) bad[tc & 3][0] = bad[tc & 3][1] = bad_read[tc & 3] = 0;
                    }
                    tm_wait_st();
                    tc_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full + i);
                    tc++;
                }
                if (j < n) {
                    wait_for(pv_done + ((tc - 1) & 1), ((tc - 1) >> 1) & 1, &dead, a.err);
                    __syncwarp();
                    tc_after();
                    take_over<C, false>(mine, sums, since());
                    stood = m;
                }
            }
            // the next group's queries, then this one's outputs
            group_is(cur ^ 1, next());
            row = queries(cur ^ 1);
            const Seg &sg = soft_s[cur];
            const bool whole = sg.f0 == sg.f1;
            const long long row_out = out_s[cur][r];
            const float l = l0 + l1;
            if (n > 0) {
                wait_for(&o_full, groups & 1, &dead, a.err);
                __syncwarp();
                tc_after();
                if (n > C::SPAN) {
                    take_over<C, true>(mine, sums, since());
                    tc_after();
                    bar_sync(1, SM_WARPS * 32);                        // the place is read; parts may lie there now
                }
            }
            const float f = !whole ? 1.0f : l == 0.f ? 0.f : sig_s[cur][r] / l;
            const int mrows = sg.c1 - sg.c0 + 1 - 32 * warp;          // rows of this warp
            // 32 columns of outputs at a time; rows leave by 16-byte pieces, eight lanes a row
            auto leave = [&](uint8_t *base, long long to, int size, int c, bool vec) {   // a row's 128 bytes, from byte `to` + 128 c of base on
                __syncwarp();
#pragma unroll
                for (int it = 0; it < 8; it++) {
                    const int rr = 4 * it + lane / 8, pc = lane % 8;
                    const long long at = __shfl_sync(0xffffffffu, to, rr);
                    const uint4 v = *reinterpret_cast<const uint4 *>(stg + rr * 128 + ((pc ^ (rr & 7)) << 4));
                    if (rr >= mrows) continue;
                    uint8_t *dst = base + at + 128 * c + 16 * pc;
                    if (vec) *reinterpret_cast<uint4 *>(dst) = v;
                    else if (size == 4) {
                        reinterpret_cast<uint32_t *>(dst)[0] = v.x, reinterpret_cast<uint32_t *>(dst)[1] = v.y;
                        reinterpret_cast<uint32_t *>(dst)[2] = v.z, reinterpret_cast<uint32_t *>(dst)[3] = v.w;
                    } else {
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int y = 0; y < 8; y++) reinterpret_cast<uint16_t *>(dst)[y] = (uint16_t)(w[y >> 1] >> (16 * (y & 1)));
                    }
                }
                __syncwarp();
            };
#pragma unroll 1
            for (int c = 0; c < HD / 32; c++) {
                float o[32];
                __syncwarp();
                if (n > 0) {
                    tm_ld32(mine + 32 * c, o);
                    tm_wait_ld(o, 32);
                }
#pragma unroll
                for (int x = 0; x < 32; x++) o[x] = n == 0 || l == 0.f ? 0.f : o[x] * f;
                if (!whole || sizeof(T) == 4) {
#pragma unroll
                    for (int y = 0; y < 8; y++) *reinterpret_cast<float4 *>(stg + own + ((y ^ cut) << 4)) = make_float4(o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]);
                    if (!whole) leave((uint8_t *)slot, (long long)r * HD * 4, 4, c, true);
                    else leave((uint8_t *)a.out, row_out * 4, 4, c, ovec);
                } else if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        T v[8];
#pragma unroll
                        for (int z = 0; z < 8; z++) v[z] = from_f32<T>(o[8 * y + z]);
                        *reinterpret_cast<uint4 *>(stg + own + (((4 * (c & 1) + y) ^ cut) << 4)) = *reinterpret_cast<const uint4 *>(v);
                    }
                    if (c & 1) leave((uint8_t *)a.out, row_out * 2, 2, c >> 1, ovec);
                }
            }
            if (n > 0) {
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&o_free);
                groups++;
            }
            if (!whole) {
                // parts are added in CTA order; many of them in two steps (paged4_attn.cu)
                const int parts = sg.f1 - sg.f0 + 1, mine_p = (int)blockIdx.x - sg.f0, runs = parts > 2 * RUN ? (parts + RUN - 1) / RUN : 1;
                if (row_out >= 0) {
                    slot[R * HD + r] = l == 0.f ? -INFINITY : m;
                    slot[R * HD + R + r] = l;
                }
                auto last_of = [&](unsigned int *ticket, int count) {
                    bar_sync(1, SM_WARPS * 32);
                    if (tid == 0) {
                        unsigned int was;
                        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(was) : "l"(ticket) : "memory");
                        const bool last = was == (unsigned)(count - 1);
                        if (last) *ticket = 0u;
                        last_s = last;
                    }
                    bar_sync(1, SM_WARPS * 32);
                    return last_s != 0;
                };
                float *wt = reinterpret_cast<float *>(smem + C::STG_OFF);
                const int rows = sg.c1 - sg.c0 + 1;
                if (runs == 1) {
                    if (last_of(a.tickets + sg.f0, parts)) join<C>(a, sg.f0, rows, wt, sig_s[cur], out_s[cur], 0, 1, parts, true, ovec);
                } else {
                    const int run = mine_p / RUN, count = min(RUN, parts - run * RUN);
                    if (last_of(a.tickets + MAX_CTAS * (run == 0 ? 1 : 2) + sg.f0 + run * RUN, count)) {
                        join<C>(a, sg.f0, rows, wt, sig_s[cur], out_s[cur], run * RUN, 1, count, false, ovec);
                        if (last_of(a.tickets + sg.f0, runs)) join<C>(a, sg.f0, rows, wt, sig_s[cur], out_s[cur], 0, RUN, runs, true, ovec);
                    }
                }
                bar_sync(1, SM_WARPS * 32);   // last_s is free again, and the staging
            }
            bar_sync(1, SM_WARPS * 32);       // the group is done with: its place is the one behind the next's
        }
    }
    tc_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::TCOLS));
    }
}

template <typename C>
int launch_one(const AttnParams &a, cudaStream_t s, const char *who) {
    static bool set[64];
    int dev = 0;
    cudaGetDevice(&dev);
    cudaError_t e = cudaSuccess;
    if (dev < 0 || dev >= 64 || !set[dev]) {
        e = cudaFuncSetAttribute(attn_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
        if (e == cudaSuccess && dev >= 0 && dev < 64) set[dev] = true;
    }
    using T = typename C::T;
    const int per = 16 / (int)sizeof(T);
    const int qvec = (uintptr_t)a.q % 16 == 0 && a.ldq % per == 0, ovec = (uintptr_t)a.out % 16 == 0 && a.ldout % per == 0;
    if (e == cudaSuccess) e = launch_pdl(attn_kernel<C>, dim3(sm_count()), dim3(THREADS), C::SMEM, s, a, qvec, ovec);
    return e == cudaSuccess ? 0 : cuda_fail(who, e);
}
template <typename T>
int launch(const AttnParams &a, cudaStream_t s, const char *who) {
    return a.pool.hd == 256 ? launch_one<Cfg<T, 256>>(a, s, who) : a.pool.hd == 128 ? launch_one<Cfg<T, 128>>(a, s, who) : launch_one<Cfg<T, 64>>(a, s, who);
}

}  // namespace

int attn_wide(const AttnParams &a, int type, cudaStream_t s, const char *who) {
    return type == T_F32 ? launch<float>(a, s, who) : type == T_F16 ? launch<__half>(a, s, who) : launch<__nv_bfloat16>(a, s, who);
}

}  // namespace paged4
}  // namespace spk
