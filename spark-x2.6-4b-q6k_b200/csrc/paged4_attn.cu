// paged4_attn.cu — causal grouped-query attention of each sequence's new rows over its pages of the 4-bit cache, for few
// rows: decode steps and small verify batches.
//
//   out[t][h] = sigmoid(gate[t][h]) * sum_j p_j V_j,  p = softmax_j(scale * q[t][h] . K_j),
//   j in [0, pos_t], with a window in (pos_t - window, pos_t]. A row that sees nothing gets 0; one that sees a token with a
//   poisoned group gets NaN, and no other does.
//
// What bounds it: the cached bytes (288 a token and KV head of 256), so they go from the copies straight to the registers that multiply
// them: cvt.f16x2.e2m1x2 and a product with the group's scale, both exact, give the operands of mma.sync m16n8k16. (The tensor memory path would
// write them to shared memory as f16 and read them back, eight times the cached bytes each way, which the cache's own rate does not leave room for.)
//   S^T[16 tokens][8 rows] = K Q^T:    A = keys, B = the tile's 8 query rows as f16 (f32 rows are two terms)
//   O^T[16 dims][8 rows]  += V^T P^T:  A = values, two tokens' codes of a dim side by side, B = the weights, which are the scores'
//                                      accumulators turned round (f32 rows': two terms)
// Four f32 rows or fewer have their second terms in the columns of the other four, which costs nothing.
// The contraction's order is free, so a lane takes 16 (8) consecutive bytes of a token as its share of K.
// Queries stand on a power of two of their row (2^14 to 2^15 at the largest), weights are 2^(s - m) with the row's largest at
// 2^12 to 2^15: a reference m moves only when a score passes it by 15, and a weight is kept down to 2^-24, 2^-36 of the
// largest (half of it in its last bit). l adds the weights as they were rounded.
// The matrix instructions cut their sums towards 0: a warp's 2048 blocks of values of one sign in one accumulator end up 1.5e-4 short. So f32 and f16
// rows have a block's products in an accumulator of their own, added in f32 (1.1e-6; 131072 keys of one f32 row 50.7 -> 51.7 us, 24 x 8 f16 rows
// 28.9 -> 29.2); bf16's half unit is 26 times what is lost.
//
// Work split: paged_line.cuh's line of groups of 8 query rows. A CTA's warps take a group's blocks of 16 tokens in turn, each
// with a ring of its own that cp.async fills and a softmax of its own; they meet at the end of the group. Groups that
// several CTAs share leave (O, m, l) in the workspace, and the last CTA to arrive adds the parts in CTA order.
//
// Measured: one f32 row of 16 heads on 4 of 256 over 131072 keys 51.8 us (151 MB of cache, 2.9 TB/s: some 600 warp instructions a block, 45 % of the
// issue slots used by 8 warps an SM, 240 registers each), of which the start and the joining of 74 parts in two steps are some 15; 64 bf16 rows of up
// to 9000 keys 33.1 us (48 MB); 24 x 8 f16 rows of 32 heads on 4 of 128 29.1 us; one row under a window of 512 14.6 us, launch, plan, queries, tiles and
// joining each behind the one before.
#include <limits.h>

#include "paged4.cuh"
#include "paged_line.cuh"
#include "paged_tc.cuh"

namespace spk {
namespace paged4 {
namespace {

using paged::Seg;
using paged::Seq;
using paged::Walk;
using paged::ex2;
using paged::from_f32;
using paged::to_f32;

constexpr int R = 8;                                    // query rows of a group
constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_CTAS_ALL = 512;                       // CTAs of a call: the parts of a group
constexpr int RUN = 16, MAX_JOIN = 32;                  // parts that are added together; at most (a lane each)
static_assert(2 * RUN <= MAX_JOIN && MAX_CTAS_ALL <= RUN * MAX_JOIN, "");
constexpr int COST = 20;                                // a group's fixed cost in blocks (64 bf16 rows 33.3 us; 37.5 with 10, 45.9 with 5, 35.4 with 40)

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of f16, a row's two in a lane, the other way round
__device__ __forceinline__ uint32_t transpose(uint32_t a) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
// n bytes of a copy of N (4, 8 or 16); the rest becomes 0
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void *src, int n) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}

template <bool B>
struct Flag {
    static constexpr bool value = B;
};

template <typename T_, int HD_, int WARPS_, int STAGES_, int CTAS_>
struct Cfg {
    using T = T_;
    static constexpr int HD = HD_, WARPS = WARPS_, THREADS = WARPS * 32, STAGES = STAGES_, CTAS = CTAS_;
    static constexpr bool TWO = sizeof(T) == 4;          // two f16 terms of queries and weights
    static constexpr int ROW = HD / 2, SROW = HD / GROUP;   // bytes of a token's codes, of its scales
    static constexpr int STAGE = BLOCK * 2 * (ROW + SROW);  // a block: codes of keys, of values, scales of keys, of values
    static constexpr int V_OFF = BLOCK * ROW, KS_OFF = 2 * BLOCK * ROW, VS_OFF = KS_OFF + BLOCK * SROW;
    static constexpr int STEPS = HD / 16;                // k16 steps of a score
    static constexpr int QREG = TWO ? 4 : 2;             // words of a lane's share of a query step
    static constexpr int Q_BYTES = STEPS * 32 * QREG * 4;
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int MERGE = WARPS * R * HD * 4;     // the warps' sums at a group's end, where the rings were
    // a merge of parts: their weights, and what the threads that share a value add up
    static constexpr int JOIN = R * MAX_JOIN * 4 + THREADS * 16;
    static constexpr int SMEM = Q_BYTES + (RING > MERGE ? (RING > JOIN ? RING : JOIN) : (MERGE > JOIN ? MERGE : JOIN));
    static constexpr int TB = WARPS;                     // blocks of a tile of the line: one a warp
    static constexpr int WORDS = HD / 64;                // words of 8 dims in a lane's share of a token's values
};

// Sums and parts hold the four values of a lane of an output tile side by side, lane after lane: the first dim of those at `at`.
template <int HD>
__device__ __forceinline__ int dims_of(int at) { return (at >> 2 & 7) * (HD / 8) + (at >> 5) * 4; }

// Four outputs of row r of a group's tile
template <typename C>
__device__ __forceinline__ void output(const AttnParams &a, const Seg &sg, int r, int at, float4 o, float L, float gate) {
    using T = typename C::T;
    const float f = L == 0.f ? 0.f : gate / L;
    if (L == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);
    const int col = sg.c0 + r;
    T *dst = (T *)a.out + (long long)(sg.r0 + col / a.group) * a.ldout + (long long)(sg.kvh * a.group + col % a.group) * C::HD + dims_of<C::HD>(at);
    dst[0] = from_f32<T>(o.x * f);
    dst[1] = from_f32<T>(o.y * f);
    dst[2] = from_f32<T>(o.z * f);
    dst[3] = from_f32<T>(o.w * f);
}

// Part p of a group, in CTA order: CTA f0's second slot, the others' first one
template <typename C>
__device__ __forceinline__ float *part_of(const AttnParams &a, const Seg &sg, int p) {
    return a.part + ((size_t)(sg.f0 + p) * 2 + (p == 0)) * part_floats(R, C::HD);
}

// The sum of n parts of a group, `step` apart from part `at` on, by the CTA: to the outputs, or to the first one's place, which this CTA
// alone reads. Not inlined: the loads on their way would cost the main loop its registers.
template <typename C>
__device__ __noinline__ void join(const AttnParams &a, const Seg &sg, float *wt, const float *gate_s, int at, int step, int n, bool done) {
    constexpr int HD = C::HD, WARPS = C::WARPS;
    __shared__ float M_s[R], L_s[R];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cols = sg.c1 - sg.c0 + 1;
    auto part = [&](int p) { return part_of<C>(a, sg, p); };
    float *red = wt + R * MAX_JOIN;
    // an item: 4 values of a row; `ways` threads share its parts, 8 loads on their way
    const int items = cols * (HD / 4), ways = max(1, min(C::THREADS / items, (n + 7) / 8));
    const int way = ways > 1 ? tid / items : 0, a0 = n * way / ways, a1 = n * (way + 1) / ways;
    float4 v[8];
    auto load = [&](int x, int p) {
        const int r = x / (HD / 4), d = 4 * (x % (HD / 4));
#pragma unroll
        for (int y = 0; y < 8; y++)   // past the last part: the last one again, left out
            v[y] = __ldcg(reinterpret_cast<const float4 *>(part(at + step * min(p + y, a1 - 1)) + r * HD + d));
    };
    const int first = ways > 1 ? tid % items : tid;
    if (first < items && way < ways) load(first, a0);
    for (int r = warp; r < cols; r += WARPS) {   // the parts' weights: a warp per row
        const float m = lane < n ? __ldcg(part(at + step * lane) + R * HD + r) : -INFINITY, x = lane < n ? __ldcg(part(at + step * lane) + R * HD + R + r) : 0.f;
        float M = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float f = m == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : ex2(m - M);
        if (lane < n) wt[r * MAX_JOIN + lane] = f;
        const float L = warp_sum(m == -INFINITY ? x : x * f);
        if (lane == 0) M_s[r] = M, L_s[r] = L;
    }
    __syncthreads();
    for (int x0 = 0; x0 < items; x0 += C::THREADS) {   // one turn where several threads share an item
        const int x = ways > 1 ? first : x0 + tid, r = x / (HD / 4), d = 4 * (x % (HD / 4));
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        const bool own = x < items && way < ways;
        if (own)
            for (int p = a0; p < a1; p += 8) {
                if (x0 > 0 || p > a0) load(x, p);
#pragma unroll
                for (int y = 0; y < 8; y++) {
                    const float f = wt[r * MAX_JOIN + min(p + y, a1 - 1)];
                    if (p + y < a1) o.x = fmaf(v[y].x, f, o.x), o.y = fmaf(v[y].y, f, o.y), o.z = fmaf(v[y].z, f, o.z), o.w = fmaf(v[y].w, f, o.w);
                }
            }
        if (ways > 1) {
            if (own && way > 0) *reinterpret_cast<float4 *>(red + 4 * ((way - 1) * items + x)) = o;
            __syncthreads();
            if (own && way == 0)
                for (int w = 1; w < ways; w++) {
                    const float4 y = *reinterpret_cast<const float4 *>(red + 4 * ((w - 1) * items + x));
                    o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
                }
        }
        if (own && way == 0) {
            if (done) output<C>(a, sg, r, d, o, L_s[r], gate_s[r]);
            else {
                float *to = part(at);
                __stcg(reinterpret_cast<float4 *>(to + r * HD + d), o);
                if (d == 0) __stcg(to + R * HD + r, M_s[r]), __stcg(to + R * HD + R + r, L_s[r]);
            }
        }
    }
}

template <typename C>
__global__ void __launch_bounds__(C::THREADS, C::CTAS) attn_kernel(const AttnParams a) {
    using T = typename C::T;
    constexpr int HD = C::HD, ROW = C::ROW, SROW = C::SROW, STEPS = C::STEPS, WARPS = C::WARPS, WORDS = C::WORDS;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t pre[MAX_SEQ + 1], wsum[WARPS];
    __shared__ float up_s[R], m_s[WARPS][R], l_s[WARPS][R], gate_s[R];
    __shared__ int pos_s[R];
    __shared__ Seg seg_s[2];                                // this group and the next one: the slowest warp still reads the first
    __shared__ Walk walk_s;
    __shared__ int last_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    uint8_t *qs = smem, *ring = smem + C::Q_BYTES + warp * C::STAGES * C::STAGE;
    const uint32_t ring_u = smem_u32(ring);

    pdl_trigger();
    pdl_wait();
    // the line: an exclusive scan over the sequences
    uint32_t base = 0;
    for (int s0 = 0; s0 < a.b.nseq; s0 += C::THREADS) {
        const int s = s0 + tid;
        uint32_t n = 0;
        if (s < a.b.nseq) {
            const Seq q = paged::seq_of(a, s, R);
            n = paged::before(q, q.tiles, COST) * a.pool.kv_heads;
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
    if (tid == 0) {
        pre[a.b.nseq] = base;
        seg_s[0].k0 = -1;
    }
    __syncthreads();
    const uint32_t chunk = max((base + gridDim.x - 1) / gridDim.x, (uint32_t)C::TB), x0 = chunk * blockIdx.x;
    for (int s = tid; s < a.b.nseq; s += C::THREADS)
        if (pre[s] <= x0 && x0 < pre[s + 1]) {
            Walk w;
            w.chunk = chunk;
            w.x0 = x0;
            w.x1 = min(base, x0 + chunk);
            paged::walk_at(a, pre, s, R, COST, w);
            Seg first;
            if (paged::walk_next<C::TB>(a, pre, R, COST, w, first)) seg_s[0] = first;
            walk_s = w;
        }
    __syncthreads();

    const int per = a.pool.page_tokens / BLOCK;
    // Where the lane's 16-byte pieces of a block (piece lane + 32 x) lie in a stage: keys in order, pieces of odd tokens in each other's
    // halves (heads of 256); values with tokens 2t of a phase in neighbouring rows, so that both are read without bank conflicts.
    const int tok_l = lane / (ROW / 16), pc_l = lane % (ROW / 16), slot_l = (tok_l >> 1 & 3) | (tok_l & 1) << 2 | (tok_l & 8);
    const uint32_t kd = tok_l * ROW + 16 * (HD == 256 ? pc_l ^ 4 * (tok_l & 1) : pc_l);
    const uint32_t vd = C::V_OFF + slot_l * ROW + 16 * (HD == 256 ? pc_l ^ 2 * (slot_l & 3) : HD == 128 ? pc_l ^ (slot_l & 2) : pc_l);
    const uint32_t vd_odd = C::V_OFF + (slot_l + 2) * ROW + 16 * (pc_l ^ 2 * ((slot_l + 2) & 3));   // heads of 256: 4 tokens on
    auto kdst = [&](int x) { return kd + 512 * x; };
    auto vdst = [&](int x) { return HD == 256 ? ((x & 1) ? vd_odd : vd) + 1024 * (x >> 1) : vd + 512 * x; };
    const uint32_t sd = (lane < 16 ? C::KS_OFF : C::VS_OFF) + (lane & 15) * SROW;
    const uint8_t *k_l = a.pool.k + 16 * lane, *v_l = a.pool.v + 16 * lane, *s_l = (lane < 16 ? a.pool.ks : a.pool.vs) + (lane & 15) * SROW;
    for (int turn = 0;; turn ^= 1) {
        const Seg sg = seg_s[turn];
        if (sg.k0 < 0) break;
        const int cols = sg.c1 - sg.c0 + 1;
        // blocks of this warp: first + WARPS i, i < count
        const int nblk = min(sg.nblk, sg.k1 * C::TB), first = sg.k0 * C::TB + warp, count = first < nblk ? (nblk - first + WARPS - 1) / WARPS : 0;
        const int *table = a.b.table + (size_t)sg.s * a.b.max_pages;
        // the tile's queries, on their way while the blocks' places are looked up
        constexpr int QROWS = (R + WARPS - 1) / WARPS;
        T qraw[QROWS][HD / 32];
#pragma unroll
        for (int y = 0; y < QROWS; y++) {
            const int r = warp + y * WARPS, col = sg.c0 + r, tok = col / a.group, h = sg.kvh * a.group + col % a.group;
            const T *src = (const T *)a.q + (long long)(sg.r0 + tok) * a.ldq + (long long)h * HD;
#pragma unroll
            for (int i = 0; i < HD / 32; i++) qraw[y][i] = r < cols ? src[lane + 32 * i] : from_f32<T>(0.f);
        }
        // lane i has the place in the pool of block 32 c + i of the warp's; -1: a page that is none
        auto places = [&](int c) {
            const int i = 32 * c + lane;
            long long at = -1;
            if (i < count) {
                const int blk = sg.start / BLOCK + first + WARPS * i, page = __ldg(table + blk / per);
                if (page >= 0 && page < a.pool.pages) at = (long long)row_index(a.pool, page, sg.kvh, blk % per * BLOCK);
                else if (a.err) atomicExch(a.err, DEV_BAD_INDEX);
            }
            return at;
        };
        long long pl = places(0), pl_next = places(1);
        uint32_t to_stage = 0;
        auto fetch = [&](int i) {
            if (i < count) {
                const long long at = __shfl_sync(0xffffffffu, pl, i & 31);
                if ((i & 31) == 31) {
                    pl = pl_next;
                    pl_next = places(i / 32 + 2);
                }
                const int tok0 = sg.start + (first + WARPS * i) * BLOCK;
                const uint32_t st = ring_u + to_stage;
                to_stage = to_stage == (C::STAGES - 1) * C::STAGE ? 0 : to_stage + C::STAGE;
                const size_t row = at < 0 ? 0 : (size_t)at;
                const uint8_t *kc = k_l + row * ROW, *vc = v_l + row * ROW, *sc = s_l + row * SROW;
                const uint32_t sdst = st + sd;
                if (at >= 0 && tok0 >= sg.see0 && tok0 + BLOCK - 1 <= sg.p_hi) {
#pragma unroll
                    for (int x = 0; x < ROW / 32; x++) {
                        copy_async<16>(st + kdst(x), kc + 512 * x, 16);
                        copy_async<16>(st + vdst(x), vc + 512 * x, 16);
                    }
                    copy_async<SROW>(sdst, sc, SROW);
                } else {   // tokens that no row sees arrive as zeros
                    auto live = [&](int tok) { return at >= 0 && tok0 + tok >= sg.see0 && tok0 + tok <= sg.p_hi; };
#pragma unroll
                    for (int x = 0; x < ROW / 32; x++) {
                        const int n = live((lane + 32 * x) / (ROW / 16)) ? 16 : 0;
                        copy_async<16>(st + kdst(x), kc + 512 * x, n);
                        copy_async<16>(st + vdst(x), vc + 512 * x, n);
                    }
                    copy_async<SROW>(sdst, sc, live(lane & 15) ? SROW : 0);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < C::STAGES - 1; i++) fetch(i);

        // f32 rows, four of them at most: the second terms take the columns of rows 4..7
        const bool spare = C::TWO && cols <= 4;
        // the tile's queries, f16 on the row's own power of two, where the lanes' shares of B lie
#pragma unroll
        for (int y = 0; y < QROWS; y++) {
            const int r = warp + y * WARPS, col = sg.c0 + r, tok = col / a.group, h = sg.kvh * a.group + col % a.group;
            if (r >= R) break;
            const bool real = r < cols;
            float x[HD / 32], mx = 0.f;
#pragma unroll
            for (int i = 0; i < HD / 32; i++) {
                x[i] = to_f32<T>(qraw[y][i]);
                mx = fmaxf(mx, fabsf(x[i]));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            // 2^e brings the largest into [2^14, 2^15)
            const int e = mx > 0.f && mx < INFINITY ? min(14 - ilogbf(mx), 126) : 0;
            const float f = __int_as_float((e + 127) << 23);
#pragma unroll
            for (int i = 0; i < HD / 32; i++) {
                const int d = lane + 32 * i;
                const int part = HD == 256 ? d >> 7 : 0, tt = HD == 64 ? d >> 4 : d >> 5 & 3, w = HD == 64 ? d >> 3 & 1 : d >> 3 & 3;
                const int step = (HD == 64 ? 2 * w : 8 * part + 2 * w) + (d >> 2 & 1), reg = d >> 1 & 1;
                const __half hi = __float2half_rn(x[i] * f);
                __half *q = reinterpret_cast<__half *>(qs) + ((step * 32 + 4 * r + tt) * C::QREG + reg) * 2 + (d & 1);
                if (r < 4 || !spare) *q = hi;
                if constexpr (C::TWO) {
                    const __half lo = __float2half_rn(x[i] * f - __half2float(hi));
                    if (!spare) q[4] = lo;
                    else if (r < 4) q[16 * C::QREG * 2] = lo;      // the columns of rows 4..7
                }
            }
            if (lane == 0) {
                up_s[r] = a.scale * __int_as_float((127 - e) << 23);
                pos_s[r] = real ? max(sg.pos0 + tok, -1) : -1;   // all before the first token alike
                gate_s[r] = real && a.gate ? 1.0f / (1.0f + __expf(-to_f32<T>(((const T *)a.gate)[(long long)(sg.r0 + tok) * a.ldgate + h]))) : 1.0f;
            }
        }
        __syncthreads();

        uint32_t qr[STEPS][2];
#pragma unroll
        for (int x = 0; x < STEPS; x++) {
            const uint2 v = *reinterpret_cast<const uint2 *>(qs + (x * 32 + lane) * C::QREG * 4);
            qr[x][0] = v.x, qr[x][1] = v.y;
        }
        // the lane's rows: columns 2t and 2t + 1 of the scores and the outputs
        const int row0 = spare ? 2 * (t & 1) : 2 * t;
        const float up0 = up_s[row0], up1 = up_s[row0 + 1];
        const int pos0 = pos_s[row0], pos1 = pos_s[row0 + 1], back = a.window > 0 ? a.window : INT_MAX;   // a row sees (pos - back, pos]
        float acc[HD / 16][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 16; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[i][e] = 0.f;
        uint32_t at_stage = 0;

        auto blocks = [&](auto spare_) {
        constexpr bool SPARE = decltype(spare_)::value, APART = !__is_same(typename C::T, __nv_bfloat16);
        for (int i = 0; i < count; i++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
            __syncwarp();
            fetch(i + C::STAGES - 1);
            const uint8_t *st = ring + at_stage;
            at_stage = at_stage == (C::STAGES - 1) * C::STAGE ? 0 : at_stage + C::STAGE;
            const int tok0 = sg.start + (first + WARPS * i) * BLOCK;
            // scores: tokens g and g + 8 (c[.][0], c[.][1] and c[.][2], c[.][3]) of the lane's two rows, even and odd steps apart
            float c[2][4] = {};
            uint32_t kbad = 0;            // poisoned scales of keys: of token g in the lower half, of g + 8 in the upper one
#pragma unroll
            for (int h = 0; h < (HD == 256 ? 2 : 1); h++) {
                uint32_t w[2][4], sc[2][2], sb[2];
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const int tok = 8 * n + g;
                    if constexpr (HD == 64) {
                        const uint2 v = *reinterpret_cast<const uint2 *>(st + tok * ROW + 8 * t);
                        w[n][0] = v.x, w[n][1] = v.y, w[n][2] = w[n][3] = 0;
                        sb[n] = st[C::KS_OFF + tok * SROW + t];
                        sc[n][0] = sc[n][1] = sb[n] * 0x00800080u;
                    } else {
                        const uint4 v = *reinterpret_cast<const uint4 *>(st + tok * ROW + 16 * (HD == 256 ? (4 * h + t) ^ 4 * (g & 1) : t));
                        w[n][0] = v.x, w[n][1] = v.y, w[n][2] = v.z, w[n][3] = v.w;
                        sb[n] = *reinterpret_cast<const uint16_t *>(st + C::KS_OFF + tok * SROW + 8 * h + 2 * t);
                        sc[n][0] = (sb[n] & 0xff) * 0x00800080u;
                        sc[n][1] = (sb[n] >> 8) * 0x00800080u;
                    }
                }
                kbad |= poisoned(sb[0] | sb[1] << 16);
#pragma unroll
                for (int x = 0; x < (HD == 64 ? 2 : 4); x++) {
                    uint32_t k[2][4];
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        codes_f16(w[n][x], k[n]);
#pragma unroll
                        for (int y = 0; y < 4; y++) k[n][y] = hmul2(k[n][y], sc[n][x >> 1]);
                    }
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const int step = 8 * h + 2 * x + y;
                        mma(c[y], k[0][2 * y], k[1][2 * y], k[0][2 * y + 1], k[1][2 * y + 1], qr[step][0], qr[step][1]);
                        if constexpr (C::TWO && !SPARE) {
                            const uint2 v = *reinterpret_cast<const uint2 *>(qs + (step * 32 + lane) * 16 + 8);
                            mma(c[y], k[0][2 * y], k[1][2 * y], k[0][2 * y + 1], k[1][2 * y + 1], v.x, v.y);
                        }
                    }
                }
            }
            float s[4];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                s[x] = c[0][x] + c[1][x];
                if constexpr (SPARE) s[x] += __shfl_xor_sync(0xffffffffu, s[x], 2);
                s[x] *= x & 1 ? up1 : up0;
            }
            // what a row does not see; rows that are none have no place in the outputs
            if (tok0 + BLOCK - 1 > sg.p_lo || tok0 <= sg.p_hi - back) {
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int p = tok0 + g + 8 * (x >> 1), pos = x & 1 ? pos1 : pos0;
                    if (p > pos || p <= pos - back) s[x] = -INFINITY;
                }
            }
            // the values' scales of the lane's tokens in their product: 2t, 2t + 1, 2t + 8, 2t + 9
            uint32_t vs[4];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const uint8_t *at = st + C::VS_OFF + (2 * t + (x & 1) + 8 * (x >> 1)) * SROW;
                vs[x] = HD == 256 ? *reinterpret_cast<const uint16_t *>(at + 2 * g) : HD == 128 ? at[g] : at[g >> 1];
            }
            // A key's group is looked at like a value's: under byte 248, an infinity, a score may be -inf and its weight 0.
            if (__any_sync(0xffffffffu, poisoned(vs[0] | vs[1] << 16) | poisoned(vs[2] | vs[3] << 16) | kbad)) {
                uint32_t bad = (kbad & 0xffff ? 1u << g : 0u) | (kbad >> 16 ? 1u << (g + 8) : 0u);         // a bit a token of the block
#pragma unroll
                for (int x = 0; x < 4; x++)
                    if (poisoned(vs[x])) {
                        bad |= 1u << (2 * t + (x & 1) + 8 * (x >> 1));
                        vs[x] = 0;
                    }
                bad = __reduce_or_sync(0xffffffffu, bad);
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int tok = g + 8 * (x >> 1), p = tok0 + tok, pos = x & 1 ? pos1 : pos0;
                    if ((bad >> tok & 1) && p <= pos && p > pos - back) s[x] = NAN;
                }
            }
            // a row's reference moves when one of its scores passes it by W_MAX
            const float t0 = fmaxf(s[0], s[2]), t1 = fmaxf(s[1], s[3]);
            if (__any_sync(0xffffffffu, t0 > m0 + W_MAX || t1 > m1 + W_MAX)) {
                float x0 = t0, x1 = t1;
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, o));
                    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, o));
                }
                const float was0 = m0, was1 = m1;
                if (x0 > m0 + W_MAX) m0 = x0 - W_TOP;
                if (x1 > m1 + W_MAX) m1 = x1 - W_TOP;
                const float f0 = was0 == -INFINITY ? 0.f : ex2(was0 - m0), f1 = was1 == -INFINITY ? 0.f : ex2(was1 - m1);
                l0 *= f0, l1 *= f1;
#pragma unroll
                for (int d = 0; d < HD / 16; d++) acc[d][0] *= f0, acc[d][1] *= f1, acc[d][2] *= f0, acc[d][3] *= f1;
            }
            const float ref0 = m0 == -INFINITY ? 0.f : m0, ref1 = m1 == -INFINITY ? 0.f : m1;
            const float w0 = ex2(s[0] - ref0), w1 = ex2(s[1] - ref1), w2 = ex2(s[2] - ref0), w3 = ex2(s[3] - ref1);
            uint32_t p0 = pack_f16(w0, w1), p1 = pack_f16(w2, w3), e0 = 0, e1 = 0;
            const float2 h0 = unpack_f16(p0), h1 = unpack_f16(p1);
            if constexpr (C::TWO) {
                e0 = pack_f16(w0 - h0.x, w1 - h0.y);
                e1 = pack_f16(w2 - h1.x, w3 - h1.y);
                l0 += w0 + w2, l1 += w1 + w3;
                if (SPARE && t >= 2) p0 = e0, p1 = e1;
            } else {
                l0 += h0.x + h1.x, l1 += h0.y + h1.y;
            }
            p0 = transpose(p0), p1 = transpose(p1);       // from token by row to row by token
            if constexpr (C::TWO && !SPARE) e0 = transpose(e0), e1 = transpose(e1);
            // values: two tokens' codes of a dim in a byte, their scales in a pair
            uint32_t w[4][WORDS];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int slot = t | (x & 1) << 2 | (x >> 1) << 3;
                const uint8_t *at = st + C::V_OFF + slot * ROW;
                if constexpr (HD == 256) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(at + 16 * (g ^ 2 * (slot & 3)));
                    w[x][0] = v.x, w[x][1] = v.y, w[x][2] = v.z, w[x][3] = v.w;
                } else if constexpr (HD == 128) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(at + 16 * ((g >> 1) ^ (slot & 2)) + 8 * (g & 1));
                    w[x][0] = v.x, w[x][1] = v.y;
                } else {
                    w[x][0] = *reinterpret_cast<const uint32_t *>(at + 4 * g);
                }
            }
#pragma unroll
            for (int y = 0; y < WORDS; y++) {
                uint32_t sa, sb;      // scales of the group: tokens 2t and 2t + 1, 2t + 8 and 2t + 9
                if (HD == 256 && y >= 2) {
                    sa = __byte_perm(vs[0], vs[1], 0x5212) >> 1;
                    sb = __byte_perm(vs[2], vs[3], 0x5212) >> 1;
                } else {
                    sa = __byte_perm(vs[0], vs[1], 0x4202) >> 1;
                    sb = __byte_perm(vs[2], vs[3], 0x4202) >> 1;
                }
                const uint32_t lo = 0x0f0f0f0fu;
                uint32_t ae[4], ao[4], be[4], bo[4];   // even and odd dims of the pair's codes
                codes_f16((w[0][y] & lo) | (w[1][y] << 4 & ~lo), ae);
                codes_f16((w[0][y] >> 4 & lo) | (w[1][y] & ~lo), ao);
                codes_f16((w[2][y] & lo) | (w[3][y] << 4 & ~lo), be);
                codes_f16((w[2][y] >> 4 & lo) | (w[3][y] & ~lo), bo);
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const uint32_t a0 = hmul2(ae[x], sa), a1 = hmul2(ao[x], sa), a2 = hmul2(be[x], sb), a3 = hmul2(bo[x], sb);
                    if constexpr (APART) {   // sums of blocks in f32 additions: the matrix instructions cut theirs towards 0
                        float d[4] = {};
                        mma(d, a0, a1, a2, a3, p0, p1);
                        if constexpr (C::TWO && !SPARE) mma(d, a0, a1, a2, a3, e0, e1);
#pragma unroll
                        for (int z = 0; z < 4; z++) acc[4 * y + x][z] += d[z];
                    } else {
                        mma(acc[4 * y + x], a0, a1, a2, a3, p0, p1);
                    }
                }
            }
        }
        };
        if (C::TWO && spare) blocks(Flag<true>());
        else blocks(Flag<false>());
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        // the rows' sums over their eight lanes
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, o);
            l1 += __shfl_xor_sync(0xffffffffu, l1, o);
        }
        if (g == 0 && (!spare || t < 2)) {
            m_s[warp][row0] = m0, m_s[warp][row0 + 1] = m1;
            l_s[warp][row0] = l0, l_s[warp][row0 + 1] = l1;
        }
        __syncthreads();                                  // the rings are done with, too
        // columns 2t, 2t + 1 of acc on the CTA's common reference, into the warps' share of the rings
        float *mine = reinterpret_cast<float *>(smem + C::Q_BYTES) + warp * R * HD;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = 2 * t + e, rm = spare ? r & 3 : r;
            float M = -INFINITY;
            for (int w = 0; w < WARPS; w++) M = fmaxf(M, m_s[w][rm]);
            const float mw = m_s[warp][rm], f = mw == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : ex2(mw - M);
#pragma unroll
            for (int d = 0; d < HD / 16; d += 2) {
                float4 v = make_float4(acc[d][e] * f, acc[d][2 + e] * f, acc[d + 1][e] * f, acc[d + 1][2 + e] * f);
                *reinterpret_cast<float4 *>(mine + r * HD + 16 * d + 4 * g) = v;   // as dims_of() says
            }
        }
        __syncthreads();
        const bool whole = sg.f0 == sg.f1;
        float *slot = a.part + ((size_t)blockIdx.x * 2 + (sg.k0 == 0 ? 1 : 0)) * part_floats(R, HD);
        const float *sums = reinterpret_cast<const float *>(smem + C::Q_BYTES);
        for (int x = tid; x < cols * (HD / 4); x += C::THREADS) {
            const int r = x / (HD / 4), d = 4 * (x % (HD / 4));
            float M = -INFINITY, L = 0.f;
            for (int w = 0; w < WARPS; w++) M = fmaxf(M, m_s[w][r]);
            for (int w = 0; w < WARPS; w++) L += m_s[w][r] == -INFINITY ? l_s[w][r] : l_s[w][r] * ex2(m_s[w][r] - M);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int w = 0; w < WARPS; w++) {
                const float4 v = *reinterpret_cast<const float4 *>(sums + (w * R + r) * HD + d);
                o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
                if (spare) {
                    const float4 y = *reinterpret_cast<const float4 *>(sums + (w * R + r + 4) * HD + d);
                    o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
                }
            }
            if (whole) output<C>(a, seg_s[turn], r, d, o, L, gate_s[r]);
            else {
                *reinterpret_cast<float4 *>(slot + r * HD + d) = o;
                if (d == 0) {
                    slot[R * HD + r] = M;
                    slot[R * HD + R + r] = L;
                }
            }
        }
        if (!whole) {
            // Parts are added in CTA order. Many of them (a long sequence of few rows) in two steps, so that no CTA reads more than a few: the last
            // CTA of each RUN to arrive leaves its run's sum in the place of the run's first part, and the last one of those adds the runs.
            const int parts = sg.f1 - sg.f0 + 1, mine = (int)blockIdx.x - sg.f0, runs = parts > 2 * RUN ? (parts + RUN - 1) / RUN : 1;
            float *wt = reinterpret_cast<float *>(smem + C::Q_BYTES);
            auto last_of = [&](unsigned int *ticket, int n) {
                __syncthreads();
                if (tid == 0) {   // releases what all of them stored before the barrier, and acquires the others' stores
                    unsigned int was;
                    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(was) : "l"(ticket) : "memory");
                    const bool last = was == (unsigned)(n - 1);
                    if (last) *ticket = 0u;
                    last_s = last;
                }
                __syncthreads();
                return last_s != 0;
            };
            if (runs == 1) {
                if (last_of(a.tickets + sg.f0, parts)) join<C>(a, seg_s[turn], wt, gate_s, 0, 1, parts, true);
            } else {
                const int run = mine / RUN, n = min(RUN, parts - run * RUN);
                if (last_of(a.tickets + MAX_CTAS_ALL * (run == 0 ? 1 : 2) + sg.f0 + run * RUN, n)) {
                    join<C>(a, seg_s[turn], wt, gate_s, run * RUN, 1, n, false);
                    if (last_of(a.tickets + sg.f0, runs)) join<C>(a, seg_s[turn], wt, gate_s, 0, RUN, runs, true);
                }
            }
        }
        if (tid == 0) {
            Walk w = walk_s;
            Seg nx;
            if (!paged::walk_next<C::TB>(a, pre, R, COST, w, nx)) nx.k0 = -1;
            walk_s = w;
            seg_s[turn ^ 1] = nx;
        }
        __syncthreads();
    }
}

// Rows per KV head up to which a sequence is this kernel's. Each 8 of them read the cache again (from L2); the kernel for many rows takes 128
// at once, and as long for one. All sequences alike (us, here / there; bf16, heads of 256 and in brackets of 128; f32 crosses over 8 to 16 rows later, so its borders lie higher):
//   64 sequences of 1200 keys   24 rows 88 117 (56 90)    40: 130 117 (80 89)     48: 150 119 (92 91)     64: 192 121 (117 90)
//   24 of 5000                  24 rows 103 134 (68 117)  40: 157 130 (99 111)    48: 182 132 (115 112)   64: 235 135 (146 112)
// Where a batch has rows on both sides, both kernels run, one behind the other, and neither fills the GPU: 24 sequences of 8 to 64 rows, 37 on average,
// heads of 128: 63 us here, 82 there, 85 with the border at 40. So what counts is where most of the work is, which the mean over the sequences says:
//   - under mean_many rows, few sequences have more, and one kernel for up to 128 rows is better than two: 60 sequences of 4 rows and 4 of 96, 1200
//     keys: 48 us, 91 with the border at 64 (heads of 128: 33 and 62); 4 of 128 among them 55 and 101; 48 sequences of 20000 keys, four of 128 rows: 307 and 247.
//   - from mean_many on, all but the smallest go to the other kernel: 40 to 64 rows, 52 on average, 5000 keys: 121 us, 166 with the border at 64; the
//     smallest stay: 63 sequences of 4 rows and one of 1024: 93, 108 all there. 16 sequences of 500 keys, 48 rows on average, lose (34 to 56).
// Over some 430 batches of 1 to 192 rows, 500 to 20000 keys, heads of 64, 128 and 256 this takes 1.05 times as long as the best border for each
// batch; 64 for all of them 1.13, 32 1.20. With few (sequence, KV head) pairs the other kernel's parts are many and small, and the border lies higher:
//   1 sequence of 16000 keys    128 rows 71 110 (47 64)   256: 123 114 (79 69)    512: 226 105 (143 68)
constexpr long long FEW_PAIRS = 8, NARROW_FEW = 256, NARROW_MOST = 128;
constexpr long long narrow_least(bool f32) { return f32 ? 48 : 32; }
constexpr long long mean_many(int hd, bool f32) { return hd == 256 ? (f32 ? 48 : 44) : 60; }   // rows per KV head of a sequence
constexpr size_t TICKETS = 3 * MAX_CTAS_ALL * sizeof(unsigned int);   // before the partials: three words per CTA
constexpr int MAX_CTAS = 3;                             // of an SM

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
    if (e == cudaSuccess) e = launch_pdl(attn_kernel<C>, dim3(C::CTAS * sm_count()), dim3(C::THREADS), C::SMEM, s, a);
    return e == cudaSuccess ? 0 : cuda_fail(who, e);
}

template <typename T>
int launch(const AttnParams &a, cudaStream_t s, const char *who) {
    return a.pool.hd == 256   ? launch_one<Cfg<T, 256, 4, 4, 2>>(a, s, who)
           : a.pool.hd == 128 ? launch_one<Cfg<T, 128, 4, 4, 3>>(a, s, who)
                              : launch_one<Cfg<T, 64, 4, 4, 3>>(a, s, who);
}

}  // namespace
}  // namespace paged4
}  // namespace spk

extern "C" {

size_t spk_paged4_attn_workspace_bytes(int head_dim) {
    using namespace spk::paged4;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
    const size_t narrow = (size_t)MAX_CTAS * part_floats(R, head_dim), wide = part_floats(WIDE_R, head_dim);
    return TICKETS + (size_t)spk::sm_count() * 2 * (narrow > wide ? narrow : wide) * sizeof(float);
}

int spk_paged4_attn(const spk_kv4_pool *pool, const spk_kv_batch *batch, const spk_paged4_attn_args *p, void *stream) {
    using namespace spk;
    using namespace spk::paged4;
    const char *who = "spk_paged4_attn";
    if (check_pool(pool, who) || paged::check_batch(batch, who)) return -1;
    if (!p) return set_error("%s: null arguments", who);
    if (p->type < T_F32 || p->type > T_BF16) return set_error("%s: type %d (0 f32, 1 f16, 2 bf16)", who, p->type);
    if (p->heads < 1 || p->heads % pool->kv_heads) return set_error("%s: %d heads over %d KV heads", who, p->heads, pool->kv_heads);
    if (p->window < 0) return set_error("%s: window %d", who, p->window);
    if (batch->rows == 0) return 0;
    if (!p->q || !p->out || !p->workspace) return set_error("%s: null buffer", who);
    const long long width = (long long)p->heads * pool->head_dim;
    if (batch->rows > 1 && (p->ldq < width || p->ldout < width || (p->gate && p->ldgate < p->heads)))
        return set_error("%s: row strides %lld, %lld, %lld", who, p->ldq, p->ldout, p->ldgate);
    const int size = p->type == T_F32 ? 4 : 2;
    if (((uintptr_t)p->q | (uintptr_t)p->out | (uintptr_t)p->gate) % size) return set_error("%s: unaligned rows", who);
    if ((uintptr_t)p->workspace % 16) return set_error("%s: the workspace is not 16-byte aligned", who);
    if (sm_count() * MAX_CTAS > MAX_CTAS_ALL) return set_error("%s: a device of %d SMs", who, sm_count());
    AttnParams a;
    a.pool = pool_of(pool);
    a.b = paged::batch_of(batch);
    a.q = p->q;
    a.gate = p->gate;
    a.out = p->out;
    a.ldq = p->ldq;
    a.ldgate = p->ldgate;
    a.ldout = p->ldout;
    a.heads = p->heads;
    a.group = p->heads / pool->kv_heads;
    a.window = p->window;
    a.scale = (p->scale != 0.f ? p->scale : 1.0f / sqrtf((float)pool->head_dim)) * LOG2E;
    a.tickets = (unsigned int *)p->workspace;
    a.part = (float *)((uint8_t *)p->workspace + TICKETS);
    a.err = device_error_ptr();
    const cudaStream_t s = (cudaStream_t)stream;
    const bool few = (long long)batch->nseq * pool->kv_heads <= FEW_PAIRS;
    const bool f32 = p->type == T_F32;
    const long long narrow = few ? NARROW_FEW : (long long)batch->rows * a.group / batch->nseq < mean_many(pool->head_dim, f32) ? NARROW_MOST : narrow_least(f32);
    // the lines of work, at their longest: every row tile as long as the page table and a tile's tokens (before()); here a sequence has
    // `narrow` rows at most
    const bool many = (long long)batch->rows * a.group > narrow;          // some sequence may have more
    const double tokens = (double)batch->max_pages * pool->page_tokens, pairs = pool->kv_heads;
    const double here = fmin((double)batch->rows * a.group / R, (double)batch->nseq * (narrow / R)) + batch->nseq;
    const double there = (double)batch->rows * a.group / WIDE_R + batch->nseq;
    auto line = [&](double tiles, int R_, int cost) { return tiles * ((tokens + R_ / a.group + 3 + tiles / 32768) / BLOCK + cost + 5) * pairs; };
    if (line(here, R, COST) > 2147483000.0 || (many && line(there, WIDE_R, WIDE_COST) > 2147483000.0))
        return set_error("%s: %d rows over up to %d pages of %d tokens are too much for one call", who, batch->rows, batch->max_pages, pool->page_tokens);
    if (many) {
        // Which sequences a kernel has is decided where row0 is read; the arguments only say how many rows there may be. One sequence that may have many
        // rows is the other kernel's, however few it has.
        const bool one = batch->nseq == 1;
        a.from = one ? 0 : narrow + 1;
        a.to = LLONG_MAX;
        const int rc = attn_wide(a, p->type, s, who);
        if (rc || one) return rc;
    }
    a.from = 0;
    a.to = narrow;
    return p->type == T_F32 ? launch<float>(a, s, who) : p->type == T_F16 ? launch<__half>(a, s, who) : launch<__nv_bfloat16>(a, s, who);
}

}  // extern "C"
