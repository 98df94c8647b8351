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
//   S[16][8 tokens] = Q K^T:  A = the tile's 8 query rows as f16 (rows 8..15: what f16 left of f32 rows), B = keys
//   O^T[16 dims][8]  += V^T P^T:  A = values, two tokens' codes of a dim side by side, B = the weights, which are the S
//                                 accumulators as they lie; f32 rows' weights are two f16 terms.
// The contraction's order is free, so a lane takes 16 (8) consecutive bytes of a token as its share of K.
// Queries stand on a power of two of their row (2^14 to 2^15 at the largest), weights are 2^(s - m) with the row's largest at
// 2^12 to 2^15: a reference m moves only when a score passes it by 15, and a weight is kept down to 2^-24, 2^-36 of the
// largest (half of it in its last bit). l adds the weights as they were rounded.
//
// Work split: paged_line.cuh's line of groups of 8 query rows. A CTA's warps take a group's blocks of 16 tokens in turn, each
// with a ring of its own that cp.async fills and a softmax of its own; they meet at the end of the group. Groups that
// several CTAs share leave (O, m, l) in the workspace, and the last CTA to arrive adds the parts in CTA order.
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
constexpr int COST = 8;                                 // a group's fixed cost in blocks

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
// n bytes of a copy of N (4, 8 or 16); the rest becomes 0
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void *src, int n) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}

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
    static constexpr int SMEM = Q_BYTES + (RING > MERGE ? RING : MERGE);
    static constexpr int TB = WARPS;                     // blocks of a tile of the line: one a warp
    static constexpr int WORDS = HD / 64;                // words of 8 dims in a lane's share of a token's values
};

template <typename C>
__global__ void __launch_bounds__(C::THREADS, C::CTAS) attn_kernel(const AttnParams a) {
    using T = typename C::T;
    constexpr int HD = C::HD, ROW = C::ROW, SROW = C::SROW, WARPS = C::WARPS, WORDS = C::WORDS;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t pre[MAX_SEQ + 1], wsum[WARPS];
    __shared__ float up_s[R], m_s[WARPS][R], l_s[WARPS][R], gate_s[R];
    __shared__ int pos_s[R];
    __shared__ Seg seg_s;
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
        seg_s.k0 = -1;
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
            if (paged::walk_next<C::TB>(a, pre, R, COST, w, first)) seg_s = first;
            walk_s = w;
        }
    __syncthreads();

    const int per = a.pool.page_tokens / BLOCK;
    while (true) {
        const Seg sg = seg_s;
        if (sg.k0 < 0) break;
        const int cols = sg.c1 - sg.c0 + 1;
        // blocks of this warp: first + WARPS i, i < count
        const int nblk = min(sg.nblk, sg.k1 * C::TB), first = sg.k0 * C::TB + warp, count = first < nblk ? (nblk - first + WARPS - 1) / WARPS : 0;
        const int *table = a.b.table + (size_t)sg.s * a.b.max_pages;
        // lane i has the page of block 32 c + i of the warp's
        auto pages = [&](int c) {
            const int i = 32 * c + lane;
            int page = 0;
            if (i < count) {
                page = __ldg(table + (sg.start / BLOCK + first + WARPS * i) / per);
                if (page < 0 || page >= a.pool.pages) {
                    if (a.err) atomicExch(a.err, DEV_BAD_INDEX);
                    page = -1;
                }
            }
            return page;
        };
        int pg = pages(0), pg_next = pages(1);
        auto fetch = [&](int i) {
            if (i < count) {
                const int page = __shfl_sync(0xffffffffu, pg, i & 31);
                if ((i & 31) == 31) {
                    pg = pg_next;
                    pg_next = pages(i / 32 + 2);
                }
                const int blk = first + WARPS * i, tok0 = sg.start + blk * BLOCK, in = (sg.start / BLOCK + blk) % per * BLOCK;
                const size_t at = row_index(a.pool, max(page, 0), sg.kvh, in);
                const uint32_t st = ring_u + (i % C::STAGES) * C::STAGE;
                // tokens that no row sees arrive as zeros
                auto live = [&](int tok) { return page >= 0 && tok0 + tok >= sg.see0 && tok0 + tok <= sg.p_hi; };
                constexpr int PIECES = ROW / 16;
#pragma unroll
                for (int x = lane; x < BLOCK * PIECES; x += 32) {
                    const int tok = x / PIECES, pc = x % PIECES;
                    const int kp = HD == 256 ? pc ^ 4 * (tok & 1) : pc;
                    const int slot = (tok >> 1 & 3) | (tok & 1) << 2 | (tok & 8), vp = HD == 256 ? pc ^ 2 * (slot & 3) : HD == 128 ? pc ^ (slot & 2) : pc;
                    const int n = live(tok) ? 16 : 0;
                    copy_async<16>(st + tok * ROW + 16 * kp, a.pool.k + (at + tok) * ROW + 16 * pc, n);
                    copy_async<16>(st + C::V_OFF + slot * ROW + 16 * vp, a.pool.v + (at + tok) * ROW + 16 * pc, n);
                }
                const int tok = lane & 15;
                copy_async<SROW>(st + (lane < 16 ? C::KS_OFF : C::VS_OFF) + tok * SROW, (lane < 16 ? a.pool.ks : a.pool.vs) + (at + tok) * SROW, live(tok) ? SROW : 0);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < C::STAGES - 1; i++) fetch(i);

        // the tile's queries, f16 on the row's own power of two, where the lanes' shares of A lie
        for (int r = warp; r < R; r += WARPS) {
            const int col = sg.c0 + r, tok = col / a.group, h = sg.kvh * a.group + col % a.group;
            const bool real = r < cols;
            float x[HD / 32], mx = 0.f;
            const T *src = (const T *)a.q + (long long)(sg.r0 + tok) * a.ldq + (long long)h * HD;
#pragma unroll
            for (int i = 0; i < HD / 32; i++) {
                x[i] = real ? to_f32<T>(src[lane + 32 * i]) : 0.f;
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
                __half *q = reinterpret_cast<__half *>(qs) + (((step * 32 + 4 * r + tt) * C::QREG + (C::TWO ? 2 * reg : reg)) * 2 + (d & 1));
                const __half hi = __float2half_rn(x[i] * f);
                *q = hi;
                if constexpr (C::TWO) q[2] = __float2half_rn(x[i] * f - __half2float(hi));
            }
            if (lane == 0) {
                up_s[r] = a.scale * __int_as_float((127 - e) << 23);
                pos_s[r] = real ? sg.pos0 + tok : -1;
                gate_s[r] = real && a.gate ? 1.0f / (1.0f + __expf(-to_f32<T>(((const T *)a.gate)[(long long)(sg.r0 + tok) * a.ldgate + h]))) : 1.0f;
            }
        }
        __syncthreads();

        const float up = up_s[g];
        const int pos = pos_s[g], low = a.window > 0 ? pos - a.window : -1;   // the row sees (low, pos]
        float acc[HD / 16][4], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 16; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[i][e] = 0.f;

        for (int i = 0; i < count; i++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
            __syncwarp();
            fetch(i + C::STAGES - 1);
            const uint8_t *st = ring + (i % C::STAGES) * C::STAGE;
            const int tok0 = sg.start + (first + WARPS * i) * BLOCK;
            // scores of tokens 0..7 (s[0], s[1]: tokens 2t, 2t + 1) and 8..15
            float s[4];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int tok = 8 * n + g;
                float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < (HD == 256 ? 2 : 1); h++) {
                    uint32_t w[4], sc[2];
                    if constexpr (HD == 64) {
                        const uint2 v = *reinterpret_cast<const uint2 *>(st + tok * ROW + 8 * t);
                        w[0] = v.x, w[1] = v.y, w[2] = w[3] = 0;
                        const uint32_t b = st[C::KS_OFF + tok * SROW + t];
                        sc[0] = sc[1] = b * 0x00800080u;
                    } else {
                        const uint4 v = *reinterpret_cast<const uint4 *>(st + tok * ROW + 16 * (HD == 256 ? (4 * h + t) ^ 4 * (tok & 1) : t));
                        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                        const uint32_t b = *reinterpret_cast<const uint16_t *>(st + C::KS_OFF + tok * SROW + 8 * h + 2 * t);
                        sc[0] = (b & 0xff) * 0x00800080u;
                        sc[1] = (b >> 8) * 0x00800080u;
                    }
#pragma unroll
                    for (int x = 0; x < (HD == 64 ? 2 : 4); x++) {
                        uint32_t k[4];
                        codes_f16(w[x], k);
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            const uint8_t *q = qs + ((8 * h + 2 * x + y) * 32 + lane) * C::QREG * 4;
                            const uint32_t b0 = hmul2(k[2 * y], sc[x >> 1]), b1 = hmul2(k[2 * y + 1], sc[x >> 1]);
                            if constexpr (C::TWO) {
                                const uint4 v = *reinterpret_cast<const uint4 *>(q);
                                mma(c, v.x, v.y, v.z, v.w, b0, b1);
                            } else {
                                const uint2 v = *reinterpret_cast<const uint2 *>(q);
                                mma(c, v.x, 0u, v.y, 0u, b0, b1);
                            }
                        }
                    }
                }
                s[2 * n] = (C::TWO ? c[0] + c[2] : c[0]) * up;
                s[2 * n + 1] = (C::TWO ? c[1] + c[3] : c[1]) * up;
            }
            // the lane's tokens of the values: 2t, 2t + 1, 2t + 8, 2t + 9
            uint32_t vs[4];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int tok = 2 * t + (x & 1) + 8 * (x >> 1);
                const uint8_t *at = st + C::VS_OFF + tok * SROW;
                vs[x] = HD == 256 ? *reinterpret_cast<const uint16_t *>(at + 2 * g) : HD == 128 ? at[g] : at[g >> 1];
                // what the row does not see
                const int p = tok0 + tok;
                if (p > pos || p <= low) s[x] = -INFINITY;
            }
            if (__any_sync(0xffffffffu, poisoned(vs[0] | vs[1] << 16) | poisoned(vs[2] | vs[3] << 16))) {
                uint32_t bad = 0;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    if (poisoned(vs[x])) {
                        bad |= 1u << x;
                        vs[x] = 0;
                    }
                }
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) bad |= __shfl_xor_sync(0xffffffffu, bad, o);
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int p = tok0 + 2 * t + (x & 1) + 8 * (x >> 1);
                    if ((bad >> x & 1) && p <= pos && p > low) s[x] = NAN;
                }
            }
            // a row's reference moves when one of its scores passes it by W_MAX
            const float most = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
            if (__any_sync(0xffffffffu, most > m + W_MAX)) {
                float x = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                const float was = m;
                if (x > m + W_MAX) m = x - W_TOP;
                const float f = was == -INFINITY ? 0.f : ex2(was - m);
                l *= f;
                const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
                for (int d = 0; d < HD / 16; d++) acc[d][0] *= f0, acc[d][1] *= f1, acc[d][2] *= f0, acc[d][3] *= f1;
            }
            const float ref = m == -INFINITY ? 0.f : m;
            float p[4];
#pragma unroll
            for (int x = 0; x < 4; x++) p[x] = ex2(s[x] - ref);
            const uint32_t p0 = pack_f16(p[0], p[1]), p1 = pack_f16(p[2], p[3]);
            uint32_t e0 = 0, e1 = 0;
            const float2 h0 = unpack_f16(p0), h1 = unpack_f16(p1);
            if constexpr (C::TWO) {
                e0 = pack_f16(p[0] - h0.x, p[1] - h0.y);
                e1 = pack_f16(p[2] - h1.x, p[3] - h1.y);
                l += (p[0] + p[1]) + (p[2] + p[3]);
            } else {
                l += (h0.x + h0.y) + (h1.x + h1.y);
            }
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
                    mma(acc[4 * y + x], a0, a1, a2, a3, p0, p1);
                    if constexpr (C::TWO) mma(acc[4 * y + x], a0, a1, a2, a3, e0, e1);
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        // the row's sum over its four lanes
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) {
            m_s[warp][g] = m;
            l_s[warp][g] = l;
        }
        __syncthreads();                                  // the rings are done with, too
        // columns 2t, 2t + 1 of acc on the CTA's common reference, into the warps' share of the rings
        float *mine = reinterpret_cast<float *>(smem + C::Q_BYTES) + warp * R * HD;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = 2 * t + e;
            float M = -INFINITY;
            for (int w = 0; w < WARPS; w++) M = fmaxf(M, m_s[w][r]);
            const float mw = m_s[warp][r], f = mw == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : ex2(mw - M);
#pragma unroll
            for (int d = 0; d < HD / 16; d += 2) {
                float4 v = make_float4(acc[d][e] * f, acc[d][2 + e] * f, acc[d + 1][e] * f, acc[d + 1][2 + e] * f);
                *reinterpret_cast<float4 *>(mine + r * HD + g * (HD / 8) + 2 * d) = v;
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
            }
            if (whole) {
                const float f = L == 0.f ? 0.f : gate_s[r] / L;
                const int col = sg.c0 + r;
                T *dst = (T *)a.out + (long long)(sg.r0 + col / a.group) * a.ldout + (long long)(sg.kvh * a.group + col % a.group) * HD + d;
                dst[0] = from_f32<T>(L == 0.f ? 0.f : o.x * f);
                dst[1] = from_f32<T>(L == 0.f ? 0.f : o.y * f);
                dst[2] = from_f32<T>(L == 0.f ? 0.f : o.z * f);
                dst[3] = from_f32<T>(L == 0.f ? 0.f : o.w * f);
            } else {
                *reinterpret_cast<float4 *>(slot + r * HD + d) = o;
                if (d == 0) {
                    slot[R * HD + r] = M;
                    slot[R * HD + R + r] = L;
                }
            }
        }
        if (!whole) {   // the last CTA of the group adds all parts in CTA order
            const int parts = sg.f1 - sg.f0 + 1;
            __syncthreads();
            if (tid == 0) {
                __threadfence();   // for all of them: their stores came before the barrier
                const bool last = atomicAdd(a.tickets + sg.f0, 1u) == (unsigned)(parts - 1);
                if (last) a.tickets[sg.f0] = 0u;
                __threadfence();
                last_s = last;
            }
            __syncthreads();
            if (last_s) {
                const size_t step = (size_t)2 * part_floats(R, HD);
                const float *p0 = a.part + (size_t)sg.f0 * step;   // CTA f0: slot 1, the others: slot 0
                auto part = [&](int p) { return p0 + p * step + (p == 0 ? part_floats(R, HD) : 0); };
                for (int x = tid; x < cols * (HD / 4); x += C::THREADS) {
                    const int r = x / (HD / 4), d = 4 * (x % (HD / 4));
                    float M = -INFINITY, L = 0.f;
                    for (int p = 0; p < parts; p++) M = fmaxf(M, __ldcg(part(p) + R * HD + r));
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int p = 0; p < parts; p++) {
                        const float mp = __ldcg(part(p) + R * HD + r), lp = __ldcg(part(p) + R * HD + R + r);
                        const float f = mp == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : ex2(mp - M);
                        const float4 v = __ldcg(reinterpret_cast<const float4 *>(part(p) + r * HD + d));
                        L = mp == -INFINITY ? L + lp : fmaf(lp, f, L);
                        o.x = fmaf(v.x, f, o.x), o.y = fmaf(v.y, f, o.y), o.z = fmaf(v.z, f, o.z), o.w = fmaf(v.w, f, o.w);
                    }
                    const float f = L == 0.f ? 0.f : gate_s[r] / L;
                    const int col = sg.c0 + r;
                    T *dst = (T *)a.out + (long long)(sg.r0 + col / a.group) * a.ldout + (long long)(sg.kvh * a.group + col % a.group) * HD + d;
                    dst[0] = from_f32<T>(L == 0.f ? 0.f : o.x * f);
                    dst[1] = from_f32<T>(L == 0.f ? 0.f : o.y * f);
                    dst[2] = from_f32<T>(L == 0.f ? 0.f : o.z * f);
                    dst[3] = from_f32<T>(L == 0.f ? 0.f : o.w * f);
                }
            }
        }
        if (tid == 0) {
            Walk w = walk_s;
            Seg nx;
            if (!paged::walk_next<C::TB>(a, pre, R, COST, w, nx)) nx.k0 = -1;
            walk_s = w;
            seg_s = nx;
        }
        __syncthreads();
    }
}

constexpr long long NARROW = 64;                       // rows per KV head up to which a sequence is this kernel's
constexpr size_t TICKETS = 4096;                        // bytes before the partials: one word per CTA
constexpr int MAX_CTAS = 3;                             // of an SM

template <typename C>
int launch_one(const AttnParams &a, cudaStream_t s, const char *who) {
    // the line of work, at its longest: every row tile as long as the page table and a tile's tokens (before())
    const long long tiles = (long long)a.b.rows * a.group / R + a.b.nseq;
    const long long blocks = ((long long)a.b.max_pages * a.pool.page_tokens + R / a.group + 3 + (tiles >> 15)) / BLOCK + COST + 4;
    if ((double)tiles * blocks * a.pool.kv_heads > 2147483000.0)
        return set_error("%s: %d rows over up to %d pages of %d tokens are too much for one call", who, a.b.rows, a.b.max_pages, a.pool.page_tokens);
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
    return a.pool.hd == 256   ? launch_one<Cfg<T, 256, 4, 3, 3>>(a, s, who)
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
    if ((size_t)sm_count() * MAX_CTAS * sizeof(unsigned int) > TICKETS) return set_error("%s: a device of %d SMs", who, sm_count());
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
    if ((long long)batch->rows * a.group > NARROW) {
        // some sequence may have many rows
        a.from = NARROW + 1;
        a.to = LLONG_MAX;
        const int rc = attn_wide(a, p->type, s, who);
        if (rc || batch->nseq == 1) return rc;
    }
    a.from = 0;
    a.to = NARROW;
    return p->type == T_F32 ? launch<float>(a, s, who) : p->type == T_F16 ? launch<__half>(a, s, who) : launch<__nv_bfloat16>(a, s, who);
}

}  // extern "C"
