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
#include <limits.h>

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
constexpr int COST = 32;                                // a group's fixed cost in blocks
constexpr int NONE = INT_MIN;                           // no page

template <typename T_, int HD_>
struct Cfg {
    using T = T_;
    static constexpr int HD = HD_;
    static constexpr bool TWO = sizeof(T) == 4;
    // log2 of the largest weight at a new reference: the further under W_MAX, the fewer moves, each of which takes a warp's outputs
    // through its registers; a weight is kept down to 2^-24 under it.
    static constexpr float TOP = TWO ? 10.0f : 6.0f;
    static constexpr int TILE = N * HD * 2;             // bytes of a tile's keys (or values) in f16
    static constexpr int CH = N * 128;                  // 64 dims of them
    static constexpr int V_OFF = 2 * TILE, Q_OFF = 4 * TILE;
    static constexpr size_t SMEM = Q_OFF + (TWO ? R * HD * 2 : 0) + 1024;
    static constexpr int PARTS = HD / 32;               // a thread's shares of a token
    static constexpr int UNITS = N * PARTS / (DQ_WARPS * 32);   // shares of a thread (0: half of the threads have one)
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
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {   // a in the low half
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// 8 values of a row
template <typename T>
__device__ __forceinline__ void row8(const T *p, bool vec, float *x) {
    if constexpr (sizeof(T) == 4) {
        if (vec) {
            const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
            return;
        }
    } else if (vec) {
        const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (__is_same(T, __half)) {
                const float2 f = unpack_f16(w[i]);
                x[2 * i] = f.x, x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = to_f32<T>(p[i]);
}

// What a softmax thread knows of its row
struct Row {
    float up, sig;                                      // factor of its scores, sigmoid of its gate
    int pos, low;                                       // it sees the tokens (low, pos]
    long long out;                                      // where its output lies (-1: no row)
};

template <typename C>
__global__ void __launch_bounds__(THREADS, 1) attn_kernel(const AttnParams a, const int qvec, const int ovec) {
    using T = typename C::T;
    constexpr int HD = C::HD;
    constexpr bool TWO = C::TWO;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_k[2], empty_k[2], full_v[2], empty_v[2], s_full[2], p_full[2], pv_done[2], q_full, o_full, o_free;
    __shared__ uint32_t pre[MAX_SEQ + 1], wsum[WARPS];
    __shared__ uint32_t bad[4][2];                      // tokens of a tile with poisoned values
    __shared__ Walk walk_s;
    __shared__ Seg seg_s;
    __shared__ int dead, last_s;
    __shared__ uint32_t tmem_s;
    uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(full_k + i, DQ_WARPS);
            mbar_init(full_v + i, DQ_WARPS);
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
    if (tid < 8) bad[tid >> 1][tid & 1] = 0;
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
    auto next = [&](Seg &g) {
        if (!walk_next<TB>(a, pre, R, COST, w, g)) g.k0 = -1;
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
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint64_t b = desc(kb + i * C::TILE + (k / 4) * C::CH + (k % 4) * 32, 0);
                    mma_ts(d, tmem + C::QC + 8 * k, b, id_s, k > 0);
                    if constexpr (TWO) mma_ss(d, desc(qb + (k / 4) * QCH + (k % 4) * 32, 0), b, id_s, true);
                }
                mma_commit(empty_k + i);
                mma_commit(s_full + i);
            }
            __syncwarp();
            kc++;
        };
        for (; sg.k0 >= 0; next(sg)) {
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
                        mma_ts(tmem, tmem + C::SC + i * N + 8 * k, b, id_o, j > 0 || k > 0);
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
        // codes to f16. Thread: token `tok` of a tile, 32 dims `part` (and `part` + 4 at heads of 256)
        const int dt = tid - SM_WARPS * 32, tok = dt % N, part = dt / N, per = a.pool.page_tokens / BLOCK;
        constexpr int U = C::UNITS > 0 ? C::UNITS : 1;
        const bool idle = part >= C::PARTS;
        uint32_t kc = 0, vc = 0;
        for (; sg.k0 >= 0; next(sg)) {
            const int n = tiles_of(sg);
            const int *table = a.b.table + (size_t)sg.s * a.b.max_pages;
            // the page of the thread's token of tile j, as the table has it; NONE where no row sees the token
            auto page_of = [&](int j) {
                const int blk = (sg.k0 + j) * TB + tok / BLOCK, at = sg.start + (sg.k0 + j) * N + tok;
                return j >= n || blk >= sg.nblk || at < sg.see0 || at > sg.p_hi ? NONE : __ldg(table + (sg.start / BLOCK + blk) / per);
            };
            auto row_of = [&](int page, int j) {
                const int blk = sg.start / BLOCK + (sg.k0 + j) * TB + tok / BLOCK;
                return row_index(a.pool, page, sg.kvh, blk % per * BLOCK + tok % BLOCK);
            };
            struct Raw {
                uint4 c[U];
                uint32_t s[U], vs[U];            // vs, beside keys: their tokens' scales of values, looked at for poison
            };
            auto load = [&](Raw &raw, bool keys, int page, int j) {
#pragma unroll
                for (int u = 0; u < U; u++) raw.c[u] = make_uint4(0, 0, 0, 0), raw.s[u] = raw.vs[u] = 0;
                const bool seen = page != NONE, there = page >= 0 && page < a.pool.pages;
                if (seen && !there && a.err) atomicExch(a.err, DEV_BAD_INDEX);
                if (there && !idle) {
                    const size_t at = row_of(page, j);
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const int x = part + 4 * u;
                        raw.c[u] = __ldg(reinterpret_cast<const uint4 *>((keys ? a.pool.k : a.pool.v) + at * (HD / 2)) + x);
                        raw.s[u] = __ldg(reinterpret_cast<const uint16_t *>((keys ? a.pool.ks : a.pool.vs) + at * (HD / GROUP)) + x);
                        if (keys) raw.vs[u] = __ldg(reinterpret_cast<const uint16_t *>(a.pool.vs + at * (HD / GROUP)) + x);
                    }
                }
            };
            auto convert = [&](const Raw &raw, uint8_t *to, bool keys) {
                if (idle) return;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int x = part + 4 * u;
                    uint32_t s2 = raw.s[u];
                    if (!keys) {   // poisoned values become 0: their tokens' weights say NaN where they are seen
                        if ((s2 & 0xff) >= POISON) s2 &= 0xff00;
                        if ((s2 >> 8) >= POISON) s2 &= 0x00ff;
                    }
                    const uint32_t sc[2] = {(s2 & 0xff) * 0x00800080u, (s2 >> 8) * 0x00800080u};
                    const uint32_t wd[4] = {raw.c[u].x, raw.c[u].y, raw.c[u].z, raw.c[u].w};
                    uint8_t *row = to + (x >> 1) * C::CH + tok * 128;
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        uint32_t h[4];
                        codes_f16(wd[y], h);
                        const uint4 v = make_uint4(hmul2(h[0], sc[y >> 1]), hmul2(h[1], sc[y >> 1]), hmul2(h[2], sc[y >> 1]), hmul2(h[3], sc[y >> 1]));
                        *reinterpret_cast<uint4 *>(row + ((((x & 1) * 4 + y) ^ (tok & 7)) << 4)) = v;
                    }
                }
            };
            if (n == 0) continue;
            // items: K0, K1, V0, K2, V1, .. V(n-1). Two are on their way while one is converted; a tile's page comes before them.
            int p0 = NONE, p1 = NONE, p2 = page_of(0);               // pages of the last keys' tile, the one before, the one behind
            auto load_item = [&](Raw &raw, int m) {
                if (m >= 2 * n) return;
                if (m == 0 || ((m & 1) && m < 2 * n - 1)) {      // keys of tile (m + 1) / 2
                    p1 = p0;
                    p0 = p2;
                    load(raw, true, p0, (m + 1) / 2);
                    p2 = page_of((m + 1) / 2 + 1);
                } else if (m == 2 * n - 1) {
                    load(raw, false, p0, n - 1);
                } else {
                    load(raw, false, p1, m / 2 - 1);
                }
            };
            auto item = [&](Raw &raw, int m) {
                const bool keys = m == 0 || ((m & 1) && m < 2 * n - 1);
                const uint32_t c = keys ? kc : vc, i = c & 1;
                if (c > 1) wait_for((keys ? empty_k : empty_v) + i, ((c >> 1) - 1) & 1, &dead, a.err);
                if (keys) {
                    uint32_t poison = 0;
#pragma unroll
                    for (int u = 0; u < U; u++) poison |= poisoned(raw.vs[u]);
                    if (poison) atomicOr(&bad[c & 3][tok >> 5], 1u << (tok & 31));
                }
                convert(raw, smem + (keys ? 0 : C::V_OFF) + i * C::TILE, keys);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive((keys ? full_k : full_v) + i);
                if (keys) kc++;
                else vc++;
                load_item(raw, m + 2);
            };
            Raw ra, rb;
            load_item(ra, 0);
            load_item(rb, 1);
            for (int m = 0; m < 2 * n; m += 2) {
                item(ra, m);
                item(rb, m + 1);
            }
        }
    } else {
        const int r = tid;
        const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);   // the warp's lanes of tensor memory
        __shared__ float sig_s[R];
        __shared__ long long out_s[R];
        uint32_t tc = 0, groups = 0;
        // the row of a group that is this thread's, its queries to where the MMAs read them
        auto queries = [&](const Seg &g) {
            Row row{0.f, 1.f, -1, -1, -1};
            if (g.k0 < 0) return row;
            const int col = g.c0 + r, tok = col / a.group, h = g.kvh * a.group + col % a.group;
            const bool real = col <= g.c1;
            const T *src = (const T *)a.q + (long long)(g.r0 + tok) * a.ldq + (long long)h * HD;
            if (real) {
                row.pos = g.pos0 + tok;
                row.low = a.window > 0 ? row.pos - a.window : -1;
                row.out = (long long)(g.r0 + tok) * a.ldout + (long long)h * HD;
                if (a.gate) row.sig = 1.0f / (1.0f + __expf(-to_f32<T>(((const T *)a.gate)[(long long)(g.r0 + tok) * a.ldgate + h])));
            }
            if (tiles_of(g) == 0) return row;
            float mx = 0.f;
            if (real)
#pragma unroll 4
                for (int d = 0; d < HD; d += 8) {
                    float x[8];
                    row8<T>(src + d, qvec, x);
#pragma unroll
                    for (int i = 0; i < 8; i++) mx = fmaxf(mx, fabsf(x[i]));
                }
            const int e = mx > 0.f && mx < INFINITY ? min(14 - ilogbf(mx), 126) : 0;   // 2^e brings the largest into [2^14, 2^15)
            const float f = __int_as_float((e + 127) << 23);
            row.up = a.scale * __int_as_float((127 - e) << 23);
#pragma unroll 2
            for (int c = 0; c < HD / 32; c++) {
                uint32_t hi[16];
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    float x[8];
                    if (real) row8<T>(src + 32 * c + 8 * y, qvec, x);
                    else {
#pragma unroll
                        for (int i = 0; i < 8; i++) x[i] = 0.f;
                    }
                    uint32_t lo[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float p = x[2 * i] * f, q = x[2 * i + 1] * f;
                        hi[4 * y + i] = pack_f16(p, q);
                        const float2 b = unpack_f16(hi[4 * y + i]);
                        lo[i] = pack_f16(p - b.x, q - b.y);
                    }
                    if constexpr (TWO)
                        *reinterpret_cast<uint4 *>(smem + C::Q_OFF + (c >> 1) * QCH + r * 128 + ((((c & 1) * 4 + y) ^ (r & 7)) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                __syncwarp();
                tm_st16(mine + C::QC + 16 * c, hi);
            }
            tm_wait_st();
            tc_before();
            if constexpr (TWO) fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full);
            return row;
        };
        Row row = queries(sg);
        while (sg.k0 >= 0) {
            const int n = tiles_of(sg);
            float m = -INFINITY, l0 = 0.f, l1 = 0.f;
            for (int j = 0; j < n; j++) {
                const uint32_t i = tc & 1;
                wait_for(s_full + i, (tc >> 1) & 1, &dead, a.err);
                __syncwarp();
                tc_after();
                const int t0 = sg.start + (sg.k0 + j) * N;
                const bool edge = __any_sync(0xffffffffu, t0 + N - 1 > row.pos || t0 <= row.low);
                const uint32_t b0 = *(volatile uint32_t *)&bad[tc & 3][0], b1 = *(volatile uint32_t *)&bad[tc & 3][1];   // tokens with poisoned values
                // 32 of the row's scores under a reference. They are read twice, for the largest and for the weights: 64 of
                // them do not fit the registers beside the rest.
                auto scores = [&](int c, float ref, float (&s)[32]) {
                    tm_ld32(mine + C::SC + i * N + 32 * c, s);
                    tm_wait_ld(s, 32);
                    const f32x2 up2 = pack2(row.up, row.up), ref2 = pack2(-ref, -ref);
#pragma unroll
                    for (int x = 0; x < 32; x += 2) {
                        const float2 v = unpack2(fma2(pack2(s[x], s[x + 1]), up2, ref2));
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
                };
                const float ref = m == -INFINITY ? 0.f : m;
                float mx = -INFINITY;
#pragma unroll
                for (int c = 0; c < N / 32; c++) {
                    float s[32], m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    scores(c, ref, s);
#pragma unroll
                    for (int x = 0; x < 32; x += 2) asm("max.f32 %0, %0, %1, %2;" : "+f"(m4[x / 2 & 3]) : "f"(s[x]), "f"(s[x + 1]));
                    mx = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
                }
                const bool move = mx > W_MAX || (m == -INFINITY && mx > -INFINITY);
                if (__any_sync(0xffffffffu, move)) {
                    const float delta = move ? mx - C::TOP : 0.f, f = m == -INFINITY ? 0.f : ex2(-delta);
                    if (move) m = ref + delta;
                    l0 *= f, l1 *= f;
                    if (j > 0) {   // what the outputs have so far, behind the products before
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
                    }
                }
                const float now = m == -INFINITY ? 0.f : m;
                uint32_t hi[N / 32][16], lo[N / 32][16];   // the weights lie where the scores were: f32's second terms wait for the last of those
#pragma unroll
                for (int c = 0; c < N / 32; c++) {
                    float s[32];
                    scores(c, now, s);
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        const float p = ex2(s[2 * x]), q = ex2(s[2 * x + 1]);
                        hi[c][x] = pack_f16(p, q);
                        if constexpr (__is_same(T, __nv_bfloat16)) l0 += p, l1 += q;   // f16's rounding is beneath bf16's
                        else {
                            const float2 b = unpack_f16(hi[c][x]);
                            if constexpr (TWO) {
                                lo[c][x] = pack_f16(p - b.x, q - b.y);
                                l0 += p, l1 += q;
                            } else {
                                l0 += b.x, l1 += b.y;
                            }
                        }
                    }
                    if constexpr (!TWO) tm_st16(mine + C::SC + i * N + 16 * c, hi[c]);
                }
                if constexpr (TWO) {
#pragma unroll
                    for (int c = 0; c < N / 32; c++) {
                        tm_st16(mine + C::SC + i * N + 16 * c, hi[c]);
                        tm_st16(mine + C::SC + i * N + N / 2 + 16 * c, lo[c]);
                    }
                }
                if (b0 | b1) {
                    bar_sync(1, SM_WARPS * 32);
                    if (tid < 2) bad[tc & 3][tid] = 0;
                    __syncwarp();
                }
                tm_wait_st();
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + i);
                tc++;
            }
            // the next group's queries, then this one's outputs
            Seg nx = sg;
            next(nx);
            const Row rn = queries(nx);
            const bool whole = sg.f0 == sg.f1, real = row.out >= 0;
            const float l = l0 + l1;
            float *slot = a.part + ((size_t)blockIdx.x * 2 + (sg.k0 == 0 ? 1 : 0)) * part_floats(R, HD);
            if (n > 0) {
                wait_for(&o_full, groups & 1, &dead, a.err);
                __syncwarp();
                tc_after();
            }
            const float f = !whole ? 1.0f : l == 0.f ? 0.f : row.sig / l;
#pragma unroll 1
            for (int c = 0; c < HD / 32; c++) {
                float o[32];
                __syncwarp();
                if (n > 0) {
                    tm_ld32(mine + 32 * c, o);
                    tm_wait_ld(o, 32);
                }
                if (!real) continue;
#pragma unroll
                for (int x = 0; x < 32; x++) o[x] = n == 0 || l == 0.f ? 0.f : o[x] * f;
                if (!whole) {
#pragma unroll
                    for (int x = 0; x < 32; x += 4) *reinterpret_cast<float4 *>(slot + (size_t)r * HD + 32 * c + x) = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
                } else {
                    T *dst = (T *)a.out + row.out + 32 * c;
                    if constexpr (sizeof(T) == 4) {
                        if (ovec) {
#pragma unroll
                            for (int x = 0; x < 32; x += 4) *reinterpret_cast<float4 *>(dst + x) = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
                            continue;
                        }
                    } else if (ovec) {
#pragma unroll
                        for (int x = 0; x < 32; x += 8) {
                            T v[8];
#pragma unroll
                            for (int y = 0; y < 8; y++) v[y] = from_f32<T>(o[x + y]);
                            *reinterpret_cast<uint4 *>(dst + x) = *reinterpret_cast<const uint4 *>(v);
                        }
                        continue;
                    }
#pragma unroll
                    for (int x = 0; x < 32; x++) dst[x] = from_f32<T>(o[x]);
                }
            }
            if (n > 0) {
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&o_free);
                groups++;
            }
            if (!whole) {   // the last CTA of the group adds all parts in CTA order
                const int parts = sg.f1 - sg.f0 + 1, rows = sg.c1 - sg.c0 + 1;
                if (real) {
                    slot[R * HD + r] = l == 0.f ? -INFINITY : m;
                    slot[R * HD + R + r] = l;
                }
                sig_s[r] = row.sig;
                out_s[r] = row.out;
                bar_sync(1, SM_WARPS * 32);
                if (tid == 0) {
                    __threadfence();   // for all of them: their stores came before the barrier
                    const bool last = atomicAdd(a.tickets + sg.f0, 1u) == (unsigned)(parts - 1);
                    if (last) a.tickets[sg.f0] = 0u;
                    __threadfence();
                    last_s = last;
                }
                bar_sync(1, SM_WARPS * 32);
                if (last_s) {
                    const size_t step = (size_t)2 * part_floats(R, HD);
                    const float *p0 = a.part + (size_t)sg.f0 * step;   // CTA f0: slot 1, the others: slot 0
                    auto part = [&](int p) { return p0 + p * step + (p == 0 ? part_floats(R, HD) : 0); };
                    for (int x = tid; x < rows * (HD / 4); x += SM_WARPS * 32) {
                        const int rr = x / (HD / 4), d = 4 * (x % (HD / 4));
                        float M = -INFINITY, L = 0.f;
                        for (int p = 0; p < parts; p++) M = fmaxf(M, __ldcg(part(p) + R * HD + rr));
                        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                        for (int p = 0; p < parts; p++) {
                            const float mp = __ldcg(part(p) + R * HD + rr), lp = __ldcg(part(p) + R * HD + R + rr);
                            const float fp = mp == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : ex2(mp - M);
                            const float4 v = __ldcg(reinterpret_cast<const float4 *>(part(p) + rr * HD + d));
                            L = mp == -INFINITY ? L + lp : fmaf(lp, fp, L);
                            o.x = fmaf(v.x, fp, o.x), o.y = fmaf(v.y, fp, o.y), o.z = fmaf(v.z, fp, o.z), o.w = fmaf(v.w, fp, o.w);
                        }
                        const float fo = L == 0.f ? 0.f : sig_s[rr] / L;
                        T *dst = (T *)a.out + out_s[rr] + d;
                        dst[0] = from_f32<T>(L == 0.f ? 0.f : o.x * fo);
                        dst[1] = from_f32<T>(L == 0.f ? 0.f : o.y * fo);
                        dst[2] = from_f32<T>(L == 0.f ? 0.f : o.z * fo);
                        dst[3] = from_f32<T>(L == 0.f ? 0.f : o.w * fo);
                    }
                }
                bar_sync(1, SM_WARPS * 32);   // sig_s, out_s and last_s are free again
            }
            sg = nx;
            row = rn;
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
