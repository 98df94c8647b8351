// paged_attn.cu — causal grouped-query attention of each sequence's new rows over its pages of the
// 8-bit cache, on the tcgen05 tensor cores: decode steps, verify batches and prompt chunks.
//
//   out[t][h] = sigmoid(gate[t][h]) * sum_j p_j V_j,  p = softmax_j(scale * rope(q[t][h]) . K_j),
//   j in [0, pos_t], with a window in (pos_t - window, pos_t]; K_j = dk[block of j] * k_j and
//   V_j = dv[block] * v_j with the cached e4m3 bytes k, v. A row that sees nothing gets 0.
//
// With w_j = exp(s_j) dv_j the value scale rides in the exponent: s'_j = s_j + log dv_j, one
// running reference m per row, O = sum exp(s'_j - m) v_j and l = sum exp(s'_j - m) / dv_j, so the
// largest term of O's sum is what the weights are relative to, whatever the scales are.
//
// The cache is read as it lies. Keys (and values) are the A operand, 128 tokens (128 dims) tall,
// e4m3 straight from the bulk copies; the query rows are the N columns of the B operand, and what
// 8 bits lack is made up in columns: a number x is the sum of T e4m3 terms, x = t0 + t1 / 32 +
// t2 / 1024 .., each term the rounding of what the ones before left (4 bits and a sign a term), and
// each term has a column of its own, so that it keeps its own scale:
//   S^T[128 keys][term, row]  = K . q^T     scores: sum of a row's TQ columns
//   O^T[hd][term, row]       += V^T . P^T   weights split the same way, TP bytes a row
// Products of e4m3 pairs are exact and are added in f32. A number near the largest keeps about
// 4.6 bits a term: two terms hold a bf16 query (8 bits), three an f16 one, five an f32 one.
//
// Weights need range, too: a row's keys may share what one key leaves them, 2^-17 of it each in a cache of 131072.
// What the last term cannot hold is lost, and it is lost from O alone. Its smallest byte is 2^-9 under the terms'
// steps (32 each, LAST before the last), and a row's largest weight stands at 2^6 to 2^8, so n keys
// lose at most n times these shares of the row's sum:
//   bf16 three terms 2^-10 / (32 x 128) / 2^6 = 2^-28;  f16 four 2^-32 (2^-31, the weights are taken by f16);  f32 five 2^-37
// which at 131072 keys is a quarter of half a unit of bf16 and of f16. (Two terms, 2^-21, lose whole contexts:
// behind a first token of value 0 with nine tenths of the weight, a third of 32768 others' sum was gone.)
//
// What bounds it: for few rows the cached bytes, read once per KV head (an MMA of 16 columns costs
// what its A bytes cost to read from shared memory, and the softmax runs on keys x rows alone); for
// prompt chunks the softmax's instructions, 48 or 64 bf16 rows against each 128 keys. Measured, heads of 256, 4 a KV
// head: one f32 row over 131072 keys 63 us (269 MB, 4.3 TB/s; some 20 us are start, queries and joining);
// 64 bf16 rows of as many sequences of up to 9000 keys 43 us (86 MB; a change of group costs as much as several
// tiles); 2048 rows behind 6144 cached ones: bf16 570 us (240 GFLOP, 0.42 PFLOP/s; the tensor pipe is busy a quarter
// of the time, the issue slots half of it), f16 750, f32 1030.
//
// Work split: all (sequence, KV head, row tile) groups stand in one line, each as long as the
// tokens it reads plus COST for its fixed cost; the line is cut into equal ranges, one per CTA,
// one CTA per SM. A 128-token tile belongs to the CTA in whose range its first token falls. A group
// that several CTAs share leaves (O, m, l) in the workspace; the last CTA to arrive (a ticket that it
// resets) adds the parts in CTA order.
//
// Warps: 0 the groups and the copies of keys and scales, 1 MMA issue, 2 the copies of values, 3-6 the
// queries of the next group (of the first one with the others' help), 7.. softmax:
// a thread per key, and per output dim at the end of a group.
#include "paged_line.cuh"
#include "paged_tc.cuh"

namespace spk {
namespace paged {
namespace {

constexpr float M_NONE = -INFINITY;   // reference of a part that has seen nothing
// Weights are 2^(s' - m): a new reference sits W_TOP below the largest score, so weights start at 64, and
// it moves only when a score passes m + 8, so they end at 256 (e4m3 holds 448). More room above would cost
// the small ones (the terms' bytes end at 2^-9), less would move the reference more often.
constexpr float W_TOP = 6.0f, W_MAX = 8.0f;
constexpr float STEP = 32.0f;         // a term's scale over the one before: half an ulp of 256 is 8
constexpr float LOG2E = 1.4426950408889634f;
constexpr int TILE = 128, TB = TILE / BLOCK;   // keys of a tile, its blocks
constexpr int FIRST_Q = 3, Q_WARPS = 4;   // the warps of the queries
constexpr int SQ = 4;                 // groups known ahead

struct AttnParams {
    Pool pool;
    Batch b;
    const void *q, *gate;
    void *out;
    long long ldq, ldgate, ldout;
    int qvec;
    const float *freq;
    int pdim, heads, group, window;
    float scale;                      // softmax scale * log2(e)
    unsigned int *tickets;            // [gridDim.x], zero at rest
    float *part;                      // [gridDim.x][2][PART]
    int *err;
    __device__ __forceinline__ bool takes(long long) const { return true; }
};

// R rows a tile, queries of TQ terms, weights of TP. SG warpgroups share a tile's rows (wide tiles: more
// warps hide the softmax's latencies); PG sets of them take the groups in turn (narrow tiles: one
// set's last products and outputs run beside the next one's first scores).
template <int HD_, int R_, int TQ_, int TP_, int SG_, int PG_>
struct Cfg {
    static constexpr int HD = HD_, R = R_, TQ = TQ_, TP = TP_, SG = SG_, PG = PG_;
    static constexpr int CS = (TQ * R + 15) / 16 * 16, CO = (TP * R + 15) / 16 * 16;   // columns of scores, of outputs
    // a step of 64 loses nothing of the largest weights (what the terms before leave is at most 8, times the
    // step), one of 128 a bit of those past 128, which bf16 does not have
    static constexpr float LAST = TP == 3 ? 128.0f : 64.0f;
    // The tensor cores cut their f32 sums towards 0: n keys of values of one sign end up to n x 3.3e-10 short (131072:
    // 4.3e-5 of the sum), which f32 outputs would show. Theirs leave the tensor memory every 64 tiles (2.7e-6).
    static constexpr int RUN = TP >= 5 ? 64 : 0;
    static constexpr int RG = R / SG;                         // rows of a warpgroup, side by side
    static constexpr int CH = SG == 1 ? R : 8;                // rows handled together
    static constexpr int NC = RG / CH;
    static constexpr int LD = 8;                              // columns of a tensor-memory access
    // columns of a chunk: all, or CH a term
    static constexpr int LCS = SG == 1 ? (TQ * R + 7) / 8 * 8 : CH * TQ, LCO = SG == 1 ? (TP * R + 7) / 8 * 8 : CH * TP;
    static constexpr int KB = BLOCK * HD;                     // bytes of a block's keys (or values)
    static constexpr int SLOT = TB * KB;                      // a tile's keys (or values)
    // slots of keys and of values: a tile's keys are done with its scores, its values much later
    static constexpr int NK = SG > 1 ? (HD == 256 ? 2 : 4) : HD == 256 ? 3 : HD == 128 ? 6 : 8;
    static constexpr int NV = SG > 1 ? (HD == 256 ? 1 : 2) : NK;
    static constexpr int SCR = NK <= 4 ? 8 : 16;              // tiles whose scales are kept: the copies are up to NK + 3 ahead
    // P: 16 keys of every column, then the next 16, 64 bytes further than they need so that the byte
    // stores of a warp's two runs of 16 keys meet different banks.
    static constexpr int PK = CO * 16 + 64, PB = TILE / 16 * PK, NP = 2;
    static constexpr int HH = HD == 256 ? 2 : 1;              // 128-dim halves of the output
    static constexpr int TC = 2 * CS + HH * PG * CO, TCOLS = TC <= 64 ? 64 : TC <= 128 ? 128 : TC <= 256 ? 256 : 512;
    static constexpr int MW = 160 * (SG == 1 ? 1 : 4);        // weights that a merge of parts holds at once
    static constexpr size_t V_OFF = (size_t)NK * SLOT, Q_OFF = V_OFF + (size_t)NV * SLOT, P_OFF = Q_OFF + (size_t)2 * CS * HD;
    static constexpr size_t SMEM = P_OFF + (size_t)NP * PB;
    // a group's fixed cost in blocks: what evened out the CTAs' times over 64 sequences of 1 to 9000 tokens
    // (narrow: 8 40.3 us, 16 41.3, 32 41.5, 64 46.8) and 24 of 8 rows each (wide: 8 41 us, 16 36, 32 32, 64 37)
    static constexpr int COST = PG == 1 ? 32 : 16;
    static constexpr int LAG = PG == 1 ? 2 : 1;               // tiles that the values are behind the scores
    static constexpr int WARPS = FIRST_Q + Q_WARPS + 4 * SG * PG, THREADS = WARPS * 32;
    static constexpr int PART = (R * (HD + 2) + 3) / 4 * 4;   // floats of a partial: O, then m, then l; read 16 bytes at a time
    static_assert(TC <= 512 && R % SG == 0 && RG % CH == 0, "");
    // access x of chunk ch of warpgroup sg: its column
    static __device__ __forceinline__ int col(int sg, int ch, int x) { return SG == 1 ? 8 * x : x * R + sg * RG + ch * CH; }
    static constexpr int TS = SG == 1 ? R : CH;               // a chunk's terms lie this far apart
};

// ------------------------------------------------------------------ tensor cores
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {   // K-major, no swizzle
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc), "r"(0u)
        : "memory");
}
// K columns of this thread's lane; tm_wait before their use
template <int K>
__device__ __forceinline__ void tm_ld(uint32_t addr, float *v) {
    static_assert(K == 8, "");
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "r"(addr));
}
template <int K>
__device__ __forceinline__ void tm_st(uint32_t addr, const float *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"f"(v[0]), "f"(v[1]),
                 "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "r"(addr)
                 : "memory");
}
// The loads have landed; their registers pass through, so no use of them moves up.
template <int K>
__device__ __forceinline__ void tm_wait(float (&v)[K]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < K; i++) asm volatile("" : "+f"(v[i]));
}

// e4m3 pair (low byte a) and its values
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 e4m3x2_f32(uint32_t w) {
    return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3)));
}

// Two weights as TP e4m3 terms, a pair of bytes each. Up to four terms go by f16, whose 11 bits and 2^-24
// they hold.
template <typename C>
__device__ __forceinline__ void split(float a, float b, uint32_t (&w)[C::TP]) {
    constexpr int T = C::TP;
    if constexpr (T <= 4) {
        __half2 h = __floats2half2_rn(a, b);
#pragma unroll
        for (int t = 0; t < T; t++) {
            uint16_t x;
            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(x) : "r"(*reinterpret_cast<const uint32_t *>(&h)));
            w[t] = x;
            if (t + 1 < T) {
                uint32_t f;
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(f) : "h"(x));
                h = __hmul2(__hsub2(h, *reinterpret_cast<const __half2 *>(&f)), __float2half2_rn(t + 2 < T ? STEP : C::LAST));
            }
        }
    } else {
#pragma unroll
        for (int t = 0; t < T; t++) {
            w[t] = e4m3x2(a, b);
            if (t + 1 < T) {
                const float2 v = e4m3x2_f32(w[t]);
                a = (a - v.x) * (t + 2 < T ? STEP : C::LAST);
                b = (b - v.y) * (t + 2 < T ? STEP : C::LAST);
            }
        }
    }
}
__device__ __forceinline__ float warp_max(float x) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ bool bar_or(int id, int n, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %3, 0;\n\tbarrier.cta.red.or.pred q, %1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(id), "r"(n), "r"((uint32_t)x)
        : "memory");
    return r != 0;
}

// Not inlined: an SM fetches a call's instructions anew (about 100 KB), and a dozen copies of this one were 5 to
// 10 KB of them (64 sequences 41.5 -> 40.2 us, 24 x 8 drafted tokens 31.2 -> 30.4).
__device__ __noinline__ float2 turn_of(int pos, float freq) {
    float2 t;
    angle(pos, freq, t.x, t.y);
    return t;
}

template <typename T, typename C>
__global__ void __launch_bounds__(C::THREADS, 1) attn_kernel(const AttnParams a) {
    constexpr int HD = C::HD, CS = C::CS, CO = C::CO, TQ = C::TQ, TP = C::TP, R = C::R, NK = C::NK, NV = C::NV, QB = 2, NP = C::NP, SCR = C::SCR;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ uint64_t full_k[NK], empty_k[NK], full_v[NV], empty_v[NV], sc_full[SCR], p_full[2], pv_done[2], q_full[QB], q_empty[QB];
    // a set waits on barriers that only its own tiles move, or on ones that its tile's scores imply: a wait by
    // parity must not start more than a phase early or end more than one late
    __shared__ uint64_t s_full[C::PG][2];
    __shared__ uint64_t seg_full[SQ], seg_empty[SQ], o_full[C::PG];   // o_full: a group's sums are complete
    __shared__ Seg segs[SQ];                            // the CTA's groups, as warp 0 finds them; k0 < 0: no more
    __shared__ float4 scales[SCR][TB];                  // dk, log2 dv, 1 / dv of a tile's blocks
    __shared__ uint32_t pre[MAX_SEQ + 1], wsum[C::WARPS];
    __shared__ __align__(16) float q_up[4][(R + 3) / 4 * 4];   // score factors of a tile's rows: the softmax may be two behind
    __shared__ int dead;                                // a wait ran out: what follows no longer waits
    constexpr int G = C::SG * C::PG;
    __shared__ float red[G][4][C::RG];                  // per row: the warps' maxima, then their sums
    __shared__ __align__(16) float mref[G][(C::RG + 3) / 4 * 4];   // per row: -m, the reference
    __shared__ uint32_t moved[G][4];                    // the warps' chunks whose reference has to move
    __shared__ __align__(16) float fs[G][(C::RG + 3) / 4 * 4];     // per row: a factor for all of its outputs
    __shared__ int pos_s[C::PG][R];                     // per row: position, -1 past the tile's last row
    __shared__ size_t out_s[C::PG][R];                  // per row: where its output lies
    __shared__ float merge_s[C::PG][2 * C::MW];         // a row's weights of the parts, and their sums before
    __shared__ int last_in[C::PG];
    __shared__ uint32_t tmem_s;
    __shared__ Walk walk_s;                             // the walk behind the CTA's first group
    uint8_t *qs = smem + C::Q_OFF, *ps = smem + C::P_OFF;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    if (tid == 0) {
        for (int i = 0; i < NK; i++) {
            mbar_init(full_k + i, 1);
            mbar_init(empty_k + i, 1);
        }
        for (int i = 0; i < NV; i++) {
            mbar_init(full_v + i, 1);
            mbar_init(empty_v + i, 1);
        }
        for (int i = 0; i < SCR; i++) mbar_init(sc_full + i, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(p_full + i, 4 * C::SG);
            mbar_init(pv_done + i, 1);
        }
        for (int i = 0; i < QB; i++) {
            mbar_init(q_full + i, Q_WARPS);
            mbar_init(q_empty + i, 1);
        }
        for (int i = 0; i < C::PG; i++) {
            mbar_init(&s_full[i][0], 1);
            mbar_init(&s_full[i][1], 1);
            mbar_init(o_full + i, 1);
        }
        for (int i = 0; i < SQ; i++) {
            mbar_init(seg_full + i, 1);
            mbar_init(seg_empty + i, 2 + Q_WARPS + 4 * C::SG * C::PG);
        }
        dead = 0;
        segs[0].k0 = -1;
        fence_mbar_init();
    }
    if (warp == 1) {   // this warp owns the tensor memory
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)),
                     "r"((uint32_t)C::TCOLS)
                     : "memory");
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
    for (int s0 = 0; s0 < a.b.nseq; s0 += C::THREADS) {
        const int s = s0 + tid;
        uint32_t u = 0;
        if (s < a.b.nseq) {
            const Seq q = seq_of(a, s, R);
            u = before(q, q.tiles, C::COST) * a.pool.kv_heads;
        }
        uint32_t x = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) wsum[warp] = x;
        __syncthreads();
        uint32_t add = base, all = base;
        for (int w = 0; w < C::WARPS; w++) {
            if (w < warp) add += wsum[w];
            all += wsum[w];
        }
        if (s < a.b.nseq) pre[s] = add + x - u;
        base = all;
        __syncthreads();
    }
    if (tid == 0) pre[a.b.nseq] = base;
    __syncthreads();

    // the CTA's range; the thread of the sequence where it starts finds its first group for all
    const uint32_t chunk = max((base + gridDim.x - 1) / gridDim.x, (uint32_t)TB), x0 = chunk * blockIdx.x;
    for (int s = tid; s < a.b.nseq; s += C::THREADS)
        if (pre[s] <= x0 && x0 < pre[s + 1]) {
            Walk w;
            w.chunk = chunk;
            w.x0 = x0;
            w.x1 = min(base, x0 + chunk);
            walk_at(a, pre, s, R, C::COST, w);
            Seg g;
            if (walk_next<TB>(a, pre, R, C::COST, w, g)) segs[0] = g;
            walk_s = w;
        }
    __syncthreads();
    // group n of the CTA, for the warps that follow warp 0; false: there is none. A dead CTA walks on.
    auto group = [&](uint32_t n, Seg &g) {
        if (n > 0 && !wait_for(seg_full + n % SQ, (n / SQ) & 1, nullptr, a.err)) return false;
        g = segs[n % SQ];
        __syncwarp();
        if (lane == 0) mbar_arrive(seg_empty + n % SQ);
        return g.k0 >= 0;
    };
    // the tiles of a group for a warp that copies: lane l < 8 has block l, whose page comes two tiles ahead, so
    // that its place is known a tile ahead
    const int per = a.pool.page_tokens / BLOCK;
    auto copy_group = [&](const Seg &g, auto &&tile) {
        const int blk0 = g.start / BLOCK, nblk = g.nblk, k1 = g.k1, kvh = g.kvh;
        const int *table = a.b.table + (size_t)g.s * a.b.max_pages;
        auto page_of = [&](int k) {
            int page = 0;
            if (k < k1 && lane < min(TB, nblk - k * TB)) {
                page = __ldg(table + (blk0 + k * TB + lane) / per);
                if (page < 0 || page >= a.pool.pages) {
                    if (a.err) atomicExch(a.err, DEV_BAD_INDEX);
                    page = 0;
                }
            }
            return page;
        };
        auto place_of = [&](int page, int k) { return block_index(a.pool, page, kvh, (blk0 + k * TB + lane) % per); };
        int page = page_of(g.k0), ahead = page_of(g.k0 + 1);
        size_t bi = place_of(page, g.k0);
        for (int k = g.k0; k < k1 && nblk > 0; k++) {
            const size_t next = place_of(ahead, k + 1);
            ahead = page_of(k + 2);
            tile(min(TB, nblk - k * TB), bi, k == g.k0, k + 1 < k1 ? min(TB, nblk - (k + 1) * TB) : 0, next);
            bi = next;
        }
    };
    Seg g;
    if (segs[0].k0 < 0) {
    } else if (warp == 0) {   // ------------------------------------------------------ groups, keys, scales
        uint32_t i = 0;
        Walk w = walk_s;
        g = segs[0];
        if (lane == 0) mbar_arrive(seg_full);   // group 0 is there
        for (uint32_t n = 1; g.k0 >= 0; n++) {
            Seg nx;
            if (!walk_next<TB>(a, pre, R, C::COST, w, nx)) nx.k0 = -1;
            if (n >= SQ) wait_for(seg_empty + n % SQ, ((n / SQ) - 1) & 1, nullptr, a.err);
            __syncwarp();
            if (lane == 0) {
                segs[n % SQ] = nx;
                mbar_arrive(seg_full + n % SQ);
            }
            float2 ahead = make_float2(0.f, 1.f);   // the next tile's scales, on their way
            copy_group(g, [&](int nb, size_t bi, bool first, int nb1, size_t bi1) {
                float2 sc = ahead;
                if (first && lane < nb) sc = make_float2(__ldg(a.pool.ks + bi), __ldg(a.pool.vs + bi));
                if (lane < nb1) ahead = make_float2(__ldg(a.pool.ks + bi1), __ldg(a.pool.vs + bi1));
                if (i < NK || wait_for(empty_k + i % NK, ((i / NK) - 1) & 1, &dead, a.err)) {
                    if (lane == 0) mbar_arrive_expect_tx(full_k + i % NK, nb * C::KB);
                    __syncwarp();
                    if (lane < nb)
                        bulk_g2s(smem + (size_t)(i % NK) * C::SLOT + lane * C::KB, a.pool.k + bi * C::KB, C::KB, full_k + i % NK);
                }
                if (lane < TB) scales[i % SCR][lane] = make_float4(sc.x, log2f(sc.y), 1.0f / sc.y, 0.f);
                __syncwarp();
                if (lane == 0) mbar_arrive(sc_full + i % SCR);
                i++;
            });
            g = nx;
        }
        if (*(volatile int *)&dead)   // copies in flight land before the CTA's memory goes
            for (uint32_t x = i > NK ? i - NK : 0; x < i; x++)
                for (uint32_t y = 0; y < (1u << 20) && !mbar_try_wait(full_k + x % NK, (x / NK) & 1); y++) {}
    } else if (warp == 2) {   // ------------------------------------------------------ values
        uint32_t i = 0;
        for (uint32_t n = 0; group(n, g); n++)
            copy_group(g, [&](int nb, size_t bi, bool, int, size_t) {
                uint64_t *full = full_v + i % NV;
                uint8_t *vd = smem + C::V_OFF + (size_t)(i % NV) * C::SLOT;
                if (i < NV || wait_for(empty_v + i % NV, ((i / NV) - 1) & 1, &dead, a.err)) {
                    if (nb & 1) {   // the MMAs take values by two blocks: the missing one is 0
                        for (int o = 16 * lane; o < C::KB; o += 512)
                            *reinterpret_cast<uint4 *>(vd + nb * C::KB + o) = make_uint4(0, 0, 0, 0);
                        fence_proxy_async();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive_expect_tx(full, nb * C::KB);
                    __syncwarp();
                    if (lane < nb) bulk_g2s(vd + lane * C::KB, a.pool.v + bi * C::KB, C::KB, full);
                }
                i++;
            });
        if (*(volatile int *)&dead)
            for (uint32_t x = i > NV ? i - NV : 0; x < i; x++)
                for (uint32_t y = 0; y < (1u << 20) && !mbar_try_wait(full_v + x % NV, (x / NV) & 1); y++) {}
    } else if (warp == 1) {   // ------------------------------------------------------ MMAs
        // The whole warp walks and waits and one elected thread issues, so the walk's state and the descriptors
        // are the same in all its lanes (all of it in a branch of lane 0: 4 % more for a 2048-row chunk).
        const bool one = elect_one();
        const uint32_t desc0 = (1u << 4) | ((128u >> 4) << 24);
        const uint32_t sdesc = desc0 | ((uint32_t)(CS >> 3) << 17), odesc = desc0 | ((uint32_t)(CO >> 3) << 17);
        const uint32_t so = __shfl_sync(0xffffffffu, tmem, 0), oo = so + 2 * CS;
        // descriptors move by their address field alone
        const uint64_t kdesc = smem_desc(smem_u32(smem), 128, 8 * HD);
        const uint64_t qdesc = smem_desc(smem_u32(qs), 128, 8 * HD);
        const uint64_t vdesc = smem_desc(smem_u32(smem) + (uint32_t)C::V_OFF, C::KB, 128);
        const uint64_t pdesc = smem_desc(smem_u32(ps), C::PK, 128);
        uint32_t i = 0, qi = 0;   // tiles whose scores were issued; groups with tiles
        uint32_t sets[C::PG] = {};   // tiles of each set
        // Up to LAG tiles' values are still to come. A wide tile's scores go before the values of the tile two
        // before it, into the buffer that its softmax has just left, so that the softmax finds them ready; a
        // narrow tile waits for memory, and its values leave their slot sooner. The oldest late tile is i - nlate.
        struct Late {
            int nb, po;           // its blocks, where its sums lie
            bool first, last;     // of its sums; of its group
        };
        Late l0 = {0, 0, false, false}, l1 = l0;   // the oldest, the one behind it
        int nlate = 0;
        auto weights = [&]() {    // of the oldest late tile: there
            const uint32_t t = i - nlate;
            const bool ok = wait_for(p_full + (t & 1), (t >> 1) & 1, &dead, a.err);
            tc_after();
            return ok;
        };
        auto values = [&](uint32_t t, bool ok) {   // of the oldest late tile, whose weights are there
            const Late l = l0;
            l0 = l1;
            nlate--;
            const uint32_t st = t % NV;
            if (!wait_for(full_v + st, (t / NV) & 1, &dead, a.err)) ok = false;
            __syncwarp();
            tc_after();
            if (one && ok) {
                const uint64_t vd = vdesc + st * (C::SLOT / 16), pd = pdesc + (t % NP) * (C::PB / 16);
#pragma unroll
                for (int kk = 0; kk < TB / 2; kk++)
                    if (2 * kk < l.nb)
#pragma unroll
                        for (int h = 0; h < C::HH; h++)
                            mma_e4m3(oo + (l.po + h) * CO, vd + (2 * kk * C::KB + h * 2048) / 16, pd + kk * (2 * C::PK / 16),
                                     odesc, !l.first || kk > 0);
                mma_commit(pv_done + (t & 1));
                if (l.last) mma_commit(o_full + l.po / C::HH);
                mma_commit(empty_v + st);
            }
            __syncwarp();
        };
        auto flush = [&]() {
            while (nlate) {
                const uint32_t t = i - nlate;
                values(t, weights());
            }
        };
        for (uint32_t n = 0;; n++) {
            // but not behind a group that is not there yet or has no tile: whoever is to make room for one
            // may be waiting for them
            if (n > 0 && !__all_sync(0xffffffffu, mbar_try_wait(seg_full + n % SQ, (n / SQ) & 1))) {
                flush();
                if (!wait_for(seg_full + n % SQ, (n / SQ) & 1, nullptr, a.err)) break;
            }
            __syncwarp();
            const int k0 = __shfl_sync(0xffffffffu, segs[n % SQ].k0, 0), k1 = __shfl_sync(0xffffffffu, segs[n % SQ].k1, 0);
            const int nblk = __shfl_sync(0xffffffffu, segs[n % SQ].nblk, 0);
            if (lane == 0) mbar_arrive(seg_empty + n % SQ);
            if (k0 < 0) break;
            if (nblk == 0) {
                flush();
                continue;
            }
            const uint32_t qb = qi % QB;
            if (!__all_sync(0xffffffffu, mbar_try_wait(q_full + qb, (qi / QB) & 1))) flush();
            const bool q_here = wait_for(q_full + qb, (qi / QB) & 1, &dead, a.err);
            for (int k = k0; k < k1; k++) {
                const uint32_t st = i % NK;
                const bool there = nlate < 2 || weights();   // with LAG 2: then its scores' buffer is free, too
                const bool ok = wait_for(full_k + st, (i / NK) & 1, &dead, a.err) && q_here;
                __syncwarp();
                tc_after();
                if (one && ok) {
                    const uint64_t kd = kdesc + st * (C::SLOT / 16), qd = qdesc + qb * (CS * HD / 16);
#pragma unroll
                    for (int kk = 0; kk < HD / 32; kk++)
                        mma_e4m3(so + (i & 1) * CS, kd + kk * 16, qd + kk * 16, sdesc, kk > 0);
#pragma unroll
                    for (int x = 0; x < C::PG; x++)
                        if (x == (int)(n % C::PG)) mma_commit(&s_full[x][sets[x] & 1]);
                    mma_commit(empty_k + st);
                    if (k + 1 == k1) mma_commit(q_empty + qb);
                }
                __syncwarp();
#pragma unroll
                for (int x = 0; x < C::PG; x++) sets[x] += x == (int)(n % C::PG);
                if (nlate == C::LAG) {
                    const uint32_t t = i - nlate;
                    values(t, C::LAG == 2 ? there : weights());
                }
                const bool fresh = C::RUN ? (k - k0) % (C::RUN ? C::RUN : 1) == 0 : k == k0;
                const Late l = {min(TB, nblk - k * TB), (int)(n % C::PG) * C::HH, fresh, k + 1 == k1};
                if (nlate == 0) l0 = l;
                else l1 = l;
                nlate++;
                i++;
            }
            qi++;
        }
        flush();
    } else if (warp >= FIRST_Q && (C::PG == 1 || warp < FIRST_Q + Q_WARPS)) {   // ---------- queries
        // a wide tile's first ones by all the warps that have nothing to do yet
        const int qw = warp - FIRST_Q;
        const bool keeps = qw < Q_WARPS;
        uint32_t qi = 0;
        for (uint32_t n = 0; n == 0 || keeps; n++) {
            if (keeps) {
                if (!group(n, g)) break;
            } else {
                g = segs[0];
            }
            if (g.nblk == 0) continue;
            const int helpers = C::PG == 1 && n == 0 ? C::WARPS - FIRST_Q : Q_WARPS, RW = (R + helpers - 1) / helpers;
            const int qb = qi % QB, c0 = g.c0, c1 = g.c1, pos0 = g.pos0;
            const T *q0 = (const T *)a.q + (size_t)g.r0 * a.ldq + (size_t)g.kvh * a.group * HD;
            // a warp takes RW rows side by side, RB at a time (they stay in registers where that is all)
            constexpr int RB = (R + Q_WARPS - 1) / Q_WARPS < 4 ? (R + Q_WARPS - 1) / Q_WARPS : 4;
            const int w0 = qw * RW;
            int d0, d1, turned = -1;
            unit_dims(lane, a.pdim, d0, d1);
            float cs[4], sn[4], fr[4];
            if (lane < a.pdim / 8)
#pragma unroll
                for (int e = 0; e < 4; e++) fr[e] = __ldg(a.freq + d0 + e);
            auto turn = [&](int tok) {   // the heads of a token share its angles
                if (lane < a.pdim / 8 && tok != turned) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float2 t = turn_of(pos0 + tok, fr[e]);
                        cs[e] = t.x, sn[e] = t.y;
                    }
                    turned = tok;
                }
            };
            Raw<T> raw[RB];
            auto load = [&](int r0) {
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    const int c = c0 + w0 + r0 + r;
                    if (r0 + r < RW && w0 + r0 + r < R && c <= c1 && lane < HD / 8)
                        raw[r].load(q0 + (size_t)(c / a.group) * a.ldq + (size_t)(c % a.group) * HD, d0, d1, a.qvec);
                    else raw[r].none();
                }
            };
            uint8_t *dst = qs + (size_t)qb * CS * HD;
#pragma unroll 1
            for (int r0 = 0; r0 < RW; r0 += RB) {
                load(r0);
                if (r0 == 0) {
                    turn((c0 + w0) / a.group);   // while the rows are on their way
                    if (qi >= QB) wait_for(q_empty + qb, ((qi / QB) - 1) & 1, &dead, a.err);
                }
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    const int row = w0 + r0 + r;
                    if (r0 + r >= RW || row >= R) continue;
                    float v[8], x[4], y[4], mx = 0.f;
                    raw[r].f32(v);
                    // times 2^(6 - e), e the exponent of the row's largest finite value, which then lies in [64, 128) (a
                    // row of nothing but values under 2^-120 lower); the rotation grows a pair by at most sqrt(2). A row's
                    // own scale: no other row decides how exactly it is held.
#pragma unroll
                    for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.f);
                    mx = warp_max(mx);
                    const uint32_t ex = min(max(__float_as_uint(mx) >> 23, 7u), 254u);
                    const float dn = __uint_as_float((260u - ex) << 23);
                    if (lane == 0) q_up[qi & 3][row] = __uint_as_float((ex - 6u) << 23) * a.scale;
#pragma unroll
                    for (int e = 0; e < 4; e++) {   // an infinity becomes a NaN, which e4m3 has
                        x[e] = fmaf(v[e], dn, v[e] - v[e]);
                        y[e] = fmaf(v[4 + e], dn, v[4 + e] - v[4 + e]);
                    }
                    turn((c0 + row) / a.group);
                    if (lane < a.pdim / 8) rotate_unit(x, y, cs, sn);
                    if (lane < HD / 8) {
#pragma unroll
                        for (int t = 0; t < TQ; t++) {
                            const int n = t * R + row;
                            uint8_t *col = dst + (n >> 3) * (8 * HD) + (n & 7) * 16;
                            const uint32_t x0 = e4m3x2(x[0], x[1]), x1 = e4m3x2(x[2], x[3]);
                            const uint32_t y0 = e4m3x2(y[0], y[1]), y1 = e4m3x2(y[2], y[3]);
                            *reinterpret_cast<uint32_t *>(col + (d0 >> 4) * 128 + (d0 & 15)) = x0 | (x1 << 16);
                            *reinterpret_cast<uint32_t *>(col + (d1 >> 4) * 128 + (d1 & 15)) = y0 | (y1 << 16);
                            if (t + 1 < TQ) {   // what is left, on the next term's scale
                                const float2 p0 = e4m3x2_f32(x0), p1 = e4m3x2_f32(x1), p2 = e4m3x2_f32(y0), p3 = e4m3x2_f32(y1);
                                x[0] = (x[0] - p0.x) * STEP, x[1] = (x[1] - p0.y) * STEP;
                                x[2] = (x[2] - p1.x) * STEP, x[3] = (x[3] - p1.y) * STEP;
                                y[0] = (y[0] - p2.x) * STEP, y[1] = (y[1] - p2.y) * STEP;
                                y[2] = (y[2] - p3.x) * STEP, y[3] = (y[3] - p3.y) * STEP;
                            }
                        }
                    }
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (helpers > Q_WARPS) bar_sync(5, helpers * 32);   // the helpers' rows are there, too
            if (keeps && lane == 0) mbar_arrive(q_full + qb);
            qi++;
        }
    }
    if (warp >= FIRST_Q + Q_WARPS && segs[0].k0 >= 0) {   // ------------------------------ softmax, outputs
        const int wg = (warp - FIRST_Q - Q_WARPS) >> 2, sg = wg % C::SG, pg = wg / C::SG;   // warpgroup: its rows, its turn
        const int q4 = warp & 3, key = 32 * q4 + lane, bid = 1 + wg;                 // the warp's lane quarter
        const uint32_t lane_at = (uint32_t)(32 * q4) << 16;
        // byte of this key in a column of P: values lie in the order of paged.cuh
        const int kbyte = (key >> 4) * C::PK + place(key & 15);
        constexpr int RG = C::RG, CH = C::CH, LCS = C::LCS, LCO = C::LCO, LD = C::LD, TS = C::TS;
        float *mr = mref[wg];
        uint32_t i = 0, qi = 0, mine_i = 0, own = 0;   // tiles and groups with tiles so far; those of this set
        for (uint32_t n = 0; group(n, g); n++) {
            const int k0 = g.k0, k1 = g.nblk > 0 ? g.k1 : k0, nblk = g.nblk, start = g.start;
            if ((int)(n % C::PG) != pg) {   // the other set's
                i += k1 - k0;
                qi += k1 > k0;
                continue;
            }
            const uint32_t otm = tmem + lane_at + 2 * CS + pg * C::HH * CO;   // the group's sums
            const int p_lo = g.p_lo, p_hi = g.p_hi, see0 = g.see0, window = a.window;
            const int row = sg * RG + key, c = g.c0 + row;   // the row that this thread keeps the books of
            const bool mine = key < RG && c <= g.c1;
            float sig = 1.0f;
            if (key < RG) {
                const int tok = c / a.group, hq = g.kvh * a.group + c % a.group;
                mr[key] = 0.f;
                pos_s[pg][row] = mine ? g.pos0 + tok : -1;
                out_s[pg][row] = (size_t)(g.r0 + tok) * a.ldout + (size_t)hq * HD;
                if (a.gate && mine) sig = to_f32(((const T *)a.gate)[(size_t)(g.r0 + tok) * a.ldgate + hq]);
            }
            float l[RG];
#pragma unroll
            for (int r = 0; r < RG; r++) l[r] = 0.f;
            float run[C::RUN ? C::HH * RG : 1];   // the outputs of the runs of tiles that are over
            bool runs = false;
            // chunk x of this thread's output dims: the terms' sums together
            auto sums = [&](int x, float (&o)[CH]) {
                const int h = x / C::NC, ch = x - h * C::NC;
                float v[LCO];
#pragma unroll
                for (int y = 0; y < LCO / LD; y++) tm_ld<LD>(otm + h * CO + C::col(sg, ch, y), v + LD * y);
                tm_wait(v);
#pragma unroll
                for (int r = 0; r < CH; r++) {
                    o[r] = v[(TP - 1) * TS + r];
#pragma unroll
                    for (int y = TP - 2; y >= 0; y--) o[r] = fmaf(o[r], 1.0f / (y == TP - 2 ? C::LAST : STEP), v[y * TS + r]);
                }
            };
            bar_sync(bid, 128);
            for (int k = k0; k < k1; k++, i++) {
                const int nb = min(TB, nblk - k * TB);
                wait_for(&s_full[pg][mine_i & 1], (mine_i >> 1) & 1, &dead, a.err);
                wait_for(sc_full + i % SCR, (i / SCR) & 1, &dead, a.err);
                mine_i++;
                __syncwarp();
                tc_after();
                const float4 sc = scales[i % SCR][key >> 4];
                const float fb = sc.y, isv = sc.z;
                const int j0 = start + k * TILE, j = j0 + key;
                const float *fq = q_up[qi & 3] + sg * RG;
                const bool edge = j0 + TILE - 1 > p_lo || (window > 0 && j0 <= p_hi - window);
                float t[RG];         // s' - m
#pragma unroll
                for (int ch = 0; ch < C::NC; ch++) {
                    float v[LCS];
#pragma unroll
                    for (int x = 0; x < LCS / LD; x++)
                        tm_ld<LD>(tmem + lane_at + (i & 1) * CS + C::col(sg, ch, x), v + LD * x);
                    tm_wait(v);
                    if constexpr (RG % 2 == 0) {
                        const f32x2 fa2 = pack2(sc.x, sc.x), fb2 = pack2(fb, fb), step2 = pack2(1.0f / STEP, 1.0f / STEP);
#pragma unroll
                        for (int r = 0; r < CH; r += 2) {
                            f32x2 u = pack2(v[(TQ - 1) * TS + r], v[(TQ - 1) * TS + r + 1]);
#pragma unroll
                            for (int x = TQ - 2; x >= 0; x--) u = fma2(u, step2, pack2(v[x * TS + r], v[x * TS + r + 1]));
                            const float2 f = *reinterpret_cast<const float2 *>(fq + ch * CH + r);
                            const float2 s = unpack2(fma2(u, mul2(fa2, pack2(f.x, f.y)), fb2));
                            t[ch * CH + r] = s.x;
                            t[ch * CH + r + 1] = s.y;
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < CH; r++) {
                            float u = v[(TQ - 1) * TS + r];
#pragma unroll
                            for (int x = TQ - 2; x >= 0; x--) u = fmaf(u, 1.0f / STEP, v[x * TS + r]);
                            t[ch * CH + r] = fmaf(u, sc.x * fq[ch * CH + r], fb);
                        }
                    }
                }
                if (edge) {
#pragma unroll
                    for (int r = 0; r < RG; r++) {
                        const int p = pos_s[pg][sg * RG + r];
                        if (j > p || (window > 0 && j <= p - window)) t[r] = -INFINITY;
                    }
                }
                uint32_t over = 0;   // chunks with a weight past 2^W_MAX
#pragma unroll
                for (int ch = 0; ch < C::NC; ch++) {
                    float mx = -INFINITY;
                    if constexpr (RG % 2 == 0) {   // the references are kept negated
#pragma unroll
                        for (int r = 0; r < CH; r += 2) {
                            const float2 n = *reinterpret_cast<const float2 *>(mr + ch * CH + r);
                            const float2 u = unpack2(add2(pack2(t[ch * CH + r], t[ch * CH + r + 1]), pack2(n.x, n.y)));
                            t[ch * CH + r] = u.x;
                            t[ch * CH + r + 1] = u.y;
                            mx = fmaxf(mx, fmaxf(u.x, u.y));
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < CH; r++) {
                            t[ch * CH + r] += mr[ch * CH + r];
                            mx = fmaxf(mx, t[ch * CH + r]);
                        }
                    }
                    over |= mx > W_MAX ? 1u << ch : 0u;
                }
                // the first tile sets the references (a row sees its earliest token there or in none of the
                // CTA's tiles); the answer is the same for the whole warpgroup
                const bool first = k == k0;
                if (bar_or(bid, 128, first || over != 0)) {
                    over = first ? (1u << C::NC) - 1u : __reduce_or_sync(0xffffffffu, over);
                    if (lane == 0) moved[wg][q4] = over;
#pragma unroll
                    for (int ch = 0; ch < C::NC; ch++)
                        if (over >> ch & 1u)   // the warp's largest; a chunk that only another warp flags moves with its own
#pragma unroll
                            for (int r = 0; r < CH; r++) {
                                const float x = warp_max(t[ch * CH + r]);
                                if (lane == 0) red[wg][q4][ch * CH + r] = x;
                            }
                        else if (lane == 0)
#pragma unroll
                            for (int r = 0; r < CH; r++) red[wg][q4][ch * CH + r] = -INFINITY;
                    bar_sync(bid, 128);
                    over = moved[wg][0] | moved[wg][1] | moved[wg][2] | moved[wg][3];
                    if (key < RG) {   // to W_TOP below the largest
                        const float x = fmaxf(fmaxf(red[wg][0][key], red[wg][1][key]), fmaxf(red[wg][2][key], red[wg][3][key]));
                        const float up = !first ? (x > W_MAX ? x - W_TOP : 0.f) : x == -INFINITY ? 0.f : x - W_TOP;
                        fs[wg][key] = up;
                        mr[key] -= up;
                    }
                    bar_sync(bid, 128);
#pragma unroll
                    for (int r = 0; r < RG; r++) {
                        const float up = fs[wg][r];
                        t[r] -= up;
                        if (!first) l[r] *= ex2(-up);
                    }
                    if (!first) {   // what is summed so far moves too, once its MMAs are done
                        wait_for(pv_done + ((i - 1) & 1), ((i - 1) >> 1) & 1, &dead, a.err);
                        __syncwarp();
                        tc_after();
#pragma unroll 1
                        for (int ch = 0; ch < C::NC; ch++) {
                            if (!(over >> ch & 1u)) continue;
#pragma unroll 1
                            for (int h = 0; h < C::HH; h++) {
                                float v[LCO];
#pragma unroll
                                for (int x = 0; x < LCO / LD; x++)
                                    tm_ld<LD>(otm + h * CO + C::col(sg, ch, x), v + LD * x);
                                tm_wait(v);
#pragma unroll
                                for (int r = 0; r < TS; r++) {
                                    const float f = ex2(-fs[wg][ch * CH + r]);
#pragma unroll
                                    for (int x = r; x < LCO; x += TS) v[x] *= f;
                                    if (C::RUN && runs && r < CH) run[h * RG + ch * CH + r] *= f;
                                }
#pragma unroll
                                for (int x = 0; x < LCO / LD; x++)
                                    tm_st<LD>(otm + h * CO + C::col(sg, ch, x), v + LD * x);
                            }
                        }
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                }
                if constexpr (C::RUN > 0)
                    if (k > k0 && (k - k0) % C::RUN == 0) {   // the next products start new sums
                        wait_for(pv_done + ((i - 1) & 1), ((i - 1) >> 1) & 1, &dead, a.err);
                        __syncwarp();
                        tc_after();
#pragma unroll 1
                        for (int x = 0; x < C::HH * C::NC; x++) {
                            float o[CH];
                            sums(x, o);
#pragma unroll
                            for (int r = 0; r < CH; r++) run[x * CH + r] = (runs ? run[x * CH + r] : 0.f) + o[r];
                        }
                        runs = true;
                    }
                if (i >= NP) wait_for(pv_done + ((i - NP) & 1), ((i - NP) >> 1) & 1, &dead, a.err);   // P's buffer is free
                uint8_t *pb = ps + (size_t)(i % NP) * C::PB + kbyte;
#pragma unroll
                for (int r = 0; r < RG; r += 2) {
                    float x[2] = {0.f, 0.f};
                    if (RG % 2 == 0 && !edge) {
                        x[0] = ex2(t[r]);
                        x[1] = ex2(t[r + 1]);
                        const float2 n = unpack2(fma2(pack2(x[0], x[1]), pack2(isv, isv), pack2(l[r], l[r + 1])));
                        l[r] = n.x;
                        l[r + 1] = n.y;
                    } else {
#pragma unroll
                        for (int e = 0; e < 2; e++)
                            if (r + e < RG) {
                                x[e] = ex2(t[r + e]);
                                if (!edge || t[r + e] != -INFINITY) l[r + e] = fmaf(x[e], isv, l[r + e]);
                            }
                    }
                    uint32_t b[TP];
                    split<C>(x[0], x[1], b);
#pragma unroll
                    for (int tt = 0; tt < TP; tt++) {
                        const int n = tt * R + sg * RG + r;
                        pb[n * 16] = (uint8_t)b[tt];
                        if (r + 1 < RG) pb[(n + 1) * 16] = (uint8_t)(b[tt] >> 8);
                    }
                }
                // values of tokens that no row sees, in a block that some are seen of: a masked place
                // never meets the product
                const int past = j0 + nb * BLOCK - 1 - p_hi, under = see0 - j0;
                if (past > 0 || under > 0) {
                    // one slot: its tile before has to be done with, or the wait reads a phase too early
                    if (NV == 1 && i > 0) wait_for(pv_done + ((i - 1) & 1), ((i - 1) >> 1) & 1, &dead, a.err);
                    wait_for(full_v + i % NV, (i / NV) & 1, &dead, a.err);
                    if (sg == 0) {
                        uint8_t *vb = smem + C::V_OFF + (size_t)(i % NV) * C::SLOT;
#pragma unroll 1
                        for (int e = 0; e < 2; e++) {
                            const int bad = e == 0 ? under : past, blk = e == 0 ? 0 : nb - 1;
                            if (bad <= 0) continue;
                            uint32_t keep[4];
#pragma unroll
                            for (int x = 0; x < 4; x++) {
                                keep[x] = 0;
#pragma unroll
                                for (int y = 0; y < 4; y++)
                                    if (e == 0 ? order(4 * x + y) >= bad : order(4 * x + y) < BLOCK - bad)
                                        keep[x] |= 0xffu << (8 * y);
                            }
#pragma unroll 1
                            for (int d = key; d < HD; d += 128) {
                                uint4 *at = reinterpret_cast<uint4 *>(vb + blk * C::KB + 16 * d);
                                uint4 u = *at;
                                u.x &= keep[0], u.y &= keep[1], u.z &= keep[2], u.w &= keep[3];
                                *at = u;
                            }
                        }
                    }
                }
                fence_proxy_async();
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + (i & 1));
            }
            if (k1 > k0) qi++;

            // the rows' sums over the keys, and the factor of a row's outputs
#pragma unroll
            for (int r = 0; r < RG; r++) {
                const float x = warp_sum(l[r]);
                if (lane == 0) red[wg][q4][r] = x;
            }
            bar_sync(bid, 128);
            const bool whole = g.f0 == g.f1;
            float *slot = a.part + ((size_t)blockIdx.x * 2 + (g.k0 == 0 ? 1 : 0)) * C::PART;
            sig = a.gate ? 1.0f + __expf(-sig) : 1.0f;   // 1 / sigmoid
            if (key < RG) {
                const float L = (red[wg][0][key] + red[wg][1][key]) + (red[wg][2][key] + red[wg][3][key]);
                // a row (or part) that saw nothing: its products are 0 or were not made
                fs[wg][key] = L == 0.f ? 0.f : whole ? 1.0f / (L * sig) : 1.0f;
                if (!whole && mine) {
                    slot[R * HD + row] = L == 0.f ? M_NONE : -mr[key];
                    slot[R * HD + R + row] = L;
                }
            }
            bar_sync(bid, 128);
            // not pv_done: the other set's tiles may have moved that on twice
            if (k1 > k0) wait_for(o_full + pg, own++ & 1, &dead, a.err);
            __syncwarp();
            tc_after();
            const int rows = g.c1 - g.c0 + 1;
#pragma unroll 1
            for (int x0 = 0; x0 < C::HH * C::NC; x0++) {
                const int h = x0 / C::NC, ch = x0 - h * C::NC, d = 128 * h + key;
                float os[CH];
                sums(x0, os);
#pragma unroll
                for (int r = 0; r < CH; r++) {
                    float o = os[r];
                    if (C::RUN && runs) o += run[x0 * CH + r];
                    const int rr = ch * CH + r, ro = sg * RG + rr;
                    const float f = fs[wg][rr];
                    if (d >= HD || ro >= rows) continue;
                    o = f == 0.f ? 0.f : o * f;
                    if (whole) ((T *)a.out)[out_s[pg][ro] + d] = from_f32<T>(o);
                    else slot[(size_t)ro * HD + d] = o;
                }
            }
            if (!whole) {   // the last CTA of the group adds all parts in CTA order
                const int parts = g.f1 - g.f0 + 1;
                constexpr int ST = 128 * C::SG;
                bar_sync(6 + pg, ST);
                if (sg == 0 && key == 0) {
                    __threadfence();   // for all of them: their stores came before the barrier
                    const bool last = atomicAdd(a.tickets + g.f0, 1u) == (unsigned)(parts - 1);
                    if (last) a.tickets[g.f0] = 0u;
                    __threadfence();
                    last_in[pg] = last;
                }
                bar_sync(6 + pg, ST);
                if (last_in[pg]) {
                    const size_t step = (size_t)2 * C::PART;
                    const float *p0 = a.part + (size_t)g.f0 * step;   // CTA f0: slot 1, the others: slot 0
                    auto part = [&](int p) { return p0 + p * step + (p == 0 ? C::PART : 0); };
                    float *wt = merge_s[pg], *wl = wt + C::MW;
                    const int RB = min(R, C::MW / parts);   // rows whose weights fit (at least one: 160 parts)
                    for (int r0 = 0; r0 < rows; r0 += RB) {
                        const int nr = min(RB, rows - r0);
                        if (key < RG && row >= r0 && row < r0 + nr) red[wg][0][key] = sig;
                        for (int x = sg * 128 + key; x < nr * parts; x += ST) {
                            const int p = x / nr, r = x - p * nr;
                            const float *pp = part(p) + R * HD + r0 + r;
                            wt[r * parts + p] = __ldcg(pp);
                            wl[r * parts + p] = __ldcg(pp + R);
                        }
                        bar_sync(6 + pg, ST);
                        for (int r = sg * 4 + q4; r < nr; r += 4 * C::SG) {   // a warp per row
                            float M = M_NONE, L = 0.f;
                            for (int p = lane; p < parts; p += 32) M = fmaxf(M, wt[r * parts + p]);
                            M = warp_max(M);
                            for (int p = lane; p < parts; p += 32) {
                                const float m = wt[r * parts + p], f = m == M_NONE ? 0.f : ex2(m - M);
                                wt[r * parts + p] = f;
                                L = fmaf(wl[r * parts + p], f, L);
                            }
                            L = warp_sum(L);
                            const float f = L == 0.f ? 0.f : 1.0f / (L * red[pg * C::SG + (r0 + r) / RG][0][(r0 + r) % RG]);
                            for (int p = lane; p < parts; p += 32) wt[r * parts + p] *= f;
                        }
                        bar_sync(6 + pg, ST);
                        const int items = nr * (HD / 4);
                        for (int x = sg * 128 + key; x < items; x += ST) {
                            const int r = x / (HD / 4), d = 4 * (x - r * (HD / 4));
                            const size_t at = (size_t)(r0 + r) * HD + d;
                            float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
                            for (int pb = 0; pb < parts; pb += 8) {
                                float4 v[8];
#pragma unroll
                                for (int p = 0; p < 8; p++)   // past the last part: the last one again, weight 0
                                    v[p] = __ldcg(reinterpret_cast<const float4 *>(part(min(pb + p, parts - 1)) + at));
#pragma unroll
                                for (int p = 0; p < 8; p++) {
                                    const float f = pb + p < parts ? wt[r * parts + pb + p] : 0.f;
                                    O.x = fmaf(v[p].x, f, O.x);
                                    O.y = fmaf(v[p].y, f, O.y);
                                    O.z = fmaf(v[p].z, f, O.z);
                                    O.w = fmaf(v[p].w, f, O.w);
                                }
                            }
                            T *dst = (T *)a.out + out_s[pg][r0 + r] + d;
                            dst[0] = from_f32<T>(O.x);
                            dst[1] = from_f32<T>(O.y);
                            dst[2] = from_f32<T>(O.z);
                            dst[3] = from_f32<T>(O.w);
                        }
                        bar_sync(6 + pg, ST);   // the weights and last_in are free again
                    }
                }
            }
            tc_before();
            bar_sync(bid, 128);   // the rows' books are free again
        }
    }
    tc_before();
    __syncthreads();
    if (warp == 1) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::TCOLS));
    }
}

constexpr size_t TICKETS = 1024;   // bytes before the partials: one word per CTA
constexpr int MAX_R = 64;

template <typename T, typename C>
int launch_one(const AttnParams &a, cudaStream_t s, const char *who) {
    // the line of work, at its longest: every row tile as long as the page table and a tile's tokens (before())
    const long long tiles = (long long)a.b.rows * a.group / C::R + a.b.nseq;
    const long long blocks = ((long long)a.b.max_pages * a.pool.page_tokens + C::R / a.group + 3 + (tiles >> 15)) / BLOCK + C::COST + 4;
    if ((double)tiles * blocks * a.pool.kv_heads > 2147483000.0)
        return set_error("%s: %d rows over up to %d pages of %d tokens are too much for one call", who, a.b.rows,
                         a.b.max_pages, a.pool.page_tokens);
    static bool set[64];
    int dev = 0;
    cudaGetDevice(&dev);
    cudaError_t e = cudaSuccess;
    if (dev < 0 || dev >= 64 || !set[dev]) {
        e = cudaFuncSetAttribute(attn_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
        if (e == cudaSuccess && dev >= 0 && dev < 64) set[dev] = true;
    }
    if (e == cudaSuccess) e = launch_pdl(attn_kernel<T, C>, dim3(sm_count()), dim3(C::THREADS), C::SMEM, s, a);
    return e == cudaSuccess ? 0 : cuda_fail(who, e);
}

// The columns follow the rows that a sequence has per KV head on average. A tile's cost grows with its
// columns and a second tile reads the cache again, from L2; where the one outweighs the other was measured
// (us; 64 sequences of 1200 keys, 8 of 6000, 1 of 16000; heads of 256, and of 128 in brackets):
//   f32   8 rows: 6 a tile 96 47 26 (78 38 24), 24 a tile 80 47 30 (66 35 25);  16: 138 62 31 (113 49 27), 84 50 35 (69 38 29)
//   f16   4 rows: 5 a tile 32 32 22, 8 a tile 33 32 22;  8: 81 45 25 (69 36 22), 50 33 28 (42 26 23);
//         24: 8 a tile 122 61 31 (103 48 26), 32 a tile 79 48 41 (69 38 35);  32: 157 74 35 (132 59 30), 81 50 46 (69 38 36)
//   bf16  4 rows: 5 a tile 31 32 22, 10 a tile 36 32 24;  8: 79 45 25 (69 36 22), 55 34 30 (47 28 24);
//         24: 10 a tile 135 63 34 (116 51 29), 32 a tile 76 47 40 (64 36 34);  32: 173 77 38 (151 63 33), 78 48 44 (64 36 35);
//         192: 32 a tile 348 150 63 (320 121 52), 48 (64) a tile 307 129 63 (243 106 56);  256: 456 190 74 (421 154 62),
//         453 174 72 (323 129 63);  1024, 8 and 1 sequences: 658 211 (561 178), 544 183 (426 145)
// so one long sequence of up to 24 rows sets the narrow tiles' end and 192 rows the widest ones' start.
// bf16 queries of 193 rows and more are of two terms, which is what bf16 itself holds: the scores' columns that this
// saves are the output's (heads of 256: 2 x 96 + 2 x 144 of 512, 48 rows a tile, and 40 at the most with three). A
// 2048-row chunk is off by 1.8e-3 of its output, and by 1.7e-3 from the rounding to bf16 alone.
template <typename T, int HD>
int launch(const AttnParams &a, cudaStream_t s, const char *who) {
    const long long per = ((long long)a.b.rows * a.group + a.b.nseq - 1) / a.b.nseq;
    if constexpr (sizeof(T) == 4) {
        if (per <= 12) return launch_one<T, Cfg<HD, 6, 5, 5, 1, 2>>(a, s, who);
        return launch_one<T, Cfg<HD, 24, 5, 5, 3, 1>>(a, s, who);
    } else {
        constexpr bool B = __is_same(T, __nv_bfloat16);
        if (per <= 5) return launch_one<T, Cfg<HD, 5, 3, B ? 3 : 4, 1, 2>>(a, s, who);
        if (per <= 24) return launch_one<T, Cfg<HD, B ? 10 : 8, 3, B ? 3 : 4, 1, 2>>(a, s, who);
        if constexpr (B)
            if (per > 192) return launch_one<T, Cfg<HD, HD == 256 ? 48 : 64, 2, 3, HD == 256 ? 3 : 4, 1>>(a, s, who);
        return launch_one<T, Cfg<HD, 32, 3, B ? 3 : 4, 4, 1>>(a, s, who);
    }
}

template <typename T>
int launch_hd(const AttnParams &a, cudaStream_t s, const char *who) {
    return a.pool.hd == 256   ? launch<T, 256>(a, s, who)
           : a.pool.hd == 128 ? launch<T, 128>(a, s, who)
                              : launch<T, 64>(a, s, who);
}

}  // namespace
}  // namespace paged
}  // namespace spk
extern "C" {

size_t spk_paged_attn_workspace_bytes(int head_dim) {
    using namespace spk::paged;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
    return TICKETS + (size_t)spk::sm_count() * 2 * MAX_R * (head_dim + 2) * sizeof(float);
}

int spk_paged_attn(const spk_kv_pool *pool, const spk_kv_batch *batch, const spk_paged_attn_args *p, void *stream) {
    using namespace spk;
    using namespace spk::paged;
    const char *who = "spk_paged_attn";
    if (check_pool(pool, who) || check_batch(batch, who)) return -1;
    if (!p) return set_error("%s: null arguments", who);
    if (p->type < T_F32 || p->type > T_BF16) return set_error("%s: type %d (0 f32, 1 f16, 2 bf16)", who, p->type);
    if (p->heads < 1 || p->heads % pool->kv_heads)
        return set_error("%s: %d heads over %d KV heads", who, p->heads, pool->kv_heads);
    if (p->pdim < 0 || p->pdim % 8 || p->pdim > pool->head_dim || (p->pdim > 0 && !p->freq) || (uintptr_t)p->freq % 4)
        return set_error("%s: pdim %d (a multiple of 8 up to head_dim, with its frequencies)", who, p->pdim);
    if (p->window < 0) return set_error("%s: window %d", who, p->window);
    if (batch->rows == 0) return 0;
    if (!p->q || !p->out || !p->workspace) return set_error("%s: null buffer", who);
    const long long width = (long long)p->heads * pool->head_dim;
    if (batch->rows > 1 && (p->ldq < width || p->ldout < width || (p->gate && p->ldgate < p->heads)))
        return set_error("%s: row strides %lld, %lld, %lld", who, p->ldq, p->ldout, p->ldgate);
    const int size = p->type == T_F32 ? 4 : 2;
    if ((uintptr_t)p->q % size || (uintptr_t)p->out % size || (uintptr_t)p->gate % size)
        return set_error("%s: unaligned rows", who);
    if ((uintptr_t)p->workspace % 16) return set_error("%s: the workspace is not 16-byte aligned", who);
    if (sm_count() > 160) return set_error("%s: a device of %d SMs", who, sm_count());
    AttnParams a;
    a.pool = pool_of(pool);
    a.b = batch_of(batch);
    a.q = p->q;
    a.gate = p->gate;
    a.out = p->out;
    a.ldq = p->ldq;
    a.ldgate = p->ldgate;
    a.ldout = p->ldout;
    a.qvec = rows_aligned(p->q, p->ldq, size);
    a.freq = p->freq;
    a.pdim = p->freq ? p->pdim : 0;
    a.heads = p->heads;
    a.group = p->heads / pool->kv_heads;
    a.window = p->window;
    a.scale = (p->scale != 0.f ? p->scale : 1.0f / sqrtf((float)pool->head_dim)) * LOG2E;
    a.tickets = (unsigned int *)p->workspace;
    a.part = (float *)((uint8_t *)p->workspace + TICKETS);
    a.err = device_error_ptr();
    const cudaStream_t s = (cudaStream_t)stream;
    return p->type == T_F32   ? launch_hd<float>(a, s, who)
           : p->type == T_F16 ? launch_hd<__half>(a, s, who)
                              : launch_hd<__nv_bfloat16>(a, s, who);
}

}  // extern "C"
