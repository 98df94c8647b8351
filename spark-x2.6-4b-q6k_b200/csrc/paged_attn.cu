// paged_attn.cu — causal grouped-query attention of each sequence's new rows over its pages of the
// 8-bit cache, for few rows per sequence (decode steps, verify batches).
//
//   out[t][h] = sigmoid(gate[t][h]) * sum_j p_j V_j,  p = softmax_j(scale * rope(q[t][h]) . K_j),
//   j in [0, pos_t], with a window in (pos_t - window, pos_t]; K_j = dk[block of j] * k_j and
//   V_j = dv[block] * v_j with the cached e4m3 bytes k, v. A row that sees nothing gets 0.
//
// With w_j = exp(s_j) dv_j the value scale rides in the exponent: s'_j = s_j + log dv_j, one
// running reference m per row, O = sum exp(s'_j - m) v_j and l = sum exp(s'_j - m) / dv_j, so that
// the largest term of the sum is what the f16 weights are relative to, whatever the scales.
//
// What bounds it: the cached bytes, read once per KV head. A (sequence, KV head) has n * group
// query rows; a tile of R of them is one pass over the blocks, and the R rows are the 8 or 16
// columns of the tensor-core products
//   S^T[16 keys][cols] = K q^T     mma.sync m16n8k16, A = a block's key bytes as f16 (exact)
//   O^T[hd][cols]     += V^T P^T   A = a block's value bytes, P^T by movmatrix
// so no lane idles for want of rows and a block's scales are two scalars. f32 calls keep q and P as
// f16 pairs (hi + lo columns, ~22 bits), f16 and bf16 calls as one f16; q's exponent is taken out
// per row first.
//
// Work split: all (sequence, KV head, row tile, block) units in one line, cut into equal ranges,
// one per CTA, one CTA per SM; a warp owns every 8th block of a range and streams it by two bulk
// copies through its own ring of mbarrier slots, meeting the other warps only at the end of a
// (sequence, KV head, row tile). Ranges that end inside one leave (O, m, l) in the workspace and
// the last CTA to arrive (a ticket that it resets) adds them up in CTA order.
#include "paged.cuh"

namespace spk {
namespace paged {
namespace {

constexpr int AT_WARPS = 8, AT_THREADS = AT_WARPS * 32;
constexpr float M_NONE = -1e30f;      // reference of a row that has seen nothing
constexpr float P_SHIFT = 7.0f;       // weights are kept as 2^7 exp(s' - m): f16 holds them from 2^-31 to 2^8
constexpr float M_SLACK = 8.0f;       // the reference moves only when a score passes it by 2^8
constexpr float LOG2E = 1.4426950408889634f;

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
    float *part;                      // [gridDim.x][2][R * (HD + 2)]
    int *err;
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 4 e4m3 bytes as two exact f16 pairs (bytes 0,1 | bytes 2,3)
__device__ __forceinline__ void e4m3x4_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}

__device__ __forceinline__ uint32_t movm(uint32_t x) {   // 8 x 8 f16 transpose across the warp
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

__device__ __forceinline__ uint32_t f16x2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int HD, int NT, int TERMS>
struct Cfg {
    static constexpr int COLS = 8 * NT;
    static constexpr int R = COLS / TERMS;                    // query rows of a tile
    static constexpr int KB = BLOCK * HD, STAGE = 2 * KB;     // bytes of a block's keys; keys and values
    static constexpr int NS = 512 / HD;                       // ring slots of a warp (16 KB)
    static constexpr int QS = HD * 2 + 32;                    // bytes of a q column in shared memory (padded)
    static constexpr int OR = R / NT;                         // rows merged at a time (one n-tile)
    static constexpr size_t RING = (size_t)AT_WARPS * NS * STAGE;
    static constexpr size_t MERGE = (size_t)AT_WARPS * OR * HD * 4;
    static constexpr size_t SMEM = RING + MERGE + (size_t)COLS * QS;
    static constexpr int PART = R * (HD + 2);                 // floats of a partial: O, then m, then l
};

// units (16-token blocks x KV heads x row tiles) of sequence s; the first block any row sees
struct Seq {
    int r0, n, len, first_blk, nblk, tiles;
};
__device__ __forceinline__ Seq seq_of(const AttnParams &a, int s, int R) {
    Seq q;
    q.r0 = __ldg(a.b.row0 + s);
    q.n = __ldg(a.b.row0 + s + 1) - q.r0;
    q.len = __ldg(a.b.kv_len + s);
    q.first_blk = q.nblk = q.tiles = 0;
    const long long room = (long long)a.b.max_pages * a.pool.page_tokens;
    if (q.n == 0) return q;
    if (q.n < 0 || q.r0 < 0 || q.r0 > a.b.rows - q.n || q.len > room) {   // not a batch: nothing is read
        if (a.err) atomicExch(a.err, DEV_BAD_INDEX);
        q.n = 0;
        return q;
    }
    const int pos0 = q.len - q.n;
    if (a.window > 0) q.first_blk = max(0, pos0 + 1 - a.window) / BLOCK;
    // a sequence with nothing cached still has rows to write (zeros): one empty block
    q.nblk = max(1, (q.len + BLOCK - 1) / BLOCK - q.first_blk);
    q.tiles = (int)(((long long)q.n * a.group + R - 1) / R);
    return q;
}

template <typename T, int HD, int NT, int TERMS>
__global__ void __launch_bounds__(AT_THREADS, 1) attn_kernel(const AttnParams a) {
    using C = Cfg<HD, NT, TERMS>;
    constexpr int R = C::R, KT = HD / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[AT_WARPS][C::NS];
    __shared__ float4 meta[AT_WARPS][C::NS];            // a slot's dk, log2 dv, 1 / dv, and whether it was issued
    __shared__ long long pre[MAX_SEQ + 1];              // units before each sequence
    __shared__ long long wsum[AT_WARPS];
    __shared__ float wm[AT_WARPS][R], wl[AT_WARPS][R];
    __shared__ float qf[R];                             // per row: score factor
    __shared__ int qpos[R];                             // per row: position, -1 past the end
    __shared__ float cw[256];
    __shared__ int last_in;
    uint8_t *ring = smem;
    float *merge = reinterpret_cast<float *>(smem + C::RING);
    uint8_t *qs = smem + C::RING + C::MERGE;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    pdl_trigger();
    if (tid < AT_WARPS * C::NS) mbar_init(&bars[0][0] + tid, 1);
    fence_mbar_init();
    pdl_wait();

    // the line of units: an exclusive scan over the sequences
    long long base = 0;
    for (int s0 = 0; s0 < a.b.nseq; s0 += AT_THREADS) {
        const int s = s0 + tid;
        long long u = 0;
        if (s < a.b.nseq) {
            const Seq q = seq_of(a, s, R);
            u = (long long)q.nblk * q.tiles * a.pool.kv_heads;
        }
        long long x = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) wsum[warp] = x;
        __syncthreads();
        long long add = base;
        for (int w = 0; w < warp; w++) add += wsum[w];
        if (s < a.b.nseq) pre[s] = add + x - u;
        long long all = base;
        for (int w = 0; w < AT_WARPS; w++) all += wsum[w];
        base = all;
        __syncthreads();
    }
    if (tid == 0) pre[a.b.nseq] = base;
    __syncthreads();
    const long long total = base;
    // equal ranges, at least a block per warp
    long long chunk = (total + gridDim.x - 1) / gridDim.x;
    if (chunk < AT_WARPS) chunk = AT_WARPS;
    const long long u0 = chunk * blockIdx.x, u1 = min(total, u0 + chunk);
    uint32_t used = 0;   // this warp's ring uses so far (slot used % NS, parity used / NS)

    int s = 0;
    if (u0 < u1) {   // the sequence of u0: the last with pre <= u0 that has units
        int lo = 0, hi = a.b.nseq;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid] <= u0) lo = mid;
            else hi = mid;
        }
        s = lo;
    }
    for (long long u = u0; u < u1;) {
        while (pre[s + 1] <= u) s++;
        const Seq q = seq_of(a, s, R);
        const long long in = u - pre[s];
        const int gr = (int)(in / q.nblk), b0 = (int)(in - (long long)gr * q.nblk);   // group (KV head, row tile)
        const int b1 = (int)min((long long)q.nblk, b0 + (u1 - u));
        const int kvh = gr / q.tiles, tile = gr - kvh * q.tiles;
        const int pos0 = q.len - q.n;
        // blocks that some row of the tile sees
        const int c0 = tile * R, c1 = min(c0 + R, q.n * a.group) - 1;
        const int p_lo = pos0 + c0 / a.group, p_hi = pos0 + c1 / a.group;
        const int see0 = a.window > 0 ? max(0, p_lo + 1 - a.window) : 0;
        const int x0 = max(b0, see0 / BLOCK - q.first_blk), x1 = min(b1, p_hi < 0 ? 0 : p_hi / BLOCK + 1 - q.first_blk);
        const int cnt = x1 > x0 + warp ? (x1 - x0 - warp + AT_WARPS - 1) / AT_WARPS : 0;   // this warp's blocks
        const int bfirst = q.first_blk + x0 + warp;

        // 32 of the warp's blocks at a time: lane l holds block i's place in the pool and its scales
        size_t at = 0;
        float dk = 0.f, dv = 1.f;
        auto look = [&](int i0) {
            const int i = i0 + lane;
            at = 0;
            if (i < cnt) {
                const int blk = bfirst + i * AT_WARPS, per = a.pool.page_tokens / BLOCK;
                int page = __ldg(a.b.table + (size_t)s * a.b.max_pages + blk / per);
                if (page < 0 || page >= a.pool.pages) {
                    if (a.err) atomicExch(a.err, DEV_BAD_INDEX);
                    page = 0;
                }
                at = block_index(a.pool, page, kvh, blk % per);
                dk = a.pool.ks[at];
                dv = a.pool.vs[at];
            }
        };
        auto issue = [&](int i) {   // all lanes
            if ((i & 31) == 0) look(i);
            const size_t bi = __shfl_sync(0xffffffffu, at, i & 31);
            const float k_ = __shfl_sync(0xffffffffu, dk, i & 31), v_ = __shfl_sync(0xffffffffu, dv, i & 31);
            const int slot = (used + i) % C::NS;
            __syncwarp();
            if (lane == 0) {
                meta[warp][slot] = make_float4(k_, log2f(v_), 1.0f / v_, 0.f);
                uint8_t *d = ring + ((size_t)warp * C::NS + slot) * C::STAGE;
                mbar_arrive_expect_tx(&bars[warp][slot], C::STAGE);
                bulk_g2s(d, a.pool.k + bi * C::KB, C::KB, &bars[warp][slot]);
                bulk_g2s(d + C::KB, a.pool.v + bi * C::KB, C::KB, &bars[warp][slot]);
            }
            __syncwarp();
        };
        for (int i = 0; i < C::NS && i < cnt; i++) issue(i);

        // the tile's queries: a warp per row, rotated, scaled to [1, 2), as f16 (pairs)
        for (int r = warp; r < R; r += AT_WARPS) {
            const int c = c0 + r;
            const bool real = c <= c1;
            float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
            const int tok = c / a.group, pos = pos0 + tok;
            if (real && lane < HD / 8) {
                const T *src = (const T *)a.q + (size_t)(q.r0 + tok) * a.ldq + (size_t)(kvh * a.group + c % a.group) * HD;
                load_unit<T>(src, lane, a.freq, a.pdim, pos, a.qvec, x, y);
            }
            float mx = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) mx = fmaxf(mx, fmaxf(fabsf(x[e]), fabsf(y[e])));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            // 2^-e and 2^e by exponent bits; a row of zeros, denormals or infinities keeps 1
            const int ex = (int)(__float_as_uint(mx) >> 23);
            const bool ok = ex >= 2 && ex <= 252;
            const float dn = ok ? __uint_as_float((uint32_t)(254 - ex) << 23) : 1.0f;
            const float up = ok ? __uint_as_float((uint32_t)ex << 23) : 1.0f;
            if (lane < HD / 8) {
                int d0, d1;
                unit_dims(lane, a.pdim, d0, d1);
                const int col = TERMS == 2 ? (r >> 2) * 8 + (r & 3) : r;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[e] *= dn;
                    y[e] *= dn;
                }
                uint8_t *at0 = qs + (size_t)col * C::QS;
                *reinterpret_cast<uint2 *>(at0 + 2 * d0) = make_uint2(f16x2(x[0], x[1]), f16x2(x[2], x[3]));
                *reinterpret_cast<uint2 *>(at0 + 2 * d1) = make_uint2(f16x2(y[0], y[1]), f16x2(y[2], y[3]));
                if (TERMS == 2) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[e] -= __half2float(__float2half_rn(x[e]));
                        y[e] -= __half2float(__float2half_rn(y[e]));
                    }
                    at0 += 4 * C::QS;
                    *reinterpret_cast<uint2 *>(at0 + 2 * d0) = make_uint2(f16x2(x[0], x[1]), f16x2(x[2], x[3]));
                    *reinterpret_cast<uint2 *>(at0 + 2 * d1) = make_uint2(f16x2(y[0], y[1]), f16x2(y[2], y[3]));
                }
            }
            if (lane == 0) {
                qf[r] = up * a.scale;
                qpos[r] = real ? pos : -1;
            }
        }
        __syncthreads();

        // a lane's columns 2t, 2t + 1 of each n-tile are these rows (pairs: hi and lo lanes share them)
        float fac[NT][2];
        int cpos[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = nt * (R / NT) + (TERMS == 2 ? 2 * (t & 1) + e : 2 * t + e);
                fac[nt][e] = qf[r];
                cpos[nt][e] = qpos[r];
            }
        uint32_t qb[NT == 1 ? KT : 1][2];
        if constexpr (NT == 1)
#pragma unroll
            for (int c = 0; c < KT; c++) {
                const uint2 w = *reinterpret_cast<const uint2 *>(qs + (size_t)g * C::QS + 32 * c + 8 * t);
                qb[c][0] = w.x;
                qb[c][1] = w.y;
            }
        float o[NT][KT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int c = 0; c < KT; c++) o[nt][c][0] = o[nt][c][1] = o[nt][c][2] = o[nt][c][3] = 0.f;
            m[nt][0] = m[nt][1] = M_NONE;
            l[nt][0] = l[nt][1] = 0.f;
        }

        for (int i = 0; i < cnt; i++) {
            const uint32_t use = used + i;
            const int slot = use % C::NS;
            const bool here = mbar_wait(&bars[warp][slot], (use / C::NS) & 1, a.err);
            if (here) {
                const uint8_t *kb = ring + ((size_t)warp * C::NS + slot) * C::STAGE, *vb = kb + C::KB;
                const float4 mt = meta[warp][slot];
                float sc[NT][2][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int h = 0; h < 2; h++) sc[nt][h][0] = sc[nt][h][1] = sc[nt][h][2] = sc[nt][h][3] = 0.f;
                const uint8_t *ka = kb + g * 16 + 4 * t;
#pragma unroll
                for (int c = 0; c < KT; c++) {
                    uint32_t a0, a1, a2, a3;
                    e4m3x4_f16(*reinterpret_cast<const uint32_t *>(ka + c * 128), a0, a2);
                    e4m3x4_f16(*reinterpret_cast<const uint32_t *>(ka + 8 * HD + c * 128), a1, a3);
                    if constexpr (NT == 1) {
                        mma16816(sc[0][c & 1], a0, a1, a2, a3, qb[c][0], qb[c][1]);
                    } else {
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            const uint2 w =
                                *reinterpret_cast<const uint2 *>(qs + (size_t)(nt * 8 + g) * C::QS + 32 * c + 8 * t);
                            mma16816(sc[nt][c & 1], a0, a1, a2, a3, w.x, w.y);
                        }
                    }
                }
                const int j0 = (bfirst + i * AT_WARPS) * BLOCK;
                // bytes of this lane's 4 value tokens that some row sees: a masked place never meets the product
                uint32_t vmask = 0xffffffffu;
                if (j0 + BLOCK - 1 > p_hi || j0 < see0) {
                    vmask = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int j = j0 + order(4 * t + e);
                        if (j <= p_hi && j >= see0) vmask |= 0xffu << (8 * e);
                    }
                }
                const bool edge = j0 + BLOCK - 1 > p_lo || (a.window > 0 && j0 <= p_hi - a.window);
                uint32_t pb[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float sv[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float x = sc[nt][0][e] + sc[nt][1][e];
                        if (TERMS == 2) x += __shfl_xor_sync(0xffffffffu, x, 2);
                        x = fmaf(x, mt.x * fac[nt][e & 1], mt.y);
                        if (edge) {
                            const int j = j0 + g + 8 * (e >> 1), p = cpos[nt][e & 1];
                            if (j > p || (a.window > 0 && j <= p - a.window)) x = -INFINITY;
                        }
                        sv[e] = x;
                    }
                    const bool over = fmaxf(sv[0], sv[2]) > m[nt][0] + M_SLACK || fmaxf(sv[1], sv[3]) > m[nt][1] + M_SLACK;
                    if (__any_sync(0xffffffffu, over)) {
                        float mx[2] = {fmaxf(sv[0], sv[2]), fmaxf(sv[1], sv[3])};
#pragma unroll
                        for (int of = 4; of < 32; of <<= 1) {
                            mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], of));
                            mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], of));
                        }
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float nm = fmaxf(m[nt][e], mx[e]), f = ex2(m[nt][e] - nm);
                            m[nt][e] = nm;
                            l[nt][e] *= f;
#pragma unroll
                            for (int c = 0; c < KT; c++) {
                                o[nt][c][e] *= f;
                                o[nt][c][2 + e] *= f;
                            }
                        }
                    }
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        p[e] = ex2(sv[e] - m[nt][e & 1] + P_SHIFT);
                        l[nt][e & 1] = fmaf(p[e], mt.z, l[nt][e & 1]);
                    }
                    if (TERMS == 2 && t >= 2) {   // the lo columns
#pragma unroll
                        for (int e = 0; e < 4; e++) p[e] -= __half2float(__float2half_rn(p[e]));
                    }
                    pb[nt][0] = movm(f16x2(p[0], p[1]));
                    pb[nt][1] = movm(f16x2(p[2], p[3]));
                }
                const uint8_t *va = vb + g * 16 + 4 * t;
#pragma unroll
                for (int c = 0; c < KT; c++) {
                    uint32_t a0, a1, a2, a3;
                    e4m3x4_f16(*reinterpret_cast<const uint32_t *>(va + c * 256) & vmask, a0, a2);
                    e4m3x4_f16(*reinterpret_cast<const uint32_t *>(va + c * 256 + 128) & vmask, a1, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) mma16816(o[nt][c], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                }
            }
            if (i + C::NS < cnt) issue(i + C::NS);
        }
        used += cnt;

        // the warps' (O, m, l) into the tile's
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float v = l[nt][e];
#pragma unroll
                for (int of = 4; of < 32; of <<= 1) v += __shfl_xor_sync(0xffffffffu, v, of);
                l[nt][e] = v;
                const int r = nt * C::OR + (TERMS == 2 ? 2 * (t & 1) + e : 2 * t + e);
                if (g == 0 && (TERMS == 1 || t < 2)) {
                    wm[warp][r] = m[nt][e];
                    wl[warp][r] = v;
                }
            }
        __syncthreads();
        const bool whole = b0 == 0 && b1 == q.nblk;
        float *slot = a.part + ((size_t)blockIdx.x * 2 + (b0 == 0 ? 1 : 0)) * C::PART;
        if (!whole && tid < R) {
            float M = M_NONE, L = 0.f;
            for (int w = 0; w < AT_WARPS; w++) M = fmaxf(M, wm[w][tid]);
            for (int w = 0; w < AT_WARPS; w++) L = fmaf(wl[w][tid], ex2(wm[w][tid] - M), L);
            slot[R * HD + tid] = M;
            slot[R * HD + R + tid] = L;
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int rr = TERMS == 2 ? 2 * (t & 1) + e : 2 * t + e, r = nt * C::OR + rr;
                float M = M_NONE;
#pragma unroll
                for (int w = 0; w < AT_WARPS; w++) M = fmaxf(M, wm[w][r]);
                const float f = ex2(m[nt][e] - M);
                float *dst = merge + ((size_t)warp * C::OR + rr) * HD;
#pragma unroll
                for (int c = 0; c < KT; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float v = o[nt][c][2 * h + e] * f;
                        if (TERMS == 2) v += __shfl_xor_sync(0xffffffffu, v, 2);   // hi + lo columns
                        if (TERMS == 1 || t < 2) dst[16 * c + 8 * h + g] = v;
                    }
            }
            __syncthreads();
            for (int i = tid; i < C::OR * HD; i += AT_THREADS) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < AT_WARPS; w++) v += merge[(size_t)w * C::OR * HD + i];
                const int rr = i / HD, d = i - rr * HD, r = nt * C::OR + rr;
                if (whole) {
                    const int c = c0 + r;
                    if (c <= c1) {
                        float M = M_NONE, L = 0.f;
#pragma unroll
                        for (int w = 0; w < AT_WARPS; w++) M = fmaxf(M, wm[w][r]);
#pragma unroll
                        for (int w = 0; w < AT_WARPS; w++) L = fmaf(wl[w][r], ex2(wm[w][r] - M), L);
                        v = L == 0.f ? 0.f : v / L;
                        const int row = q.r0 + c / a.group, h = kvh * a.group + c % a.group;
                        if (a.gate) v /= 1.0f + __expf(-to_f32(((const T *)a.gate)[(size_t)row * a.ldgate + h]));
                        ((T *)a.out)[(size_t)row * a.ldout + (size_t)h * HD + d] = from_f32<T>(v);
                    }
                } else {
                    slot[(size_t)r * HD + d] = v;
                }
            }
            __syncthreads();
        }
        if (!whole) {   // the last CTA of the group adds all parts in CTA order
            const long long gs = u - b0, ge = gs + q.nblk;
            const int f0 = (int)(gs / chunk), f1 = (int)((ge - 1) / chunk), parts = f1 - f0 + 1;
            __threadfence();
            __syncthreads();
            if (tid == 0) last_in = atomicAdd(a.tickets + f0, 1u) == (unsigned)(parts - 1);
            __syncthreads();
            if (last_in) {
                __threadfence();
                const size_t step = (size_t)2 * C::PART;
                const float *p0 = a.part + (size_t)f0 * step;   // CTA f0: slot 1, the others: slot 0
                for (int i = tid; i < R * (HD / 4); i += AT_THREADS) {
                    const int r = i / (HD / 4), d = 4 * (i - r * (HD / 4)), c = c0 + r;
                    if (c > c1) continue;
                    float M = M_NONE;
                    for (int p = 0; p < parts; p++)
                        M = fmaxf(M, __ldcg(p0 + p * step + (p == 0 ? C::PART : 0) + R * HD + r));
                    float L = 0.f;
                    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (int p = 0; p < parts; p++) {
                        const float *pp = p0 + p * step + (p == 0 ? C::PART : 0);
                        const float f = ex2(__ldcg(pp + R * HD + r) - M);
                        const float4 v = __ldcg(reinterpret_cast<const float4 *>(pp + (size_t)r * HD + d));
                        L = fmaf(__ldcg(pp + R * HD + R + r), f, L);
                        O.x = fmaf(v.x, f, O.x);
                        O.y = fmaf(v.y, f, O.y);
                        O.z = fmaf(v.z, f, O.z);
                        O.w = fmaf(v.w, f, O.w);
                    }
                    const int row = q.r0 + c / a.group, h = kvh * a.group + c % a.group;
                    float f = L == 0.f ? 0.f : 1.0f / L;
                    if (L == 0.f) O = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (a.gate) f /= 1.0f + __expf(-to_f32(((const T *)a.gate)[(size_t)row * a.ldgate + h]));
                    T *dst = (T *)a.out + (size_t)row * a.ldout + (size_t)h * HD + d;
                    dst[0] = from_f32<T>(O.x * f);
                    dst[1] = from_f32<T>(O.y * f);
                    dst[2] = from_f32<T>(O.z * f);
                    dst[3] = from_f32<T>(O.w * f);
                }
                if (tid == 0) a.tickets[f0] = 0u;
            }
            __syncthreads();
        }
        u += b1 - b0;
    }
}

constexpr size_t TICKETS = 1024;   // bytes before the partials: one word per CTA (at most 256)

template <typename T, int HD, int NT, int TERMS>
cudaError_t launch_one(const AttnParams &a, cudaStream_t s) {
    using C = Cfg<HD, NT, TERMS>;
    static bool set[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(attn_kernel<T, HD, NT, TERMS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)C::SMEM);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) set[dev] = true;
    }
    return launch_pdl(attn_kernel<T, HD, NT, TERMS>, dim3(sm_count()), dim3(AT_THREADS), C::SMEM, s, a);
}

template <typename T, int HD>
cudaError_t launch(const AttnParams &a, cudaStream_t s) {
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
    // two n-tiles when a sequence's rows of a KV head overfill one on average
    const bool wide = (long long)a.b.rows * a.group > (long long)a.b.nseq * (8 / TERMS);
    return wide ? launch_one<T, HD, 2, TERMS>(a, s) : launch_one<T, HD, 1, TERMS>(a, s);
}

template <typename T>
cudaError_t launch_hd(const AttnParams &a, cudaStream_t s) {
    return a.pool.hd == 256 ? launch<T, 256>(a, s) : a.pool.hd == 128 ? launch<T, 128>(a, s) : launch<T, 64>(a, s);
}

}  // namespace
}  // namespace paged
}  // namespace spk

extern "C" {

size_t spk_paged_attn_workspace_bytes(int head_dim) {
    using namespace spk::paged;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
    return TICKETS + (size_t)spk::sm_count() * 2 * 16 * (head_dim + 2) * sizeof(float);
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
    if (p->pdim < 0 || p->pdim % 8 || p->pdim > pool->head_dim || (p->pdim > 0 && !p->freq))
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
    if (sm_count() > (int)(TICKETS / 4)) return set_error("%s: a device of %d SMs", who, sm_count());
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
    const cudaError_t e = p->type == T_F32   ? launch_hd<float>(a, s)
                          : p->type == T_F16 ? launch_hd<__half>(a, s)
                                             : launch_hd<__nv_bfloat16>(a, s);
    return e == cudaSuccess ? 0 : cuda_fail(who, e);
}

}  // extern "C"
