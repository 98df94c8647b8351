// paged_append.cu — new keys and values of a batch into the pages of the 8-bit cache.
//
// Row i of sequence s (rows row0[s] .. row0[s + 1] - 1) sits at position kv_len[s] - n_s + i. Its
// key is rotated (paged.cuh), then, per KV head and per block of 16 tokens that the call
// touches, for keys and for values:
//   d   = max(amax / 448, 2^-100), amax over the call's rows in the block; where the block holds
//         earlier rows (the call starts inside it) also d >= its old scale
//   q   = e4m3(x * (1 / d));  earlier rows are rounded again, e4m3(q * (d_old / d)), where d grew;
//         the block's rows after the last new one become 0
// so that a block which is read holds nothing that was not appended. A NaN or infinity makes the
// block's scale NaN or infinite (its rows read as NaN) and never a stored byte.
//
// What bounds it: the issue slots for prompts (19 warp instructions per 32 values: conversions, angles,
// the rotation, addresses), the chain of dependent loads (sequence -> page -> row) for steps. A CTA of 4
// warps takes one block, keys or values, and 256 values of a row at a time (256 / head_dim heads
// side by side): a warp 4 of the 16 rows, a lane 8 values of each, so that a head's amax is a max in registers, a
// shuffle tree and one exchange between the warps. The bytes meet in shared memory (4 KB, 16-byte
// pieces spread over the banks) and leave as 16-byte stores. Where there are many blocks a CTA walks
// several head groups, which share the rows' angles: a cosine and sine cost as much as ten values'
// rounding and storing. Measured, launched one by one on rows that are not in L2: 16384 bf16 rows of 4 heads of 256,
// keys and values, 29 us (101 MB, 3.5 TB/s, 0.54 of a copy's rate); 13 f32 prompts of up to 1501 rows 15.7 us (44 MB);
// one row 5.9 us, which is a launch's distance from the next. In a graph, over the same rows again: 27, 12.7 and 3.7 us.
#include "paged.cuh"

namespace spk {
namespace paged {

int check_pool(const spk_kv_pool *p, const char *who) {
    if (!p || !p->k || !p->v || !p->k_scale || !p->v_scale) return set_error("%s: the pool has a null buffer", who);
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
        return set_error("%s: head_dim %d (64, 128 or 256)", who, p->head_dim);
    if (p->pages < 1 || p->kv_heads < 1 || p->page_tokens < BLOCK || p->page_tokens % BLOCK)
        return set_error("%s: %d pages of %d tokens (a multiple of 16), %d KV heads", who, p->pages, p->page_tokens,
                         p->kv_heads);
    if (((uintptr_t)p->k | (uintptr_t)p->v) % 16) return set_error("%s: the pool is not 16-byte aligned", who);
    if (((uintptr_t)p->k_scale | (uintptr_t)p->v_scale) % 4) return set_error("%s: unaligned scales", who);
    return 0;
}

int check_batch(const spk_kv_batch *b, const char *who) {
    if (!b || !b->row0 || !b->kv_len || !b->table) return set_error("%s: the batch has a null buffer", who);
    if (b->nseq < 1 || b->nseq > MAX_SEQ) return set_error("%s: %d sequences (1 to %d)", who, b->nseq, MAX_SEQ);
    if (b->rows < 0 || b->max_pages < 1) return set_error("%s: %d rows, %d pages a sequence", who, b->rows, b->max_pages);
    return 0;
}

namespace {

constexpr int AP_WARPS = 4, AP_THREADS = AP_WARPS * 32, AP_ROWS = BLOCK / AP_WARPS;
constexpr int AP_WIDTH = 256;              // values of a row that a warp takes at once
template <typename T>
constexpr int AP_CTAS = sizeof(T) == 4 ? 5 : 6;   // CTAs of an SM: two items' rows stay in registers

struct AppendArgs {
    Pool pool;
    Batch b;
    const void *k, *v;
    long long ldk, ldv;
    int kvec, vvec;                        // alignment of the rows' pieces: 0 none, 1 four values, 2 eight too
    const float *freq;
    int pdim;
    int passes;                            // head groups of a CTA
    int *err;
};

// max of |a|, |b|, |c| that keeps a NaN
__device__ __forceinline__ float max_abs(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {   // low byte a
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 e4m3x2_f32(uint32_t w) {
    return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3)));
}

// 16-byte piece of the staging tile, spread so that a warp's 4-byte writes (pieces 8 apart) meet few banks
__device__ __forceinline__ int spread(int piece) { return piece ^ ((piece >> 3) & 7); }

// A block that the call appends to: its place in the pool for KV head 0, its first position, the
// call's rows lo .. hi - 1 of it; row r of the block is row `row` + r of the call.
struct Block {
    size_t at;
    int pos, lo, hi, row;
};

template <typename T, int HD, bool KEYS>
__device__ __forceinline__ void append_block(const AppendArgs &a, const Block b, uint8_t *tile, float *turn_c,
                                             float *turn_s, float (*wmax)[AP_WARPS]) {
    constexpr int LPR = HD / 8, GH = AP_WIDTH / HD, PER = AP_WIDTH / AP_THREADS;   // lanes of a head; heads; pieces of a thread
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / LPR, u = lane % LPR;
    const int pdim = KEYS ? a.pdim : 0, half = pdim / 2;
    int d0, d1;
    unit_dims(u, pdim, d0, d1);
    uint8_t *pool = KEYS ? a.pool.k : a.pool.v;
    float *scales = KEYS ? a.pool.ks : a.pool.vs;
    const T *rows = KEYS ? (const T *)a.k : (const T *)a.v;
    const long long ld = KEYS ? a.ldk : a.ldv;
    const int vec = KEYS ? a.kvec : a.vvec;
    const int g0 = blockIdx.y * a.passes, groups = min(a.passes, (a.pool.kv_heads + GH - 1) / GH - g0);
    const int lo = b.lo, hi = b.hi, per = a.pool.page_tokens / BLOCK;
    // a head group's rows come while the one before is worked on
    Raw<T> next[AP_ROWS];
    auto fetch = [&](int g) {
        const int head = g * GH + sub, from = head < a.pool.kv_heads ? lo : BLOCK;
        const T *at = rows + (long long)(b.row + 2 * warp) * ld + (long long)head * HD;
#pragma unroll
        for (int i = 0; i < AP_ROWS; i++) {
            // warp w: rows 2w, 2w + 1, 2w + 8, 2w + 9, which are bytes 4w .. 4w + 3 of a value dim
            const int dr = (i & 1) + 8 * (i >> 1), r = 2 * warp + dr;
            if (r >= from && r < hi) next[i].load(at + dr * ld, d0, d1, vec);
            else next[i].none();
        }
    };
    fetch(g0);
    if constexpr (KEYS)
        if (half) {   // the rows' angles, for all heads
            for (int r = warp; r < BLOCK; r += AP_WARPS)
                if (r >= lo && r < hi)
                    for (int i = lane; i < half; i += 32)
                        angle(b.pos + r, __ldg(a.freq + i), turn_c[r * half + i], turn_s[r * half + i]);
            __syncthreads();
        }
    for (int g = g0; g < g0 + groups; g++) {
        float x[AP_ROWS][8];
#pragma unroll
        for (int i = 0; i < AP_ROWS; i++) next[i].f32(x[i]);
        if (g + 1 < g0 + groups) fetch(g + 1);
        const int head = g * GH + sub;
        const bool real = head < a.pool.kv_heads;
        const size_t bi = b.at + (size_t)min(head, a.pool.kv_heads - 1) * per;
        // earlier rows and their scale, on their way while the new rows come in
        uint4 old[PER];
        float d_old = 0.f;
        if (lo > 0) {
            d_old = scales[bi];
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int pc = i * AP_THREADS + threadIdx.x, hd = g * GH + pc / HD;
                if (hd < a.pool.kv_heads)
                    old[i] = reinterpret_cast<const uint4 *>(pool + (b.at + (size_t)hd * per) * (BLOCK * HD))[pc % HD];
            }
        }
        float mx = 0.f;
        if (KEYS && u < pdim / 8) {
#pragma unroll
            for (int i = 0; i < AP_ROWS; i++) {
                const int r = 2 * warp + (i & 1) + 8 * (i >> 1);
                if (r < lo || r >= hi) continue;
                const float4 c4 = *reinterpret_cast<const float4 *>(turn_c + r * half + d0);
                const float4 s4 = *reinterpret_cast<const float4 *>(turn_s + r * half + d0);
                const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
                float p[4], q[4];
#pragma unroll
                for (int e = 0; e < 4; e++) p[e] = x[i][e], q[e] = x[i][4 + e];
                rotate_unit(p, q, c, s);
#pragma unroll
                for (int e = 0; e < 4; e++) x[i][e] = p[e], x[i][4 + e] = q[e];
            }
        }
#pragma unroll
        for (int i = 0; i < AP_ROWS; i++)
#pragma unroll
            for (int e = 0; e < 8; e += 2) mx = max_abs(mx, x[i][e], x[i][e + 1]);
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (u == 0) wmax[sub][warp] = mx;
        __syncthreads();   // the maxima are there, and the tile is free
        mx = max_nan(max_nan(wmax[sub][0], wmax[sub][1]), max_nan(wmax[sub][2], wmax[sub][3]));
        float d = max_nan(__fdiv_rn(mx, E4M3_MAX), SCALE_MIN);
        if (lo > 0) d = max_nan(d, d_old);
        if (lo > 0) {   // earlier rows, rounded again where the scale grew; 0 elsewhere
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int pc = i * AP_THREADS + threadIdx.x, hs = pc / HD, in = pc % HD;
                float m2 = max_nan(max_nan(wmax[hs][0], wmax[hs][1]), max_nan(wmax[hs][2], wmax[hs][3]));
                const int hd = g * GH + hs;
                if (hd >= a.pool.kv_heads) continue;
                const float o2 = scales[b.at + (size_t)hd * per];
                m2 = max_nan(max_nan(__fdiv_rn(m2, E4M3_MAX), SCALE_MIN), o2);
                const float ratio = m2 > o2 ? __fdiv_rn(o2, m2) : 1.0f;
                // keys: piece = (8-token group, 16-dim chunk, token): one token; values: one dim's 16 tokens
                const int ktok = 8 * (in / (HD / 2)) + (in & 7);
                uint32_t w[4] = {old[i].x, old[i].y, old[i].z, old[i].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t v = 0;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int t0 = KEYS ? ktok : order(4 * j + 2 * h), t1 = KEYS ? ktok : order(4 * j + 2 * h + 1);
                        uint32_t pr = (w[j] >> (16 * h)) & 0xffffu;
                        if (ratio != 1.0f) {
                            const float2 f = e4m3x2_f32(pr);
                            pr = e4m3x2(__fmul_rn(f.x, ratio), __fmul_rn(f.y, ratio));
                        }
                        if (t0 >= lo) pr &= 0xff00u;
                        if (t1 >= lo) pr &= 0x00ffu;
                        v |= pr << (16 * h);
                    }
                    w[j] = v;
                }
                reinterpret_cast<uint4 *>(tile)[spread(pc)] = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncthreads();
        }
        // the new rows (all of the tile when nothing earlier is in the block); none where the scale is no number
        const float inv = __fdiv_rn(1.0f, d);
        uint32_t q[AP_ROWS][4];   // e4m3 pairs
#pragma unroll
        for (int i = 0; i < AP_ROWS; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 y = unpack2(mul2(pack2(x[i][2 * e], x[i][2 * e + 1]), pack2(inv, inv)));
                q[i][e] = e4m3x2(y.x, y.y);
            }
        if (!(d < INFINITY))
#pragma unroll
            for (int i = 0; i < AP_ROWS; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) q[i][e] = 0;
        if (KEYS) {
#pragma unroll
            for (int i = 0; i < AP_ROWS; i++) {
                const int r = 2 * warp + (i & 1) + 8 * (i >> 1);
                if (r < lo) continue;
                const int pc = sub * HD + (r >> 3) * (HD / 2) + (r & 7);
                *reinterpret_cast<uint32_t *>(tile + 16 * spread(pc + 8 * (d0 >> 4)) + (d0 & 15)) = __byte_perm(q[i][0], q[i][1], 0x5410);
                *reinterpret_cast<uint32_t *>(tile + 16 * spread(pc + 8 * (d1 >> 4)) + (d1 & 15)) = __byte_perm(q[i][2], q[i][3], 0x5410);
            }
        } else {
            uint32_t keep = 0;   // bytes that hold earlier rows
#pragma unroll
            for (int i = 0; i < AP_ROWS; i++)
                if (2 * warp + (i & 1) + 8 * (i >> 1) < lo) keep |= 0xffu << (8 * i);
#pragma unroll
            for (int e = 0; e < 4; e++) {   // two dims: the rows' low bytes, the rows' high bytes
                const uint32_t m = __byte_perm(q[0][e], q[1][e], 0x5410), n = __byte_perm(q[2][e], q[3][e], 0x5410);
                const uint32_t w[2] = {__byte_perm(m, n, 0x6420), __byte_perm(m, n, 0x7531)};
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t *at = reinterpret_cast<uint32_t *>(tile + 16 * spread(sub * HD + 8 * u + 2 * e + h)) + warp;
                    *at = keep ? (*at & keep) | (w[h] & ~keep) : w[h];
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int pc = i * AP_THREADS + threadIdx.x, hd = g * GH + pc / HD;
            if (hd < a.pool.kv_heads)
                reinterpret_cast<uint4 *>(pool + (b.at + (size_t)hd * per) * (BLOCK * HD))[pc % HD] =
                    reinterpret_cast<const uint4 *>(tile)[spread(pc)];
        }
        if (u == 0 && warp == 0 && real) scales[bi] = d;
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(AP_THREADS, AP_CTAS<T>) append_kernel(const AppendArgs a) {
    __shared__ __align__(16) uint8_t tile[BLOCK * AP_WIDTH];
    __shared__ __align__(16) float turn_c[BLOCK * HD / 2], turn_s[BLOCK * HD / 2];
    __shared__ float wmax[AP_WIDTH / HD][AP_WARPS];
    __shared__ int4 who;      // sequence, its first row, its rows, its cached tokens
    pdl_trigger();
    if (threadIdx.x == 0) who.x = -1;
    __syncthreads();
    pdl_wait();
    const int unit = blockIdx.x;
    // Units of sequence s: row0[s] / 16 + 2 s up to the next one's; n rows touch at most
    // n / 16 + 2 blocks, so each sequence's blocks fit.
    for (int s = threadIdx.x; s < a.b.nseq; s += AP_THREADS) {
        const int r0 = __ldg(a.b.row0 + s), r1 = __ldg(a.b.row0 + s + 1), len = __ldg(a.b.kv_len + s);
        if (r1 > r0 && unit >= r0 / BLOCK + 2 * s && unit < r1 / BLOCK + 2 * s + 2) who = make_int4(s, r0, r1 - r0, len);
    }
    __syncthreads();
    const int4 w = who;
    const int first = w.w - w.z, blk = first / BLOCK + (unit - w.y / BLOCK - 2 * w.x);
    if (w.x < 0 || (first >= 0 && blk * BLOCK >= w.w)) return;   // no block
    const int per = a.pool.page_tokens / BLOCK;
    int page = -1;
    if (first >= 0 && blk >= 0 && w.y >= 0 && w.y + w.z <= a.b.rows && blk / per < a.b.max_pages)
        page = __ldg(a.b.table + (size_t)w.x * a.b.max_pages + blk / per);
    if (page < 0 || page >= a.pool.pages) {
        if (a.err && threadIdx.x == 0) atomicExch(a.err, DEV_BAD_INDEX);
        return;
    }
    const Block b{block_index(a.pool, page, 0, blk % per), blk * BLOCK, max(first - blk * BLOCK, 0),
                  min(w.w - blk * BLOCK, BLOCK), w.y + blk * BLOCK - first};
    if (blockIdx.z == 0) append_block<T, HD, true>(a, b, tile, turn_c, turn_s, wmax);
    else append_block<T, HD, false>(a, b, tile, turn_c, turn_s, wmax);
}

template <typename T, int HD>
cudaError_t launch(AppendArgs a, cudaStream_t s) {
    const int groups = (a.pool.kv_heads + AP_WIDTH / HD - 1) / (AP_WIDTH / HD);
    // A CTA walks several head groups of its block, as long as every SM still gets its CTAs: they share the
    // block's angles and hide each other's loads (in a graph: 16384 bf16 rows of 4 groups: 28 us with all 4, 30.6 with 2,
    // 38.5 with 1; 4096 rows: 10.0 with 2, 10.4 with 1, 12.8 with 4; one row: 3.8 with 1, 5.3 with 2).
    const int slots = AP_CTAS<T> * sm_count(), units = a.b.rows / BLOCK;   // whole blocks: about what there is to do
    const long long most = 2ll * groups * units / slots;
    a.passes = most < 1 ? 1 : most < groups ? (int)most : groups;
    a.passes = (groups + (groups + a.passes - 1) / a.passes - 1) / ((groups + a.passes - 1) / a.passes);
    const dim3 grid(units + 2 * a.b.nseq, (groups + a.passes - 1) / a.passes, 2);
    return launch_pdl(append_kernel<T, HD>, grid, dim3(AP_THREADS), 0, s, a);
}
template <typename T>
cudaError_t launch(const AppendArgs &a, cudaStream_t s) {
    return a.pool.hd == 256 ? launch<T, 256>(a, s) : a.pool.hd == 128 ? launch<T, 128>(a, s) : launch<T, 64>(a, s);
}

}  // namespace
}  // namespace paged
}  // namespace spk

extern "C" int spk_paged_append(const spk_kv_pool *pool, const spk_kv_batch *batch, const void *k, long long ldk,
                                const void *v, long long ldv, int type, const float *freq, int pdim, void *stream) {
    using namespace spk;
    using namespace spk::paged;
    const char *who = "spk_paged_append";
    if (check_pool(pool, who) || check_batch(batch, who)) return -1;
    if (type < T_F32 || type > T_BF16) return set_error("%s: type %d (0 f32, 1 f16, 2 bf16)", who, type);
    const long long width = (long long)pool->kv_heads * pool->head_dim;
    if (pdim < 0 || pdim % 8 || pdim > pool->head_dim || (pdim > 0 && !freq) || (uintptr_t)freq % 4)
        return set_error("%s: pdim %d (a multiple of 8 up to head_dim, with its frequencies)", who, pdim);
    if (batch->rows == 0) return 0;
    if (!k || !v) return set_error("%s: null rows", who);
    if (batch->rows > 1 && (ldk < width || ldv < width))
        return set_error("%s: row strides %lld and %lld under %lld", who, ldk, ldv, width);
    const int size = type == T_F32 ? 4 : 2;
    if ((uintptr_t)k % size || (uintptr_t)v % size) return set_error("%s: unaligned rows", who);
    if (pool->kv_heads > 65535) return set_error("%s: %d KV heads", who, pool->kv_heads);
    const AppendArgs a{pool_of(pool), batch_of(batch), k, v, ldk, ldv, rows_aligned(k, ldk, size), rows_aligned(v, ldv, size),
                       freq, freq ? pdim : 0, 1, device_error_ptr()};
    const cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t e = type == T_F32   ? launch<float>(a, s)
                          : type == T_F16 ? launch<__half>(a, s)
                                          : launch<__nv_bfloat16>(a, s);
    return e == cudaSuccess ? 0 : cuda_fail(who, e);
}
