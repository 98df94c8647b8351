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
// What bounds it: bytes (each value read once, one byte written) for prompts, the chain of
// dependent loads (sequence -> page -> row) for steps. A unit of work is one (block, KV head, keys
// or values): one CTA of 4 warps, a warp per row, a row's unit of 8 values in one thread's
// registers, so the block's amax is a max in registers, one shuffle tree and one exchange between
// the warps; the bytes meet in shared memory and leave as 16-byte stores.
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

struct AppendArgs {
    Pool pool;
    Batch b;
    const void *k, *v;
    long long ldk, ldv;
    int kvec, vvec;
    const float *freq;
    int pdim;
    int *err;
};

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// e4m3 of a and b (low byte a); a NaN is stored as 0: the block's scale tells of it
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
    if (!(a == a)) a = 0.f;
    if (!(b == b)) b = 0.f;
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float e4m3_f32(uint32_t byte) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}

// 16-byte piece of the staging tile of values, spread so that a warp's 4-byte writes (dims 4 or 8
// apart) meet fewer banks
__device__ __forceinline__ int vpiece(int d) { return d ^ ((d >> 3) & 7); }

template <typename T, int HD>
__global__ void __launch_bounds__(AP_THREADS) append_kernel(const AppendArgs a) {
    constexpr int U = HD / 8;            // units of a row, one per lane (hd 256) or fewer
    constexpr int PIECES = HD;           // 16-byte pieces of a block
    __shared__ __align__(16) uint8_t tile[BLOCK * HD];
    __shared__ int who[3];               // sequence, its first row, its rows
    __shared__ float wmax[AP_WARPS];
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int unit = blockIdx.x, head = blockIdx.y;
    const bool keys = blockIdx.z == 0;
    // Units of sequence s: row0[s] / 16 + 2 s up to the next one's; n rows touch at most
    // n / 16 + 2 blocks, so each sequence's blocks fit.
    if (threadIdx.x == 0) who[0] = -1;
    __syncthreads();
    for (int s = threadIdx.x; s < a.b.nseq; s += AP_THREADS) {
        const int r0 = __ldg(a.b.row0 + s), r1 = __ldg(a.b.row0 + s + 1);
        if (r0 / BLOCK + 2 * s <= unit && unit < r1 / BLOCK + 2 * s + 2 && r1 > r0) {
            who[0] = s;
            who[1] = r0;
            who[2] = r1 - r0;
        }
    }
    __syncthreads();
    const int s = who[0];
    if (s < 0) return;
    const int r0 = who[1], n = who[2];
    const int len = __ldg(a.b.kv_len + s), first = len - n;
    const int blk = first / BLOCK + (unit - r0 / BLOCK - 2 * s);   // block of the sequence
    if (first >= 0 && blk * BLOCK >= len) return;
    const int page_at = blk / (a.pool.page_tokens / BLOCK);
    int page = -1;
    if (first >= 0 && blk >= 0 && r0 >= 0 && r0 + n <= a.b.rows && page_at < a.b.max_pages)
        page = __ldg(a.b.table + (size_t)s * a.b.max_pages + page_at);
    if (page < 0 || page >= a.pool.pages) {   // the same for every thread
        if (threadIdx.x == 0 && a.err) atomicExch(a.err, DEV_BAD_INDEX);
        return;
    }
    const size_t bi = block_index(a.pool, page, head, blk % (a.pool.page_tokens / BLOCK));
    uint8_t *dst = (keys ? a.pool.k : a.pool.v) + bi * (BLOCK * HD);
    float *scale = (keys ? a.pool.ks : a.pool.vs) + bi;
    const int lo = max(first - blk * BLOCK, 0), hi = min(len - blk * BLOCK, BLOCK);   // the call's rows of the block
    // earlier rows and their scale, on their way while the new rows come in
    uint4 old[PIECES / AP_THREADS + (PIECES % AP_THREADS != 0)];
    float d_old = 0.f;
    if (lo > 0) {
        d_old = *scale;
#pragma unroll
        for (int i = 0; i < (PIECES + AP_THREADS - 1) / AP_THREADS; i++) {
            const int pc = i * AP_THREADS + threadIdx.x;
            if (pc < PIECES) old[i] = reinterpret_cast<const uint4 *>(dst)[pc];
        }
    }
    // warp w: rows 2w, 2w + 1, 2w + 8, 2w + 9, which are bytes 4w .. 4w + 3 of a value dim
    float x[AP_ROWS][8];
    float mx = 0.f;
    const int pdim = keys && a.freq ? a.pdim : 0;
#pragma unroll
    for (int i = 0; i < AP_ROWS; i++) {
        const int r = 2 * warp + (i & 1) + 8 * (i >> 1);
        float p[4] = {0.f, 0.f, 0.f, 0.f}, q[4] = {0.f, 0.f, 0.f, 0.f};
        if (r >= lo && r < hi && lane < U) {
            const int row = r0 + blk * BLOCK + r - first;
            const T *src = keys ? (const T *)a.k + (size_t)row * a.ldk : (const T *)a.v + (size_t)row * a.ldv;
            load_unit<T>(src + (size_t)head * HD, lane, pdim, keys ? a.kvec : a.vvec, p, q);
            if (lane < pdim / 8) {
                float c[4], sn[4];
#pragma unroll
                for (int e = 0; e < 4; e++) angle(blk * BLOCK + r, __ldg(a.freq + 4 * lane + e), c[e], sn[e]);
                rotate_unit(p, q, c, sn);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[i][e] = p[e];
            x[i][4 + e] = q[e];
            mx = max_nan(mx, max_nan(fabsf(p[e]), fabsf(q[e])));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) wmax[warp] = mx;
    __syncthreads();
    mx = max_nan(max_nan(wmax[0], wmax[1]), max_nan(wmax[2], wmax[3]));
    float d = max_nan(__fdiv_rn(mx, E4M3_MAX), SCALE_MIN);
    if (lo > 0) d = max_nan(d, d_old);
    if (lo > 0) {   // earlier rows, rounded again where the scale grew; 0 elsewhere
        const float ratio = d > d_old ? __fdiv_rn(d_old, d) : 1.0f;
#pragma unroll
        for (int i = 0; i < (PIECES + AP_THREADS - 1) / AP_THREADS; i++) {
            const int pc = i * AP_THREADS + threadIdx.x;
            if (pc >= PIECES) continue;
            // keys: piece = (8-token group, 16-dim chunk, token): one token; values: one dim's 16 tokens
            const int ktok = 8 * (pc / (HD / 2)) + (pc & 7);
            uint32_t w[4] = {old[i].x, old[i].y, old[i].z, old[i].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t v = 0;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t pr = (w[j] >> (16 * h)) & 0xffffu;
                    const int t0 = keys ? ktok : order(4 * j + 2 * h), t1 = keys ? ktok : order(4 * j + 2 * h + 1);
                    uint32_t np = ratio == 1.0f ? pr : e4m3x2(__fmul_rn(e4m3_f32(pr & 0xffu), ratio),
                                                             __fmul_rn(e4m3_f32(pr >> 8), ratio));
                    if (t0 >= lo) np &= 0xff00u;
                    if (t1 >= lo) np &= 0x00ffu;
                    v |= np << (16 * h);
                }
                w[j] = v;
            }
            reinterpret_cast<uint4 *>(tile)[keys ? pc : vpiece(pc)] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncthreads();
    }
    // the new rows (all of the tile when nothing earlier is in the block)
    const float inv = __fdiv_rn(1.0f, d);
    int d0 = 0, d1 = 0;
    unit_dims(lane, pdim, d0, d1);
    if (lane < U) {
        uint32_t q[AP_ROWS][4];   // e4m3 pairs: dims d0, d0 + 1 | d0 + 2, d0 + 3 | d1 .. | ..
#pragma unroll
        for (int i = 0; i < AP_ROWS; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) q[i][e] = e4m3x2(__fmul_rn(x[i][2 * e], inv), __fmul_rn(x[i][2 * e + 1], inv));
        if (keys) {
#pragma unroll
            for (int i = 0; i < AP_ROWS; i++) {
                const int r = 2 * warp + (i & 1) + 8 * (i >> 1);
                if (r < lo) continue;
                uint8_t *row = tile + (r >> 3) * (8 * HD) + (r & 7) * 16;
                *reinterpret_cast<uint32_t *>(row + (d0 >> 4) * 128 + (d0 & 15)) = q[i][0] | (q[i][1] << 16);
                *reinterpret_cast<uint32_t *>(row + (d1 >> 4) * 128 + (d1 & 15)) = q[i][2] | (q[i][3] << 16);
            }
        } else {
            uint32_t keep = 0;   // bytes that hold earlier rows
#pragma unroll
            for (int i = 0; i < AP_ROWS; i++)
                if (2 * warp + (i & 1) + 8 * (i >> 1) < lo) keep |= 0xffu << (8 * i);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int sh = 8 * (e & 1);
                uint32_t w = 0;
#pragma unroll
                for (int i = 0; i < AP_ROWS; i++) w |= ((q[i][e >> 1] >> sh) & 0xffu) << (8 * i);
                uint32_t *at = reinterpret_cast<uint32_t *>(tile + 16 * vpiece(e < 4 ? d0 + e : d1 + e - 4)) + warp;
                *at = keep ? (*at & keep) | (w & ~keep) : w;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < (PIECES + AP_THREADS - 1) / AP_THREADS; i++) {
        const int pc = i * AP_THREADS + threadIdx.x;
        if (pc < PIECES)
            reinterpret_cast<uint4 *>(dst)[pc] = reinterpret_cast<const uint4 *>(tile)[keys ? pc : vpiece(pc)];
    }
    if (threadIdx.x == 0) *scale = d;
}

template <typename T>
cudaError_t launch(const AppendArgs &a, cudaStream_t s) {
    const dim3 grid(a.b.rows / BLOCK + 2 * a.b.nseq, a.pool.kv_heads, 2);
    if (a.pool.hd == 256) return launch_pdl(append_kernel<T, 256>, grid, dim3(AP_THREADS), 0, s, a);
    if (a.pool.hd == 128) return launch_pdl(append_kernel<T, 128>, grid, dim3(AP_THREADS), 0, s, a);
    return launch_pdl(append_kernel<T, 64>, grid, dim3(AP_THREADS), 0, s, a);
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
    if (pdim < 0 || pdim % 8 || pdim > pool->head_dim || (pdim > 0 && !freq))
        return set_error("%s: pdim %d (a multiple of 8 up to head_dim, with its frequencies)", who, pdim);
    if (batch->rows == 0) return 0;
    if (!k || !v) return set_error("%s: null rows", who);
    if (batch->rows > 1 && (ldk < width || ldv < width))
        return set_error("%s: row strides %lld and %lld under %lld", who, ldk, ldv, width);
    const int size = type == T_F32 ? 4 : 2;
    if ((uintptr_t)k % size || (uintptr_t)v % size) return set_error("%s: unaligned rows", who);
    if (pool->kv_heads > 65535) return set_error("%s: %d KV heads", who, pool->kv_heads);
    AppendArgs a{pool_of(pool), batch_of(batch), k, v, ldk, ldv, rows_aligned(k, ldk, size), rows_aligned(v, ldv, size),
                 freq, freq ? pdim : 0, device_error_ptr()};
    const cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t e = type == T_F32   ? launch<float>(a, s)
                          : type == T_F16 ? launch<__half>(a, s)
                                          : launch<__nv_bfloat16>(a, s);
    return e == cudaSuccess ? 0 : cuda_fail(who, e);
}
