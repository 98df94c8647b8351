// paged_line.cuh — the line of work of the paged attention kernels (paged_attn.cu, paged4_attn.cu).
//
// All (sequence, KV head, row tile) groups of a call stand in one line, each as long as the tokens it reads plus a fixed
// cost; the line is cut into equal ranges, one per CTA. The kernels' parameters P give the batch `b`, `pool.page_tokens`,
// `pool.kv_heads`, `group` (query heads on a KV head), `window`, `err`, and takes(columns): whether the kernel has the
// sequences of so many rows per KV head.
#pragma once
#include "paged.cuh"

namespace spk {
namespace paged {
namespace {

// Lengths are in blocks and fit 32 bits (the entry point refuses a batch that could not).
struct Seq {
    int r0, n, len, tiles;            // rows of the call, cached tokens, row tiles
    int c, rate;                      // group j takes up to (c + rate (j + 1) / 2^15) / 16 blocks: R / group tokens more each
};
template <class P>
__device__ __forceinline__ Seq seq_of(const P &a, int s, int R) {
    Seq q;
    q.r0 = __ldg(a.b.row0 + s);
    q.n = __ldg(a.b.row0 + s + 1) - q.r0;
    q.len = max(__ldg(a.b.kv_len + s), 0);   // under 0 there is nothing to see either; positions do not leave 32 bits
    const long long room = (long long)a.b.max_pages * a.pool.page_tokens;
    if (q.n != 0 && (q.n < 0 || q.r0 < 0 || q.r0 > a.b.rows - q.n || q.len > room)) {   // not a batch: nothing is read
        if (a.err) atomicExch(a.err, DEV_BAD_INDEX);
        q.n = 0;
    }
    if (!a.takes((long long)q.n * a.group)) q.n = 0;
    q.tiles = (int)(((long long)q.n * a.group + R - 1) / R);
    const bool windowed = a.window > 0 && a.window < q.len;
    if (windowed || q.len < q.n) {    // every group alike: a window and a tile's rows, or the whole sequence
        q.c = windowed ? min(q.len, a.window + (R + a.group - 1) / a.group + BLOCK) : max(0, q.len);
        q.rate = 0;
    } else {
        q.c = q.len - q.n + 2;
        q.rate = (R * 32768 + a.group - 1) / a.group;
    }
    return q;
}
// Length of groups 0 .. j - 1: the tokens' sum (group i sees at most len - n + (i + 1) R / group + 1 of them), a
// partial block each, the fixed costs. 64 bits hold it: the entry point's bound is 2^35 on j^2 R / group.
__device__ __forceinline__ uint32_t before(const Seq &q, uint32_t j, int cost) {
    const unsigned long long t = (unsigned long long)j * q.c + ((unsigned long long)q.rate * j * (j + 1) >> 16);
    return (uint32_t)(t / BLOCK) + j * (cost + 2);
}

struct Seg {
    int s, r0, kvh;                   // sequence, its first row, KV head
    int c0, c1, pos0;                 // columns (token * group + head) of the tile, c1 the last; position of row 0
    int p_lo, p_hi, see0;             // first and last row's positions, first token that a row sees
    int start, k0, k1;                // first token of tile 0; this CTA's tiles
    int f0, f1;                       // the CTAs that share the group
    int nblk;                         // blocks from start that some row sees (0: nothing is seen)
};

// Walks a CTA's range of the line.
struct Walk {
    uint32_t x0, x1, chunk, base;     // range; the group's place
    int s, kvh, j;
    Seq q;
};
// The group of sequence s that holds the start of the CTA's range.
template <class P>
__device__ __forceinline__ void walk_at(const P &a, const uint32_t *pre, int s, int R, int cost, Walk &w) {
    w.s = s;
    w.q = seq_of(a, s, R);
    const uint32_t per = before(w.q, w.q.tiles, cost), in = w.x0 - pre[s];
    w.kvh = in / per;
    const uint32_t rem = in - w.kvh * per;
    int a0 = 0, a1 = w.q.tiles;       // the last group with before <= rem
    while (a1 - a0 > 1) {
        const int mid = (a0 + a1) >> 1;
        if (before(w.q, mid, cost) <= rem) a0 = mid;
        else a1 = mid;
    }
    w.j = a0;
    w.base = pre[s] + w.kvh * per + before(w.q, a0, cost);
}
// The next group of which this CTA has tiles (of TB blocks).
template <int TB, class P>
__device__ __noinline__ bool walk_next(const P &a, const uint32_t *pre, int R, int cost, Walk &w, Seg &g) {
    while (w.base < w.x1) {
        const int G = a.group, c0 = w.j * R, c1 = min(c0 + R, w.q.n * G) - 1, pos0 = w.q.len - w.q.n;
        const int p_lo = pos0 + c0 / G, p_hi = pos0 + c1 / G;
        const int see0 = a.window > 0 && p_lo >= a.window ? p_lo + 1 - a.window : 0, b0 = see0 / BLOCK;
        const int nblk = p_hi < 0 ? 0 : p_hi / BLOCK + 1 - b0;
        const int nt = max(1, (nblk + TB - 1) / TB);   // one empty tile where nothing is seen
        const uint32_t t0 = w.base + cost;         // tile k stands at t0 + TB k, inside the group's length
        const int d0 = (int)(w.x0 - t0), d1 = (int)(w.x1 - t0);
        const int k0 = d0 <= 0 ? 0 : (d0 + TB - 1) / TB, k1 = d1 <= 0 ? 0 : min(nt, (d1 + TB - 1) / TB);
        const bool mine = k0 < k1;
        if (mine)
            g = Seg{w.s, w.q.r0, w.kvh, c0, c1, pos0, p_lo, p_hi, see0, b0 * BLOCK, k0, k1,
                    (int)(t0 / w.chunk), (int)((t0 + (uint32_t)(TB * (nt - 1))) / w.chunk), nblk};
        const uint32_t at = before(w.q, w.j, cost);
        w.base += before(w.q, ++w.j, cost) - at;
        if (w.j == w.q.tiles) {
            w.j = 0;
            if (++w.kvh == a.pool.kv_heads) {
                w.kvh = 0;
                while (++w.s < a.b.nseq && pre[w.s + 1] == pre[w.s]) {}
                if (w.s < a.b.nseq) w.q = seq_of(a, w.s, R);
            }
        }
        if (mine) return true;
    }
    return false;
}

}  // namespace
}  // namespace paged
}  // namespace spk
