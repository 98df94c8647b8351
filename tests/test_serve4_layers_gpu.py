"""spk.serve.PagedScorer over the paged 4-bit cache, layer by layer: what each layer's append and attention make of the projections
that they are given, against a 64-bit restatement of the decoder (model.rs:475-560) over the rows as the cache has them.

The projections' own outputs are taken as they are, so nothing but the two calls is between the sides, and the bounds are theirs.
A rotated key is off by f32 rounding before its codes, under 2^-20 of its pair's length: the stored code is right for some value within
that. Attention over the cached values, against the sum W = sum_j p_j |V_j|: weights of two f16 terms 2^-21, the scores' sums, queries
of two f16 terms and the queries' rotation 2^-20 S each with S the largest sum_d size_d |K_d| scale of the row (size: the length of a query's
rotated pair), 2^-22 for each of at most 64 + n / 64 additions, the gate's exponential and the division 2^-20, weights under 2^-35 of the
largest, half of f32's unit."""
import numpy as np
import pytest

from spk.model import small_config, synth_weights

pytestmark = pytest.mark.gpu
HAVE = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
EDGES = [(0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)]   # up at the tie


class Listening:
    """A matrix of the scorer that keeps a copy of what went in or came out."""

    def __init__(self, inner, log, name, side):
        self.inner, self.log, self.name, self.side = inner, log, name, side

    def __call__(self, x, out, *a, **kw):
        if self.side == "in":
            self.log[self.name] = x.clone()
        self.inner(x, out, *a, **kw)
        if self.side == "out":
            self.log[self.name] = out.clone()
        return out


def listened(sc):
    logs = []
    for mats, _, _ in sc.layers:
        log = {}
        for name, side in (("qkv", "out"), ("attn_gate", "out"), ("out", "in")):
            mats[name] = Listening(mats[name], log, name, side)
        logs.append(log)
    return logs


def rotated(x, pos, theta, dims):
    """[rows][heads][hd] in 64 bits: (rotated, its pairs' lengths)."""
    import torch

    i = np.arange(0, dims, 2, dtype=np.float32)
    freq = (np.float32(1) / np.power(np.float32(theta), i / np.float32(dims))).astype(np.float32)
    ang = torch.from_numpy((np.array(pos, np.float32)[:, None] * freq[None]).astype(np.float64)).to(x.device)[:, None]
    c, s, h = ang.cos(), ang.sin(), dims // 2
    y, size = x.clone(), x.abs()
    y[..., :h], y[..., h:dims] = x[..., :h] * c - x[..., h:dims] * s, x[..., h:dims] * c + x[..., :h] * s
    size[..., :h] = size[..., h:dims] = torch.hypot(x[..., :h], x[..., h:dims])
    return y, size


def rows_of(cache, pages, n, side):
    """(code magnitudes, signs, scales, values) of the first n tokens of a sequence, [n][kv][hd], 64 bits."""
    import torch

    pool, b = (cache.k_pool, cache.k_scale) if side == "k" else (cache.v_pool, cache.v_scale)
    at = torch.tensor(pages, dtype=torch.long, device=pool.device)
    flat = lambda t: t[at].transpose(1, 2).reshape(-1, cache.kv_heads, t.shape[-1])[:n]  # noqa: E731
    pool, b = flat(pool), flat(b)
    code = torch.stack([pool & 15, pool >> 4], -1).flatten(-2)
    d = (b.to(torch.int16) << 7).view(torch.float16).double().repeat_interleave(16, -1)
    mag = torch.tensor(HAVE, dtype=torch.float64, device=pool.device)[(code & 7).long()]
    return code & 7, code >> 3, d, torch.where(code > 7, -mag, mag) * d


def check_layer(cfg, full, log, cache, table, seqs, len_before):
    import torch

    theta, part = (cfg.rope_theta_full, cfg.rope_partial_full) if full else (cfg.rope_theta_slide, cfg.rope_partial_slide)
    dims, window = int(cfg.head_dim * part), 0 if full else cfg.window
    H, KV, D, at = cfg.heads, cfg.kv_heads, cfg.head_dim, 0
    for s, ids in seqs.items():
        n, before = len(ids), len_before.get(s, 0)
        if not n:
            continue
        rows = log["qkv"][at:at + n].double()
        pos = list(range(before, before + n))
        q, qsize = rotated(rows[:, :cfg.q_dim].reshape(n, H, D), pos, theta, dims)
        k, ksize = rotated(rows[:, cfg.q_dim:cfg.q_dim + cfg.kv_dim].reshape(n, KV, D), pos, theta, dims)
        v = rows[:, cfg.q_dim + cfg.kv_dim:].reshape(n, KV, D)
        L = before + n
        cached = {}
        for side, x, size in (("k", k, ksize), ("v", v, None)):
            code, sign, d, value = rows_of(cache, table.held[s], L, side)
            cached[side] = value
            code, sign, d = code[before:], sign[before:], d[before:]
            slack = 0 if size is None else 2.0 ** -20 * size
            count = lambda a: sum(((a >= e * d) if up else (a > e * d)).to(torch.uint8) for e, up in EDGES)  # noqa: E731
            assert ((code >= count((x.abs() - slack).clamp(min=0))) & (code <= count(x.abs() + slack))).all(), side
            sure = (code > 0) & (x.abs() > slack)
            assert (sign[sure] == (x < 0)[sure]).all(), side
            # the scale: within half of its last of 4 bits of amax / 6
            amax = x.abs().unflatten(-1, (-1, 16)).amax(-1).repeat_interleave(16, -1)
            assert ((amax / 6 - d).abs() <= d * 2.0 ** -4 + 2.0 ** -15 + 2.0 ** -20 * amax).all(), side
        kk, vv = (cached[x].repeat_interleave(H // KV, 1) for x in "kv")            # [L][H][D]
        i, j = torch.arange(before, L, device=q.device)[:, None], torch.arange(L, device=q.device)
        hide = ~((j <= i) & (j > i - window) if window else j <= i)[:, None]
        scale = D ** -0.5
        w = (torch.einsum("nhd,jhd->nhj", q, kk) * scale).masked_fill(hide, float("-inf"))
        S = (torch.einsum("nhd,jhd->nhj", qsize, kk.abs()) * scale).masked_fill(hide, 0).amax(-1, keepdim=True)
        p = torch.softmax(w, -1)
        g = torch.sigmoid(log["attn_gate"][at:at + n].double())[..., None]
        want = torch.einsum("nhj,jhd->nhd", p, vv) * g
        W = torch.einsum("nhj,jhd->nhd", p, vv.abs())
        seen = torch.einsum("nhj,jhd->nhd", (~hide).double().expand(n, H, L), vv.abs())
        tol = W * (2.0 ** -21 + 2.0 ** -19 * S + 2.0 ** -22 * (64 + L / 64) + 2.0 ** -20) + 2.0 ** -35 * p.amax(-1, keepdim=True) * seen
        got = log["out"][at:at + n].double().reshape(n, H, D)
        assert ((got - want).abs() <= tol * g + 2.0 ** -24 * want.abs() + 2.0 ** -149).all(), s
        at += n


@pytest.mark.parametrize("shape", [dict(), dict(heads=6, kv_heads=2, head_dim=64), dict(heads=4, kv_heads=2, head_dim=256, hidden=256)])
def test_every_layer_is_its_definition(cuda, shape):
    """Prompts in one call, continued by a part and by single tokens."""
    from spk.serve import PagedScorer

    cfg = small_config(**shape)
    sc = PagedScorer(cfg, synth_weights(cfg, seed=5, exact_q80=True), pages=40, page_tokens=16, device=cuda, kv_bits=4)
    logs = listened(sc)
    rng = np.random.default_rng(6)
    ids = lambda n: rng.integers(0, cfg.vocab, n).tolist()  # noqa: E731
    for new in ({"a": ids(150), "b": [7], "c": ids(33), "d": [], "e": ids(16)}, {"c": ids(20), "a": ids(1)}, {"a": ids(1), "b": ids(1), "c": ids(1), "e": ids(1)}):
        before = dict(sc.len)
        sc.forward(new)
        for full, log, cache in zip(cfg.full, logs, sc.caches):
            check_layer(cfg, full, log, cache, sc.table, new, before)


def test_both_caches_say_nearly_the_same(cuda):
    """The same rows with keys and values in 8 and in 4 bits: each is within its test's bound of the oracle's logits, so they are within both of each other."""
    from spk.serve import PagedScorer

    cfg = small_config()
    W = synth_weights(cfg, seed=3, exact_q80=True)
    rng = np.random.default_rng(1)
    seqs = {"a": rng.integers(0, cfg.vocab, 150).tolist(), "c": rng.integers(0, cfg.vocab, 33).tolist()}
    four, eight = (PagedScorer(cfg, W, pages=40, page_tokens=16, device=cuda, kv_bits=b).forward(seqs).double() for b in (4, 8))
    assert (four - eight).norm() <= 0.38 * eight.norm()
    assert (four - eight).norm() > 0          # they are not the same cache
