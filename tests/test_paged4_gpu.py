"""spk_paged4_append, spk_paged4_read and spk_paged4_attn against a 64-bit restatement of their definitions.

Bounds. Rows that are rounded as they are (values; keys without a norm or a rotation) have one right code and scale: equality.
A rotated or normalised key is off by f32 rounding before its rounding to 4 bits: the norm's sum, square root and two products,
cosine and sine to 2 ulp, two products and a sum, under 2^-20 of its pair's length; the stored code has to be right for some value within
that, and the scale for some amax within it. Queries: the same, and their type's rounding (half a unit).

Attention reads the cache exactly (a value is an f16 number). Its error, against the sum W = sum_j p_j |V_j| of what it adds: the weights'
rounding (f16: 2^-12 each, the sum that divides by them rounded alike, so 2^-11 together; f32: two terms, 2^-22), the scores' f32 sums and their
queries' rounding (f16 rows exact, bf16 rows exact above 2^-24 of the largest, f32 rows 2^-22 of the largest): 2^-20 S with S the largest sum_d |q_d k_d|
scale of the row, the sums of the outputs, which the tensor cores cut towards 0: 2^-22 for each of at most 64 + n / 64 additions; and the output type's half unit. With the
gate's exponential and the division 2^-20 more. Weights are f16 numbers, the largest between 2^12 and 2^15 (many rows
of a sequence: 2^10, and 2^6 for 16-bit rows), so a small one is off by half of f16's last bit, 2^-25, which is 2^-37 (2^-35, 2^-31) of the
largest: that times max p sum_j |V_j| besides."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}
HAVE = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
EDGES = [(0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)]   # up at the tie


def ttype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def freqs(dev, pdim, theta=1e4):
    from spk import paged

    return paged.rope_freq(theta, pdim, dev) if pdim else None


def check_errors():
    import spk

    return spk.lib().spk_check_device_error()


class Case:
    """A 4-bit pool with random contents where sequences have tokens and poison everywhere else, a page table in random
    order, and a batch over it."""

    def __init__(self, dev, rows, old, kv=2, hd=128, page=32, heads=None, seed=0, pages=None, scales=(95, 120)):
        import torch

        from spk import paged4

        self.dev, self.rows, self.len, self.kv, self.hd, self.page = dev, rows, [a + b for a, b in zip(rows, old)], kv, hd, page
        g = self.g = torch.Generator(device=dev)
        g.manual_seed(seed)
        need = [max(0, -(-n // page)) for n in self.len]
        total = sum(need) + 2
        order = torch.randperm(total, generator=g, device=dev).int().cpu().tolist()
        if pages:
            order = [pages - 1 - p for p in order]      # the pool's far end
        width = max(1, max(need))
        self.table = [[order.pop() for _ in range(n)] + [-1] * (width - n) for n in need]
        c = self.cache = paged4.Paged4Cache(pages or total, page, kv, hd, device=dev)
        c.k_scale.fill_(255)
        c.v_scale.fill_(255)
        for s, n in enumerate(self.len):
            for i, p in enumerate(self.table[s][:need[s]]):
                m = min(page, n - i * page)
                for pool, scale in ((c.k_pool, c.k_scale), (c.v_pool, c.v_scale)):
                    pool[p].random_(0, 256, generator=g)
                    scale[p, :, :m] = torch.randint(*scales, (kv, m, hd // 16), generator=g, device=dev).to(torch.uint8)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        self.row0 = i32(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32).tolist())
        self.kv_len, self.tab = i32(self.len), i32(self.table)
        self.heads = heads or kv
        self.batch = paged4.Paged4Batch(c, self.row0, self.kv_len, self.tab, rows=sum(rows), heads=self.heads)

    def randn(self, width, typ, scale=1.0):
        import torch

        return torch.randn(sum(self.rows), width, generator=self.g, device=self.dev).mul_(scale).to(ttype(typ))

    def places(self):
        """(page, token of the page) of every row."""
        at = [(self.table[s][p // self.page], p % self.page) for s, (n, L) in enumerate(zip(self.rows, self.len)) for p in range(L - n, L)]
        return [p for p, _ in at], [o for _, o in at]

    def positions(self):
        return [p for n, L in zip(self.rows, self.len) for p in range(L - n, L)]

    def cached(self, s, name):
        """[kv][len][hd] of sequence s, in 64 bits."""
        import torch

        c, n = self.cache, self.len[s]
        take = torch.tensor(self.table[s][:-(-n // self.page)], dtype=torch.long, device=self.dev)
        pool, b = (c.k_pool, c.k_scale) if name == "k" else (c.v_pool, c.v_scale)
        return numbers(pool[take], b[take]).transpose(0, 1).reshape(self.kv, -1, self.hd)[:, :n]


def numbers(pool, b):
    import torch

    have = torch.tensor(HAVE + [-x for x in HAVE], dtype=torch.float64, device=pool.device)
    x = torch.stack([have[(pool & 15).long()], have[(pool >> 4).long()]], -1).flatten(-2)
    return x * (b.to(torch.int16) << 7).view(torch.float16).double().repeat_interleave(16, -1)


# ------------------------------------------------------------------------------------------ append

def scale_byte(amax):
    """The byte of the number of 4 significant bits nearest to amax / 6, ties to even, in 64 bits; 255 for an infinite one."""
    import torch

    m, e = torch.frexp((amax / 6).clamp(2.0 ** -14, 10240))
    b = (torch.ldexp((m * 16).round(), e - 4).half().view(torch.int16) >> 7).to(torch.uint8)
    return torch.where(amax.isfinite(), b, torch.full_like(b, 255))


def codes(x, b, slack=None):
    """The code magnitudes of x / d by comparison with the borders; with slack, the lowest and highest that some value within it has."""
    import torch

    d = (b.to(torch.int16) << 7).view(torch.float16).double().repeat_interleave(16, -1)
    lo, hi = (x.abs(), x.abs()) if slack is None else ((x.abs() - slack).clamp(min=0), x.abs() + slack)
    count = lambda a: sum(((a >= e * d) if up else (a > e * d)).to(torch.uint8) for e, up in EDGES)  # noqa: E731
    return count(lo), count(hi)


def head_rows(x, n, hd, w, eps, pos, freq, inter):
    """(rows normalised and rotated, their pairs' lengths) in 64 bits."""
    import torch

    x = x.double().reshape(-1, n, hd)
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    size = x.abs()
    if freq is None:
        return x, size
    h = freq.numel()
    ang = (torch.tensor(pos, dtype=torch.float32, device=x.device)[:, None] * freq[None]).double()
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    i, j = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if inter else (slice(0, h), slice(h, 2 * h))
    y, size = x.clone(), size.clone()
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    size[..., i] = size[..., j] = torch.hypot(x[..., i], x[..., j])
    return y, size


def unpacked(pool):
    import torch

    return torch.stack([pool & 15, pool >> 4], -1).flatten(-2)


def check_append(c, k, v, q=None, freq=None, inter=False, wq=None, wk=None, eps=1e-6, typ="f32", exact_k=False):
    import torch

    before = [t.clone() for t in (c.cache.k_pool, c.cache.v_pool, c.cache.k_scale, c.cache.v_scale)]
    q_out = torch.full_like(q.contiguous(), 777.0) if q is not None else None
    got = c.batch.append(k, v, freq=freq, interleaved=inter, q=q, q_out=q_out, q_norm=wq, k_norm=wk, eps=eps)
    assert check_errors() == 0
    pg, off = c.places()
    pos = c.positions()
    if q is not None:
        assert got is q_out
        y, size = head_rows(q, c.heads, c.hd, wq, eps, pos, freq, inter)
        y, size = y.flatten(1), size.flatten(1)
        assert ((got.double() - y).abs() <= HALF[typ] * y.abs() + TINY[typ] + 2.0 ** -20 * size).all()
    for name, x in (("k", k), ("v", v)):
        pool, scale = (c.cache.k_pool, c.cache.k_scale) if name == "k" else (c.cache.v_pool, c.cache.v_scale)
        if name == "k":
            y, size = head_rows(x, c.kv, c.hd, wk, eps, pos, freq, inter)
        else:
            y, size = x.double().reshape(-1, c.kv, c.hd), None
        code, b = unpacked(pool[pg, :, off]), scale[pg, :, off]
        amax = y.abs().unflatten(-1, (-1, 16)).amax(-1)
        if name == "v" or exact_k or (wk is None and freq is None):
            assert torch.equal(b, scale_byte(amax)), name
            lo, hi = codes(y, b)
        else:
            slack = 2.0 ** -20 * size
            s16 = slack.unflatten(-1, (-1, 16)).amax(-1)
            assert ((b >= scale_byte(amax - s16)) & (b <= scale_byte(amax + s16))).all()
            lo, hi = codes(y, b, slack)
        real = amax.isfinite().repeat_interleave(16, -1)
        assert ((code & 7 >= lo) & (code & 7 <= hi))[real].all() and (code[~real] == 0).all(), name
        sure = (y != 0) & (lo > 0) & real
        assert ((code >> 3).bool() == (y < 0))[sure].all()
    # nothing else was touched
    for was, now in zip(before, (c.cache.k_pool, c.cache.v_pool, c.cache.k_scale, c.cache.v_scale)):
        if len(pg):
            now = now.clone()
            now[pg, :, off] = was[pg, :, off]
        assert torch.equal(was, now)


APPENDS = [
    # rows, tokens before, kv, hd, page, heads, type, pdim, interleaved, norms
    ([1], [4103], 4, 256, 64, 16, "f32", 64, False, False),
    ([1], [0], 1, 64, 16, 1, "bf16", 0, False, False),
    ([1, 0, 1, 1], [5, 9, 0, 47], 2, 128, 16, 4, "f16", 128, False, True),
    ([33, 1, 0, 16, 7], [3, 0, 2, 16, 90], 4, 256, 32, 8, "f32", 256, True, False),
    ([33, 1, 0, 16, 7], [3, 0, 2, 16, 90], 3, 64, 48, 15, "bf16", 32, False, True),
    ([130, 65], [0, 1], 2, 256, 128, 10, "bf16", 64, False, True),
    ([17, 40], [31, 0], 8, 64, 16, 8, "f16", 16, True, True),
    ([50], [100000], 2, 128, 64, 6, "f32", 64, False, True),
    ([3] * 70, list(range(70)), 1, 128, 16, 3, "f16", 32, True, False),
]


@pytest.mark.parametrize("rows,old,kv,hd,page,heads,typ,pdim,inter,norm", APPENDS)
def test_append(cuda, rows, old, kv, hd, page, heads, typ, pdim, inter, norm):
    import torch

    c = Case(cuda, rows, old, kv, hd, page, heads, seed=5)
    qkv = c.randn((heads + 2 * kv) * hd, typ)
    q, k, v = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kv) * hd], qkv[:, (heads + kv) * hd:]
    w = [torch.rand(hd, generator=c.g, device=cuda) + 0.5 for _ in "qk"] if norm else [None, None]
    check_append(c, k, v, q, freqs(cuda, pdim), inter, w[0], w[1], typ=typ)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("off,pad", [(0, 1), (1, 0), (3, 5), (8, 8)])
def test_append_takes_rows_of_any_stride_and_alignment(cuda, typ, off, pad):
    c = Case(cuda, [5, 9], [0, 3], 2, 64, 16, 4, seed=6)
    wide = c.randn(8 * 64 + off + pad, typ)[:, off:]
    check_append(c, wide[:, 256:384], wide[:, 384:512], wide[:, :256], freqs(cuda, 32), typ=typ)


def test_append_in_place_and_without_queries(cuda):
    import torch

    for kw in (dict(), dict(freq=freqs(cuda, 128)), dict(freq=freqs(cuda, 64), interleaved=True), dict(q_norm=torch.rand(128, device=cuda) + 0.5)):
        c = Case(cuda, [9, 20], [4, 0], 2, 128, 16, 6, seed=7)
        k, v, q = c.randn(256, "bf16"), c.randn(256, "bf16"), c.randn(768, "bf16")
        apart = c.batch.append(k, v, q=q, **kw)
        assert c.batch.append(k, v, q=q, q_out=q, **kw) is q and torch.equal(q, apart)
        pools = [t.clone() for t in (c.cache.k_pool, c.cache.v_pool, c.cache.k_scale, c.cache.v_scale)]
        kw.pop("q_norm", None)
        assert c.batch.append(k, v, **kw) is None
        assert all(torch.equal(a, b) for a, b in zip(pools, (c.cache.k_pool, c.cache.v_pool, c.cache.k_scale, c.cache.v_scale)))


def test_values_on_and_beside_the_borders(cuda):
    """f32 values at each border times each scale, a unit under and over it: the codes are those of exact arithmetic."""
    import torch

    mant = torch.arange(8, 16, dtype=torch.float64, device=cuda) / 8
    rows = []
    for e in (-14, -13, 0, 7, 13):
        for m in mant.tolist():
            d = m * 2.0 ** e
            if d > 10240:
                continue
            for nudge in (-1, 0, 1):
                x = torch.tensor([t * d for t, _ in EDGES] + [6 * d] + [t * d for t in HAVE], dtype=torch.float32, device=cuda)
                x[:7] = torch.nextafter(x[:7], torch.full_like(x[:7], float("inf") if nudge > 0 else 0.0)) if nudge else x[:7]
                rows.append(x * torch.where(torch.arange(16, device=cuda) % 3 == 1, -1.0, 1.0))
    # amax on and beside the borders between two scales
    for e in (-14, 3, 12):
        for m in range(17, 32, 2):
            for nudge in (-1, 0, 1):
                a = torch.tensor(6 * m / 16 * 2.0 ** e, dtype=torch.float32, device=cuda)
                a = torch.nextafter(a, torch.full_like(a, float("inf") if nudge > 0 else 0.0)) if nudge else a
                rows.append(torch.cat([a[None], a * torch.linspace(-0.9, 0.9, 15, device=cuda)]))
    # next to nothing, and more than there is
    for a in (0.0, 1e-45, 1e-30, 2.0 ** -16, 6 * 2.0 ** -14, 61439.0, 61440.0, 63000.0, 65504.0, 1e30, 3.4e38):
        rows.append(torch.linspace(-1, 1, 16, device=cuda) * a)
    while len(rows) % 8:
        rows.append(torch.zeros(16, device=cuda))
    x = torch.cat(rows).reshape(-1, 128)
    for typ in ("f32", "bf16", "f16"):
        c = Case(cuda, [x.shape[0]], [0], 1, 128, 16, 1)
        t = x.to(ttype(typ))
        if typ == "f16":
            t = t.clamp(-65504, 65504)
        check_append(c, t.flip(0).contiguous(), t, typ=typ)


def test_append_of_no_numbers_poisons_their_group_alone(cuda):
    import torch

    c = Case(cuda, [6], [2], 2, 64, 16, 2)
    k, v = c.randn(128, "f32"), c.randn(128, "f32")
    v[0, 3], v[1, 40], k[2, 70], k[3, 127] = float("nan"), float("inf"), float("-inf"), float("nan")
    c.batch.append(k, v)
    pg, off = c.places()
    kb, vb = c.cache.k_scale[pg, :, off].reshape(6, 8), c.cache.v_scale[pg, :, off].reshape(6, 8)
    assert (kb == 255).nonzero().tolist() == [[2, 4], [3, 7]]
    assert (vb == 255).nonzero().tolist() == [[0, 0], [1, 2]]
    rk, rv = c.batch.read(dtype=torch.float32)
    assert rk.isnan().reshape(6, 8, 16).any(-1).nonzero().tolist() == [[2, 4], [3, 7]]
    assert rv.isnan().reshape(6, 8, 16).all(-1).nonzero().tolist() == [[0, 0], [1, 2]]


# -------------------------------------------------------------------------------------------- read

@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,old,kv,hd,page", [([1], [0], 1, 64, 16), ([40], [4000], 4, 256, 64), ([33, 0, 5, 300], [0, 4, 100, 9], 3, 128, 48), ([7] * 90, [1] * 90, 2, 64, 16)])
def test_read(cuda, typ, rows, old, kv, hd, page):
    import torch

    c = Case(cuda, rows, old, kv, hd, page, scales=(8, 227))
    pg, off = c.places()
    want = [numbers(p[pg, :, off], b[pg, :, off]).flatten(1) for p, b in ((c.cache.k_pool, c.cache.k_scale), (c.cache.v_pool, c.cache.v_scale))]
    for got, w in zip(c.batch.read(dtype=ttype(typ)), want):
        assert got.dtype == ttype(typ) and torch.equal(got.double(), w)
    # rows that lie apart, at odd places; the columns between stay
    wide = torch.full((sum(rows), 2 * kv * hd + 7), 5.0, dtype=ttype(typ), device=cuda)
    k, v = wide[:, 1:1 + kv * hd], wide[:, 4 + kv * hd:4 + 2 * kv * hd]
    c.batch.read(k, v)
    assert torch.equal(k.double(), want[0]) and torch.equal(v.double(), want[1])
    assert (wide[:, [0, 1 + kv * hd, 3 + kv * hd, -1]] == 5).all()
    only = c.batch.read(v=v)[0]
    assert only.dtype == v.dtype and torch.equal(only.double(), want[0])
    ka, sa, va, sv = c.batch.parts()
    assert torch.equal(ka.double() * sa.double().repeat_interleave(16, -1), want[0])
    assert torch.equal(va.double() * sv.double().repeat_interleave(16, -1), want[1])
    assert torch.equal(sv.view(torch.int16) >> 7, c.cache.v_scale[pg, :, off].flatten(1).to(torch.int16))
    assert check_errors() == 0


# --------------------------------------------------------------------------------------- attention

def want_attention(c, q, window=0, gate=None, scale=0.0):
    """(output, bound without the type's rounding) in 64 bits."""
    import torch

    scale = scale or c.hd ** -0.5
    two = q.dtype == torch.float32
    out, tol, at = [], [], 0
    for s, (n, L) in enumerate(zip(c.rows, c.len)):
        if n == 0:
            continue
        ks, vs = c.cached(s, "k"), c.cached(s, "v")
        bad = ~(vs.isfinite().all(-1) & ks.isfinite().all(-1))     # [kv][j]: scale bytes from 248 on are no numbers
        vs = torch.where(vs.isfinite(), vs, torch.zeros_like(vs))
        ks = torch.where(ks.isfinite(), ks, torch.zeros_like(ks))
        qq = q[at:at + n].double().reshape(n, c.kv, c.heads // c.kv, c.hd)
        i, j = torch.arange(L - n, L, device=q.device)[:, None], torch.arange(L, device=q.device)
        see = (j <= i) & (j > i - window) if window else j <= i
        w = torch.einsum("nkgd,kjd->nkgj", qq, ks) * scale
        size = torch.einsum("nkgd,kjd->nkgj", qq.abs(), ks.abs()) * abs(scale)
        hide = ~see[:, None, None]
        w = w.masked_fill(hide, float("-inf"))
        p = torch.softmax(w, -1)
        p = torch.where(hide, torch.zeros_like(p), p)       # a row that sees nothing: 0
        o = torch.einsum("nkgj,kjd->nkgd", p, vs)
        W = torch.einsum("nkgj,kjd->nkgd", p, vs.abs())
        hit = (see[:, None] & bad[None]).any(-1)            # [n][kv]
        o[hit] = float("nan")
        S = size.masked_fill(hide, 0).amax(-1, keepdim=True)
        t = W * ((2.0 ** -21 if two else 2.0 ** -11) + 2.0 ** -20 * S + 2.0 ** -22 * (64 + L / 64) + 2.0 ** -20)
        seen = torch.einsum("nj,kjd->nkd", see.double(), vs.abs())
        t = t + (2.0 ** -35 if two else 2.0 ** -31) * p.amax(-1, keepdim=True) * seen[:, :, None]
        out.append(o.reshape(n, c.heads, c.hd))
        tol.append(t.reshape(n, c.heads, c.hd))
        at += n
    o, t = torch.cat(out), torch.cat(tol)
    if gate is not None:
        sg = torch.sigmoid(gate.double())[..., None]
        o, t = o * sg, t * sg
    return o.flatten(1), t.flatten(1)


def check_attention(c, q, typ, window=0, gate=None, scale=0.0, out=None):
    import torch

    got = c.batch.attention(q, out, window=window, gate=gate, scale=scale)
    assert check_errors() == 0
    want, tol = want_attention(c, q, window, gate, scale)
    if not want.isnan().any():
        off = (got.double() - want).abs()
        bound = tol + HALF[typ] * want.abs() + TINY[typ]
        assert (off <= bound).all(), (off / bound).max()
        return got
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    assert ((got.double() - want).abs()[ok] <= (tol + HALF[typ] * want.abs() + TINY[typ])[ok]).all()
    return got


ATTNS = [
    # rows, tokens before, kv, hd, page, heads, window
    ([1], [0], 1, 64, 16, 1, 0),
    ([1], [4103], 4, 256, 64, 16, 512),
    ([1, 1, 0, 1, 1], [0, 15, 7, 16, 2000], 2, 128, 32, 8, 0),
    ([1] * 40, [37 * i for i in range(40)], 2, 256, 48, 8, 0),
    ([3, 8, 1, 0, 5], [0, 100, 31, 8, 64], 2, 64, 16, 10, 0),
    ([8, 8, 8], [500, 3, 129], 4, 128, 32, 32, 0),
    ([70, 1, 33], [0, 300, 64], 2, 256, 64, 6, 0),
    ([200], [0], 1, 128, 16, 5, 0),
    ([150, 9], [77, 130], 2, 64, 32, 16, 40),
    ([300], [1000], 1, 256, 128, 4, 17),
    ([64, 40], [3, 0], 3, 128, 16, 3, 1),
    ([5], [40], 1, 64, 16, 40, 0),
    # few rows and many in one call, both sides of where another kernel has them
    ([70, 1, 33, 5, 90, 0, 22], [0, 300, 64, 7, 1000, 5, 2], 2, 256, 64, 6, 0),
    ([70, 1, 33, 5, 90, 0, 22], [0, 300, 64, 7, 1000, 5, 2], 3, 128, 16, 9, 0),
    ([65, 64, 63, 1, 200, 2], [31, 32, 33, 0, 15, 900], 2, 64, 48, 2, 0),
    ([40, 130, 17, 3, 1, 66], [900, 5, 0, 64, 128, 300], 2, 128, 32, 8, 50),
    ([129], [5000], 2, 256, 16, 6, 0),
    ([33] * 20, [70 * i for i in range(20)], 1, 256, 32, 4, 0),
    ([257, 300], [0, 1], 8, 64, 16, 8, 7),
    ([3], [40], 1, 64, 16, 200, 0),
    ([9, 2], [100, 3], 1, 128, 16, 129, 30),
]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,old,kv,hd,page,heads,window", ATTNS)
def test_attention(cuda, rows, old, kv, hd, page, heads, window, typ):
    c = Case(cuda, rows, old, kv, hd, page, heads, seed=11)
    q = c.randn(heads * hd, typ, 0.4)
    check_attention(c, q, typ, window)
    check_attention(c, c.randn(heads * hd, typ, 3.0), typ, window, gate=c.randn(heads, typ), scale=0.01)


def test_long_context(cuda):
    for typ, hd, kv, heads in (("f32", 256, 2, 8), ("bf16", 128, 1, 8), ("f16", 64, 2, 2)):
        c = Case(cuda, [1], [70000], kv, hd, 128, heads, seed=2)
        check_attention(c, c.randn(heads * hd, typ, 0.3), typ)
        for rows in (40, 300):
            c = Case(cuda, [rows], [20000], kv, hd, 128, heads, seed=3)
            check_attention(c, c.randn(heads * hd, typ, 0.3), typ)


@pytest.mark.parametrize("typ", ["f32", "f16"])
@pytest.mark.parametrize("size", [0.05, 30.0])
@pytest.mark.parametrize("rows, nseq", [(1, 320), (128, 160)])
def test_values_of_one_sign_in_a_long_context(cuda, rows, nseq, size, typ):
    """Matrix instructions that cut their sums towards 0 are short by up to a unit, 2^-23 of the sum, each. So many sequences over the same
    pages that a block of threads has whole ones to itself. Few rows: blocks of 16 tokens by themselves (two instructions of f32) and
    f32 additions of 1024 of them a warp, each off by 2^-24 of the sum either way: their errors' root of 1024, four times over, and 2^-22. Many rows: 2048 tokens
    (f32; 16-bit types 16384) an accumulator, 256 (1024) instructions. Beside that as in want_attention: 2^-21 (2^-11) for the weights, 2^-20 for the
    scores and as much for the division, what the smallest weights lose, half a unit of the type. Large queries: keys that grow along the
    context, so that the largest score so far keeps growing, too."""
    import torch

    from spk import paged4

    n, page, hd = 65536, 128, 64
    c = paged4.Paged4Cache(n // page, page, 1, hd, device=cuda)
    g = torch.Generator(device=cuda)
    g.manual_seed(21)
    for pool, scale, keep in ((c.k_pool, c.k_scale, 0xff), (c.v_pool, c.v_scale, 0x77)):
        pool.random_(0, 256, generator=g)
        pool.bitwise_and_(keep)
        scale.copy_(torch.randint(95, 103, scale.shape, generator=g, device=cuda).to(torch.uint8))
    if size > 1:
        c.k_scale -= torch.linspace(30, 0, n // page, device=cuda).to(torch.uint8)[:, None, None, None]
    row0 = torch.arange(nseq + 1, dtype=torch.int32, device=cuda) * rows
    table = torch.arange(n // page, dtype=torch.int32, device=cuda)[None].expand(nseq, -1).contiguous()
    b = paged4.Paged4Batch(c, row0, torch.full((nseq,), n, dtype=torch.int32, device=cuda), table, rows=nseq * rows, heads=1)
    q = (torch.randn(nseq * rows, hd, generator=g, device=cuda) * size).to(ttype(typ))
    got = b.attention(q).double()
    assert check_errors() == 0
    k, v = (numbers(p, s)[:, 0].reshape(-1, hd) for p, s in ((c.k_pool, c.k_scale), (c.v_pool, c.v_scale)))
    cut = 4 * 1024 ** 0.5 * 2.0 ** -24 + 2.0 ** -22 if rows == 1 else (256 if typ == "f32" else 1024) * 2.0 ** -23
    for s in (0, 1, nseq // 2, nseq - 1):
        x = q[s * rows].double() * hd ** -0.5
        kk, vv = k[:n - rows + 1], v[:n - rows + 1]
        p = torch.softmax(kk @ x, 0)
        want = p @ vv
        bound = cut + (2.0 ** -21 if typ == "f32" else 2.0 ** -11) + 2.0 ** -20 * (kk.abs() @ x.abs()).max() + 2.0 ** -20 + HALF[typ]
        lost = (2.0 ** -35 if typ == "f32" else 2.0 ** -31) * p.max() * vv.sum(0)
        off = (got[s * rows] - want).abs()
        assert (off <= bound * want + lost).all(), (s, (off / want).max(), bound)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [[6, 40], [6, 150]])
def test_queries_of_any_size(cuda, rows, typ):
    """Rows of zeros, tiny and huge ones beside each other; scores past f32's range are none of an exact form's either."""
    c = Case(cuda, rows, [30, 5], 1, 128, 16, 2, seed=4)
    q = c.randn(256, typ)
    size = [0.0, 2.0 ** -14, 1.0, 100.0, 1e-3, 1e4]
    for r in range(q.shape[0]):
        q[r] *= size[r % 6]
    check_attention(c, q, typ, scale=1e-4)
    if typ != "f16":
        q = c.randn(256, typ)
        for r in range(q.shape[0]):
            q[r] *= [1e30, 1e-30, 1e-37, 1.0][r % 4]
        check_attention(c, q, typ, scale=1e-30)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [[4, 2], [90, 41], [200, 141]])
def test_poison_reaches_the_rows_that_see_it(cuda, rows, typ):
    """NaN groups of keys and of values: rows before them, of other sequences and other KV heads stay."""
    c = Case(cuda, rows, [60, 17], 2, 128, 16, 4, seed=8)
    for s, p, h, grp, side in ((0, c.len[0] - 2, 0, 3, "v"), (0, c.len[0] - 1, 1, 7, "k"), (1, 5, 1, 0, "v"), (0, 61, 1, 2, "v")):
        pool = c.cache.k_scale if side == "k" else c.cache.v_scale
        pool[c.table[s][p // 16], h, p % 16, grp] = 255 if p != 5 else 248
    q = c.randn(512, typ, 0.4)
    for window in (0, 20):
        got = check_attention(c, q, typ, window)
        assert got.isnan().any() and not got.isnan().all()


def test_scores_far_from_zero_and_one_key_that_takes_all(cuda):
    import torch

    for typ in ("f32", "f16", "bf16"):
        c = Case(cuda, [2, 90], [300, 100], 1, 64, 16, 4, seed=9)
        q = c.randn(256, typ)
        for scale in (3.0, -3.0):
            check_attention(c, q, typ, scale=scale)
        # every key alike but one, whose value is small: the others' share counts
        c.cache.k_pool.fill_(0x22)
        c.cache.k_scale[c.cache.k_scale != 255] = 112
        c.cache.k_pool[c.table[0][0], 0, 3] = 0x66
        q = torch.full_like(q, 0.25)
        check_attention(c, q, typ)


def test_rows_that_see_nothing_and_rows_of_nobody(cuda):
    """kv_len under the call's rows: the first ones sit before the sequence and see nothing. Rows behind the last sequence stay."""
    import torch

    from spk import paged4

    for n in (3, 70, 150):
        c = Case(cuda, [n, n], [0, 20], 2, 64, 16, 4, seed=10)
        c.kv_len[0] = n - 2
        q = c.randn(256, "f32")
        out = torch.full((2 * n + 5, 256), 9.0, device=cuda)
        qq = torch.cat([q, torch.ones(5, 256, device=cuda)])
        b = paged4.Paged4Batch(c.cache, c.row0, c.kv_len, c.tab, rows=2 * n + 5, heads=4)
        b.attention(qq, out)
        assert check_errors() == 0
        assert (out[:2] == 0).all() and (out[2 * n:] == 9).all() and not (out[2:2 * n] == 0).all(1).any()
        # appended rows and read ones of nobody
        was = c.cache.v_pool.clone()
        c.kv_len[0] = n
        k = torch.randn(2 * n + 5, 128, device=cuda)
        back = torch.full((2 * n + 5, 128), 9.0, device=cuda)
        qo = torch.full((2 * n + 5, 256), 9.0, device=cuda)
        b.append(k, k, q=qq, q_out=qo)
        b.read(back, back.clone())
        assert check_errors() == 0
        assert (back[2 * n:] == 9).all() and (qo[2 * n:] == 9).all() and (qo[:2 * n] == qq[:2 * n]).all()
        pg, off = c.places()
        now = c.cache.v_pool.clone()
        now[pg, :, off] = was[pg, :, off]
        assert torch.equal(now, was)


def test_offsets_past_32_bits(cuda):
    """A pool whose codes pass 2^32 bytes, its far end in use."""
    import torch

    c = Case(cuda, [37], [200], 4, 256, 128, 16, pages=70000, seed=12)
    assert c.cache.k_pool.numel() > 1 << 32
    qkv = c.randn(24 * 256, "bf16")
    q, k, v = qkv[:, :4096], qkv[:, 4096:5120], qkv[:, 5120:]
    c.batch.append(k, v)
    pg, off = c.places()
    got = numbers(c.cache.v_pool[pg, :, off], c.cache.v_scale[pg, :, off]).flatten(1)
    assert torch.equal(c.batch.read(dtype=torch.float32)[1].double(), got)
    d = (c.cache.v_scale[pg, :, off].to(torch.int16) << 7).view(torch.float16).double().flatten(1).repeat_interleave(16, -1)
    assert ((got - v.double()).abs() <= d).all()          # half the widest step, between codes 4 and 6
    check_attention(c, q, "bf16")


def test_bad_pages_are_reported_and_nothing_is_read_outside(cuda):
    import torch

    c = Case(cuda, [4, 5], [30, 40], 2, 64, 16, 4, seed=13)
    was = [t.clone() for t in (c.cache.k_pool, c.cache.k_scale)]
    many = Case(cuda, [150, 160], [30, 40], 2, 64, 16, 4, seed=13)
    for bad in (-1, c.cache.pages, 1 << 30, -(1 << 31)):
        many.tab[1, 0] = bad if bad != c.cache.pages else many.cache.pages
        many.batch.attention(many.randn(256, "bf16"))
        assert check_errors() != 0 and check_errors() == 0
        c.tab[1, 0] = bad                                   # a page of the cached tokens, then of the new ones
        c.batch.attention(c.randn(256, "f32"))
        assert check_errors() != 0 and check_errors() == 0
        c.tab[1] = bad
        k = c.randn(128, "f32")
        c.batch.append(k, k)
        assert check_errors() != 0 and check_errors() == 0
        c.batch.read()
        assert check_errors() != 0 and check_errors() == 0
    pg, off = c.places()
    now = c.cache.k_pool.clone()
    now[pg, :, off] = was[0][pg, :, off]
    assert torch.equal(now, was[0])


def test_a_run_of_them_in_a_graph_on_another_stream(cuda):
    """Append, attend and read as one captured graph, replayed on new rows and lengths; and call by call on a given stream."""
    import torch

    c = Case(cuda, [1, 1, 5], [20, 47, 0], 2, 128, 16, 8, seed=14)
    freq, w = freqs(cuda, 64), torch.rand(128, device=cuda) + 0.5
    qkv = c.randn(12 * 128, "bf16")
    q, k, v = qkv[:, :1024], qkv[:, 1024:1280], qkv[:, 1280:]
    qo, out, rk, rv = torch.empty_like(q.contiguous()), torch.empty(7, 1024, dtype=q.dtype, device=cuda), *(torch.empty(7, 256, device=cuda) for _ in "kv")

    def step(**kw):
        c.batch.append(k, v, freq=freq, q=q, q_out=qo, q_norm=w, k_norm=w, **kw)
        c.batch.attention(qo, out, window=30, **kw)
        c.batch.read(rk, rv, **kw)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        qkv.copy_(torch.randn(qkv.shape, generator=c.g, device=cuda))
        for t in (qo, out, rk, rv):
            t.zero_()
        graph.replay()
        got = [t.clone() for t in (qo, out, rk, rv)]
        for t in (qo, out, rk, rv):
            t.zero_()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        step(stream=s)
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(a, b) for a, b in zip(got, (qo, out, rk, rv)))
        want, tol = want_attention(c, qo, 30)
        assert ((out.double() - want).abs() <= tol + HALF["bf16"] * want.abs()).all()
    made = c.batch.append(k, v, q=q, stream=s), c.batch.attention(qo, stream=s), *c.batch.read(stream=s), *c.batch.parts(stream=s)
    s.synchronize()
    assert [t.shape[0] for t in made] == [7] * 8
    assert check_errors() == 0


def test_attention_repeats_itself(cuda):
    import torch

    for rows, old in (([1] * 9 + [50], [3000] * 9 + [900]), ([1], [60000]), ([300], [9000]), ([70] * 3, [3000] * 3)):
        c = Case(cuda, rows, old, 2, 256, 64, 8, seed=15)
        q = c.randn(2048, "bf16")
        first = c.batch.attention(q)
        for _ in range(5):
            assert torch.equal(first, c.batch.attention(q))


def test_a_row_does_not_depend_on_the_other_rows(cuda):
    """Sequences of a batch, attended together and one by one."""
    import torch

    from spk import paged4

    c = Case(cuda, [1, 4, 2], [100, 900, 31], 2, 128, 32, 8, seed=16)
    q = c.randn(1024, "f32", 0.4)
    all_ = c.batch.attention(q)
    at = 0
    for s, n in enumerate(c.rows):
        one = torch.tensor([0, n], dtype=torch.int32, device=cuda)
        b = paged4.Paged4Batch(c.cache, one, c.kv_len[s:s + 1].clone(), c.tab[s:s + 1].clone(), rows=n, heads=8)
        got = b.attention(q[at:at + n])
        assert (got - all_[at:at + n]).norm() <= 1e-6 * got.norm()
        at += n


def test_what_the_binding_refuses(cuda):
    import torch

    import spk
    from spk import paged, paged4

    c = Case(cuda, [3], [5], 2, 64, 16, 4)
    k, v, q = c.randn(128, "f32"), c.randn(128, "f32"), c.randn(256, "f32")
    b = c.batch
    bad = [
        lambda: b.append(k[:2], v), lambda: b.append(k, v.half()), lambda: b.append(k.t().contiguous().t(), v), lambda: b.append(k.cpu(), v),
        lambda: b.append(k.double(), v.double()), lambda: b.append(k, v, q=q[:, :100]), lambda: b.append(k, v, q=q, q_out=q.half()),
        lambda: b.append(k, v, q_out=q), lambda: b.append(k, v, q_norm=torch.ones(64, device=cuda)),
        lambda: b.append(k, v, k_norm=torch.ones(63, device=cuda)), lambda: b.append(k, v, k_norm=torch.ones(64, device=cuda).half()),
        lambda: b.append(k, v, k_norm=torch.ones(128, device=cuda)[::2]), lambda: b.append(k, v, k_norm=torch.ones(65, device=cuda)[1:]),
        lambda: b.append(k, v, freq=torch.ones(4, device=cuda)), lambda: b.append(k, v, freq=torch.ones(40, device=cuda)),
        lambda: b.append(k, v, freq=torch.ones(16, device=cuda).half()), lambda: b.append(k, v, k_norm=torch.ones(64, device=cuda), eps=-1.0),
        lambda: b.append(k, v, k_norm=torch.ones(64, device=cuda), eps=float("nan")),
        lambda: b.attention(q[:, :64]), lambda: b.attention(q, window=-1), lambda: b.attention(q, gate=q), lambda: b.attention(q, out=q.half()),
        lambda: b.read(k[:, :64]), lambda: b.read(k, v.half()), lambda: b.parts([k, k, k, k]), lambda: b.read(dtype=torch.float64),
        lambda: b.use(paged.PagedCache(4, 16, 2, 64, device=cuda)), lambda: b.use(paged4.Paged4Cache(4, 32, 2, 64, device=cuda)),
        lambda: paged4.Paged4Batch(paged.PagedCache(4, 16, 2, 64, device=cuda), c.row0, c.kv_len, c.tab, rows=3, heads=4),
        lambda: paged.PagedBatch(c.cache, c.row0, c.kv_len, c.tab, rows=3, heads=4),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(spk.SpkError):
            f()
            pytest.fail(f"call {i} was taken")
    assert check_errors() == 0


def test_references_past_any_unit(cuda):
    """Scores so large that a unit of them is more than the weights' range: the largest key takes all, as in f32."""
    import torch

    for rows in ([2], [300]):
        for typ in ("f32", "bf16"):
            c = Case(cuda, rows, [100], 1, 64, 16, 2, seed=17)
            c.cache.k_pool.copy_(c.cache.k_pool & 0x77)     # positive keys, one of them the largest by far
            c.cache.k_scale[c.cache.k_scale != 255] = 100
            c.cache.k_scale[c.table[0][0], 0, 3] = 140
            c.cache.k_pool[c.table[0][0], 0, 3] = 0x77
            q = torch.full((rows[0], 128), 1e4, device=cuda).to(ttype(typ))
            got = c.batch.attention(q, scale=1e20)
            want = numbers(c.cache.v_pool[c.table[0][0], 0, 3], c.cache.v_scale[c.table[0][0], 0, 3])
            assert (got.double() - want.repeat(2)).abs().max() <= HALF[typ] * want.abs().max(), (rows, typ)


def test_long_prompts_of_several_sequences_are_taken(cuda):
    """Two prompts over a table of 131072 tokens each, 8 heads a KV head: within the line of work of the kernel that has them."""
    import torch

    from spk import paged4

    c = paged4.Paged4Cache(1024 + 2, 256, 4, 64, device=cuda)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    table = torch.zeros(2, 512, dtype=torch.int32, device=cuda)
    rows = 262144
    b = paged4.Paged4Batch(c, i32([0, 20, 40]), i32([20, 20]), table, rows=rows, heads=32)
    k = torch.randn(rows, 256, device=cuda, dtype=torch.bfloat16)
    b.append(k, k)
    q = torch.randn(rows, 2048, device=cuda, dtype=torch.bfloat16)
    b.attention(q, torch.empty_like(q))          # the arguments allow 262144 rows, the batch says 40
    assert check_errors() == 0


def test_calls_without_rows(cuda):
    import torch

    c = Case(cuda, [0, 0], [5, 0], 2, 64, 16, 4)
    z = torch.empty(0, 128, device=cuda)
    assert c.batch.append(z, z, q=torch.empty(0, 256, device=cuda)).shape == (0, 256)
    assert c.batch.attention(torch.empty(0, 256, device=cuda)).shape == (0, 256)
    assert c.batch.read()[0].shape == (0, 128) and c.batch.parts()[1].shape == (0, 8)
    assert check_errors() == 0


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("most", [70, 150, 300])
def test_one_sequence_of_fewer_rows_than_the_call_allows(cuda, most, hd, typ):
    """Arguments for `most` rows of 4 heads on a KV head, row0 that says 3: those rows, and none behind them."""
    import torch

    from spk import paged4

    for kv in (1, 3, 10):                 # few pairs of sequence and KV head, and more
        c = Case(cuda, [3], [50], kv, hd, 16, 4 * kv, seed=22)
        q = c.randn(4 * kv * hd, typ, 0.4)
        qq = torch.cat([q, torch.ones(most - 3, q.shape[1], dtype=q.dtype, device=cuda)])
        out = torch.full_like(qq, 9.0)
        paged4.Paged4Batch(c.cache, c.row0, c.kv_len, c.tab, rows=most, heads=4 * kv).attention(qq, out)
        assert check_errors() == 0
        want, tol = want_attention(c, q)
        assert ((out[:3].double() - want).abs() <= tol + HALF[typ] * want.abs() + TINY[typ]).all()
        assert (out[3:] == 9).all()


def test_a_captured_chunk_replayed_with_a_shorter_one(cuda):
    """A prompt's chunks by one graph of 150 rows: the last one has fewer, which the device's arrays say."""
    import torch

    for hd, typ in ((256, "bf16"), (64, "f32")):
        c = Case(cuda, [150], [300], 2, hd, 32, 8, seed=23)
        q, k, v = c.randn(8 * hd, typ, 0.4), c.randn(2 * hd, typ), c.randn(2 * hd, typ)
        qo, out = torch.zeros_like(q), torch.zeros_like(q)

        def step():
            c.batch.append(k, v, q=q, q_out=qo)
            c.batch.attention(qo, out)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for n in (150, 40, 7, 1, 0, 65):
            c.rows, c.len = [n], [300 + n]
            c.row0.copy_(torch.tensor([0, n]))
            c.kv_len.copy_(torch.tensor([300 + n]))
            out.fill_(9.0)
            graph.replay()
            assert check_errors() == 0
            assert (out[n:] == 9).all()
            if n:
                want, tol = want_attention(c, qo[:n])
                assert ((out[:n].double() - want).abs() <= tol + HALF[typ] * want.abs() + TINY[typ]).all(), n


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [[3, 2], [150, 70]])
def test_keys_under_scales_that_are_no_numbers(cuda, rows, hd, typ):
    """Scale bytes from 248 (f16's infinity) to 255 of keys all of whose products with the queries are negative: NaN where they are seen."""
    import torch

    c = Case(cuda, rows, [60, 37], 2, hd, 16, 8, seed=24)
    c.cache.k_pool.bitwise_and_(0x77).bitwise_or_(0x11)           # no zeros, none negative
    groups = hd // 16
    for i, byte in enumerate((248, 249, 255)):
        p = 61 - 19 * i
        c.cache.k_scale[c.table[0][p // 16], 0, p % 16, (5 * i + 1) % groups] = byte
    c.cache.k_scale[c.table[1][2], 1, 4, groups - 1] = 248        # token 36 of the second sequence
    q = c.randn(8 * hd, typ, 0.2).abs().clamp(min=0.01).neg()
    for window in (0, 9):
        got = check_attention(c, q, typ, window)
        assert got.isnan().any() and not got.isnan().all()


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_poison_in_one_tile_after_another(cuda, typ):
    """Poisoned values in tile after tile of a sequence of many rows, clean tiles behind them: a window's rows are NaN while
    they see one, and numbers again after it."""
    c = Case(cuda, [400, 90], [500, 0], 2, 128, 32, 8, seed=25)
    for p in (*range(470, 640, 17), 700, 760):
        c.cache.v_scale[c.table[0][p // 32], p % 2, p % 32, p % 8] = 255 if p % 3 else 248
    for window in (30, 150):
        got = check_attention(c, c.randn(1024, typ, 0.4), typ, window)
        assert got.isnan().any() and not got.isnan().all()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_norms_of_rows_of_any_size(cuda, hd, typ):
    """Heads whose squares, or their sum, are out of f32's range: the norm is that of the formula."""
    import torch

    size = {"f32": [1e38, 1.0, 1e30, 1e19, 1e-19, 1e-25, 1e-38, 3e-41], "bf16": [1e38, 1.0, 1e30, 1e19, 1e-19, 1e-25, 1e-36, 1e-30],
            "f16": [1e4, 1.0, 100.0, 1e-3]}[typ]
    c = Case(cuda, [len(size) * 3, 5], [4, 0], 2, hd, 16, 4, seed=26)
    q, k, v = c.randn(4 * hd, typ), c.randn(2 * hd, typ), c.randn(2 * hd, typ)
    q.clamp_(-3, 3)
    k.clamp_(-3, 3)
    for i in range(q.shape[0]):
        q[i] *= size[i % len(size)]
        k[i] *= size[(i + 1) % len(size)]
    q[2, :hd] *= size[0]                             # heads of one row apart, too
    q[2].clamp_(-torch.finfo(q.dtype).max, torch.finfo(q.dtype).max)
    w = [torch.rand(hd, generator=c.g, device=cuda) + 0.5 for _ in "qk"]
    for eps in np.float32([1e-6, 0.0, 1e-35, 1e-45, 1e30]).tolist():          # eps is an f32 argument: 1e-45 is 1.4e-45
        for freq in (freqs(cuda, 32), None):
            # Rows that are nothing beside eps leave under 2^-126, where a rounding is off by up to 2^-150 whatever the value: x r; times w <= 1.5, 2.5 of
            # them; two products and a sum of the rotation, 2.5 (|cos| + |sin|) + 2 <= 6 of them (not rotated, halved and added: 4.5), beside check_append's bound.
            check_append(c, k, v, None, freq, False, None, w[1], eps=eps, typ=typ)
            got = c.batch.append(k, v, freq=freq, q=q, q_norm=w[0], k_norm=w[1], eps=eps)
            y, size = (t.flatten(1) for t in head_rows(q, 4, hd, w[0], eps, c.positions(), freq, False))
            assert ((got.double() - y).abs() <= HALF[typ] * y.abs() + TINY[typ] + 2.0 ** -20 * size + 6 * 2.0 ** -150).all()


def test_norms_of_rows_with_an_infinity(cuda):
    """x / sqrt(mean x^2 + eps): 0 beside an infinity, NaN in its place; a NaN makes its head NaN."""
    import torch

    c = Case(cuda, [3], [0], 1, 64, 16, 2)
    q, w = torch.ones(3, 128, device=cuda), torch.ones(64, device=cuda)
    q[0, 5], q[1, 70] = float("inf"), float("nan")
    got = c.batch.append(q[:, :64].contiguous(), q[:, :64].contiguous(), q=q, q_norm=w)
    assert got[0, 5].isnan() and (got[0, :5] == 0).all() and (got[0, 6:64] == 0).all() and got[1, 64:].isnan().all()
    assert not got[0, 64:].isnan().any() and not got[1, :64].isnan().any() and not got[2].isnan().any()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("hd,pdim", [(64, 16), (128, 32), (256, 64), (256, 240)])
def test_dims_that_are_not_rotated_leave_as_they_came(cuda, hd, pdim, inter, typ):
    """Infinities and zeros of either sign beside each other behind the rotated dims: the queries' bits."""
    import torch

    c = Case(cuda, [7, 30], [900, 2], 2, hd, 16, 4, seed=27)
    q, k, v = c.randn(4 * hd, typ), c.randn(2 * hd, typ), c.randn(2 * hd, typ)
    x = q.view(-1, 4, hd)
    for d, to in ((pdim, float("inf")), (pdim + 3, -0.0), (pdim + 6, float("-inf")), (hd - 1, 0.0), (hd - 4, float("inf"))):
        x[:, :, d] = to
    x[3:9, 1, pdim:] = -0.0
    got = c.batch.append(k, v, freq=freqs(cuda, pdim), q=q, interleaved=inter)
    bits = torch.int32 if typ == "f32" else torch.int16
    assert torch.equal(got.view(-1, 4, hd)[:, :, pdim:].contiguous().view(bits), x[:, :, pdim:].contiguous().view(bits))
    y, size = head_rows(q, 4, hd, None, 0.0, c.positions(), freqs(cuda, pdim), inter)
    off = (got.view(-1, 4, hd).double() - y)[:, :, :pdim].abs()
    assert (off <= HALF[typ] * y[:, :, :pdim].abs() + TINY[typ] + 2.0 ** -20 * size[:, :, :pdim]).all()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,old,kv,hd,heads,window", [([1, 3], [700, 90], 2, 256, 8, 0), ([1, 8, 2], [1000, 5, 300], 2, 128, 16, 40),
                                                         ([2], [300], 1, 64, 4, 0), ([150, 80], [90, 300], 2, 256, 8, 0), ([300], [100], 1, 64, 2, 60),
                                                         ([90, 70], [0, 33], 3, 128, 6, 0)])
def test_attention_over_every_scale_that_append_writes(cuda, rows, old, kv, hd, heads, window, typ):
    """Scale bytes 8 to 226, 2^-14 to 10240, at random in every row; all of the smallest, all of the largest."""
    c = Case(cuda, rows, old, kv, hd, 16, heads, seed=28, scales=(8, 227))
    check_attention(c, c.randn(heads * hd, typ, 2e-5), typ, window)
    check_attention(c, c.randn(heads * hd, typ, 1.0), typ, window, scale=2.0 ** -18)
    for scales in ((8, 9), (226, 227)):
        c = Case(cuda, rows, old, kv, hd, 16, heads, seed=29, scales=scales)
        check_attention(c, c.randn(heads * hd, typ, 1.0), typ, window, scale=16.0 if scales[0] == 8 else 2.0 ** -18)


@pytest.mark.parametrize("size", [0.05, 30.0])
@pytest.mark.parametrize("rows, nseq", [(1, 320), (128, 160)])
def test_bf16_values_of_one_sign_in_a_long_context(cuda, rows, nseq, size):
    """test_values_of_one_sign_in_a_long_context in bf16, whose few rows keep one accumulator: 65536 tokens are at most 1024 blocks of 16 of
    a warp, an instruction each, short by up to a unit, 2^-23 of the sum; many rows: 16384 tokens, 1024 instructions."""
    import torch

    from spk import paged4

    n, page, hd = 65536, 128, 64
    c = paged4.Paged4Cache(n // page, page, 1, hd, device=cuda)
    g = torch.Generator(device=cuda)
    g.manual_seed(31)
    for pool, scale, keep in ((c.k_pool, c.k_scale, 0xff), (c.v_pool, c.v_scale, 0x77)):
        pool.random_(0, 256, generator=g)
        pool.bitwise_and_(keep)
        scale.copy_(torch.randint(95, 103, scale.shape, generator=g, device=cuda).to(torch.uint8))
    if size > 1:
        c.k_scale -= torch.linspace(30, 0, n // page, device=cuda).to(torch.uint8)[:, None, None, None]
    row0 = torch.arange(nseq + 1, dtype=torch.int32, device=cuda) * rows
    table = torch.arange(n // page, dtype=torch.int32, device=cuda)[None].expand(nseq, -1).contiguous()
    b = paged4.Paged4Batch(c, row0, torch.full((nseq,), n, dtype=torch.int32, device=cuda), table, rows=nseq * rows, heads=1)
    q = (torch.randn(nseq * rows, hd, generator=g, device=cuda) * size).bfloat16()
    got = b.attention(q).double()
    assert check_errors() == 0
    k, v = (numbers(p, s)[:, 0].reshape(-1, hd) for p, s in ((c.k_pool, c.k_scale), (c.v_pool, c.v_scale)))
    for s in (0, 1, nseq // 2, nseq - 1):
        x = q[s * rows].double() * hd ** -0.5
        kk, vv = k[:n - rows + 1], v[:n - rows + 1]
        p = torch.softmax(kk @ x, 0)
        want = p @ vv
        bound = 1024 * 2.0 ** -23 + 2.0 ** -11 + 2.0 ** -20 * (kk.abs() @ x.abs()).max() + 2.0 ** -20 + HALF["bf16"]
        off = (got[s * rows] - want).abs()
        assert (off <= bound * want + 2.0 ** -31 * p.max() * vv.sum(0)).all(), (s, (off / want).max(), bound)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows,group", [([1] * 12 + [30], 4), ([1] * 12 + [33, 32], 4), ([2] * 9 + [16] * 5, 8), ([11] * 9, 4), ([15] * 9, 4), ([8] * 6 + [9] * 6 + [1], 4), ([7, 9] * 5 + [0, 40], 8)])
def test_sequences_on_both_sides_of_the_border(cuda, rows, group, hd, typ):
    """Few large sequences among small ones, all alike, mixed: rows per KV head on average and at most, about where the kernels change."""
    c = Case(cuda, rows, [(37 * i) % 200 for i in range(len(rows))], 1, hd, 16, group, seed=32)
    check_attention(c, c.randn(group * hd, typ, 0.4), typ)


@pytest.mark.parametrize("typ,hd,rows,calls", [("bf16", 64, [1, 1, 2], 60), ("f32", 128, [1], 60), ("f16", 256, [1, 3], 40), ("bf16", 64, [40, 33], 12), ("f32", 256, [70], 8)])
def test_step_after_step_without_a_pause(cuda, typ, hd, rows, calls):
    """Append and attend, call after call, launched one behind the other and as one graph: each call reads the lines that the one
    before it read, too, with the rows behind them written since."""
    import torch

    from spk import paged4

    n = len(rows)
    c = Case(cuda, [calls * r for r in rows], [5] * n, 2, hd, 16, 8, seed=33)
    q, k, v = c.randn(8 * hd, typ, 0.4), c.randn(2 * hd, typ), c.randn(2 * hd, typ)
    first = np.concatenate([[0], np.cumsum(c.rows)])[:-1]
    own = [sum(([first[s] + i * r + x for x in range(r)] for s, r in enumerate(rows)), []) for i in range(calls)]   # the call's rows among all
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device=cuda)  # noqa: E731
    row0 = i32(np.concatenate([[0], np.cumsum(rows)]).tolist())
    lens = [i32([5 + (i + 1) * r for r in rows]) for i in range(calls)]
    batches = [paged4.Paged4Batch(c.cache, row0, L, c.tab, rows=sum(rows), heads=8) for L in lens]
    qs, ks, vs = ([t[torch.tensor(o, device=cuda)].contiguous() for o in own] for t in (q, k, v))
    outs = [torch.zeros_like(t) for t in qs]

    def run():
        for b, x, y, z, o in zip(batches, qs, ks, vs, outs):
            b.append(y, z)
            b.attention(x, o)

    def poison():
        for s, L in enumerate(c.len):
            for p in range(5, L):
                for t in (c.cache.k_scale, c.cache.v_scale):
                    t[c.table[s][p // 16], :, p % 16] = 255

    for form in ("calls", "graph", "graph"):
        poison()
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        if form == "calls":
            run()
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            got = torch.cat(outs)
            with torch.cuda.graph(graph):
                run()
        else:
            graph.replay()
            got = torch.cat(outs)
        assert check_errors() == 0
        want, tol = want_attention(c, q)
        at = torch.tensor(sum(own, []), device=cuda)
        assert ((got.double() - want[at]).abs() <= tol[at] + HALF[typ] * want[at].abs() + TINY[typ]).all(), form


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [[3, 2], [150, 70]])
def test_scales_above_all_that_append_writes(cuda, rows, hd, typ):
    """Bytes 227 to 247, scales over 10240 under which a value may pass f16's end: NaN where they are seen, and nowhere else."""
    import torch

    c = Case(cuda, rows, [60, 37], 2, hd, 16, 8, seed=35)
    c.cache.k_pool.bitwise_or_(0x77)                # 6 or -6: past f16's end under each of these scales
    c.cache.v_pool.bitwise_or_(0x77)
    q = c.randn(8 * hd, typ, 0.2)
    clean = [t.clone() for t in (c.cache.k_scale, c.cache.v_scale)]
    for i, byte in enumerate((227, 240, 247)):
        p = 61 - 19 * i
        (c.cache.k_scale if i == 1 else c.cache.v_scale)[c.table[0][p // 16], 0, p % 16, (5 * i + 1) % (hd // 16)] = byte
    now = [t.clone() for t in (c.cache.k_scale, c.cache.v_scale)]
    for window in (0, 9):
        got = c.batch.attention(q, window=window)
        assert check_errors() == 0
        for t, was, to in zip((c.cache.k_scale, c.cache.v_scale), clean, now):
            t.copy_(torch.where(to != was, torch.full_like(to, 255), to))
        want = check_attention(c, q, typ, window)
        assert got.isnan().any() and not got.isnan().all()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~got.isnan()], want[~want.isnan()])
        for t, to in zip((c.cache.k_scale, c.cache.v_scale), now):
            t.copy_(to)


@pytest.mark.parametrize("rows", [[3, 2], [70, 9]])
@pytest.mark.parametrize("bits", [8, 4])
def test_lengths_that_are_none(cuda, rows, bits):
    """kv_len under 0, down to the smallest there is: its rows see nothing, the others are as they were. A window as large as there is one."""
    import torch

    from spk import paged, paged4

    c = Case(cuda, rows, [60, 37], 2, 64, 16, 8, seed=34)
    q = c.randn(512, "f32")
    if bits == 8:
        cache = paged.PagedCache(c.cache.pages, 16, 2, 64, device=cuda)
        for t in (cache.k_pool, cache.v_pool, cache.k_scale, cache.v_scale):
            t.fill_(1.0)
        batch = paged.PagedBatch(cache, c.row0, c.kv_len, c.tab, rows=sum(rows), heads=8)
    else:
        batch = c.batch
    first = batch.attention(q)
    assert torch.equal(batch.attention(q, window=(1 << 31) - 1), first)
    for bad in (-1, -5, -(1 << 31), -(1 << 31) + 1, 0):
        c.kv_len[0] = bad
        for window in (0, 9, (1 << 31) - 1):
            out = torch.full_like(q, 9.0)
            batch.attention(q, out, window=window)
            assert check_errors() == 0
            assert (out[:rows[0]] == 0).all()
            if window != 9:
                assert (out[rows[0]:] - first[rows[0]:]).norm() <= 1e-6 * first[rows[0]:].norm()
    c.kv_len[0] = rows[0] - 1                 # the first row alone lies before the sequence
    big, none = batch.attention(q, window=(1 << 31) - 1), batch.attention(q)
    assert torch.equal(big, none) and (big[0] == 0).all() and not (big[1:] == 0).all(1).any()
