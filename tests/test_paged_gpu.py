"""spk_paged_append and spk_paged_attn against a 64-bit restatement of their definitions.

Bounds. A stored value is the e4m3 rounding of x / d: off by at most 2^-4 of it, or 2^-10 below
2^-6, with 1e-5 of that for x and d in f32; a rotated key is off by its pair's f32 rounding besides, which the
difference of two products does not share out: cosine and sine to 2 ulp, two products and a sum, 2^-21 of the
pair's length. A scale is off by f32 rounding of a rotation and a
division: 1e-6. Attention reads the cache exactly, so its error is its type's rounding of the output
(2^-9, 2^-12 of a value for bf16, f16) and of the query and weights it splits into e4m3 terms (2^-9 for
two, 2^-13 for three, 2^-21 for five), as a relative norm: 2^-7, 2^-10, 1e-5 for bf16, f16, f32."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
TOL = {"f32": 1e-5, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}
ORDER = [2 * (b // 4) + b % 2 + 8 * (b // 2 % 2) for b in range(16)]


def ttype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def pack_k(x):   # logical [pages][kv][tokens][hd] -> as the pool lies
    p, h, t, d = x.shape
    return x.reshape(p, h, t // 8, 8, d // 16, 16).transpose(3, 4).contiguous()


def pack_v(x):
    p, h, t, d = x.shape
    return x.reshape(p, h, t // 16, 16, d)[:, :, :, ORDER].transpose(3, 4).contiguous()


def unpack_k(pool):
    p, h, g, c, _, _ = pool.shape
    return pool.double().transpose(3, 4).reshape(p, h, g * 8, c * 16)


def unpack_v(pool):
    import torch

    p, h, b, d, _ = pool.shape
    out = torch.empty(p, h, b, 16, d, dtype=torch.float64, device=pool.device)
    for i, t in enumerate(ORDER):
        out[:, :, :, t] = pool[..., i].double()
    return out.reshape(p, h, b * 16, d)


def rope(x, pos, freq):
    """x [n][heads][hd] f64; the angle is the f32 product of position and frequency."""
    import torch

    if freq is None:
        return x
    h = freq.numel()
    ang = (torch.as_tensor(pos, dtype=torch.float32, device=x.device)[:, None] * freq[None]).double()
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)


class Case:
    """A pool with random contents, a page table in random order, and a batch over it."""

    def __init__(self, dev, rows, old, kv=2, hd=128, page=32, heads=None, seed=0, spread=1.0, fill="random"):
        import torch

        from spk import paged

        self.dev, self.rows, self.len, self.kv, self.hd, self.page = dev, rows, [a + b for a, b in zip(rows, old)], kv, hd, page
        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        self.g = g
        need = [-(-n // page) for n in self.len]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=g, device=dev).int().cpu().tolist()
        width = max(1, max(need))
        self.table = [[order.pop() for _ in range(n)] + [-1] * (width - n) for n in need]
        self.cache = paged.PagedCache(pages, page, kv, hd, device=dev)
        f8 = torch.float8_e4m3fn
        rnd = lambda: torch.randn(pages, kv, page, hd, generator=g, device=dev).mul_(80).clamp_(-440, 440).to(torch.float16)  # noqa: E731
        self.cache.k_pool.copy_(pack_k(rnd()).to(f8))
        self.cache.v_pool.copy_(pack_v(rnd()).to(f8))
        for s in (self.cache.k_scale, self.cache.v_scale):
            s.copy_(torch.rand(s.shape, generator=g, device=dev).mul_(spread).exp_().mul_(0.01))
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        self.row0 = i32(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32).tolist())
        self.kv_len, self.tab = i32(self.len), i32(self.table)
        self.heads = heads or kv
        self.batch = paged.PagedBatch(self.cache, self.row0, self.kv_len, self.tab, rows=sum(rows), heads=self.heads)

    def randn(self, width, typ, scale=1.0):
        import torch

        return torch.randn(sum(self.rows), width, generator=self.g, device=self.dev).mul_(scale).to(ttype(typ))


def freqs(dev, pdim, theta=1e4):
    from spk import paged

    return paged.rope_freq(theta, pdim, dev) if pdim else None


def check_errors():
    import spk

    return spk.lib().spk_check_device_error()


# ------------------------------------------------------------------------------------------ append

def want_append(c, x, name, freq):
    """(values / scale, scales, f32's share of the error) by the definition, in 64 bits, before the rounding to e4m3."""
    import torch

    pool = unpack_k(c.cache.k_pool) if name == "k" else unpack_v(c.cache.v_pool)
    sc = (c.cache.k_scale if name == "k" else c.cache.v_scale).double().clone()
    x = x.double().reshape(-1, c.kv, c.hd)
    slack = torch.zeros_like(pool)
    at = 0
    for s, (n, L) in enumerate(zip(c.rows, c.len)):
        new = x[at:at + n]
        at += n
        pair = torch.zeros_like(new)
        if n and name == "k" and freq is not None:
            h = freq.numel()
            pair[..., :h] = pair[..., h:2 * h] = torch.hypot(new[..., :h], new[..., h:2 * h])
            new = rope(new, list(range(L - n, L)), freq)
        first = L - n
        for b in range(first // 16 * 16, L, 16) if n else []:
            pg, o = c.table[s][b // c.page], b % c.page
            lo, hi = max(b, first), min(b + 16, L)
            vals = new[lo - first:hi - first].transpose(0, 1)
            d = (vals.abs().amax((1, 2)) / 448).clamp(min=2.0 ** -100)
            if lo > b:
                was = sc[pg, :, o // 16].clone()
                d = d.maximum(was)
                pool[pg, :, o:o + lo - b] *= (was / d)[:, None, None]
            sc[pg, :, o // 16] = d
            pool[pg, :, o + lo - b:o + hi - b] = vals / d[:, None, None]
            slack[pg, :, o + lo - b:o + hi - b] = 2.0 ** -21 * pair[lo - first:hi - first].transpose(0, 1) / d[:, None, None]
            pool[pg, :, o + hi - b:o + 16] = 0
    return pool, sc, slack


def check_append(c, k, v, freq):
    want = [want_append(c, k, "k", freq), want_append(c, v, "v", None)]
    c.batch.append(k, v, freq=freq)
    assert check_errors() == 0
    for (pool, sc, slack), got, gs in zip(want, (unpack_k(c.cache.k_pool), unpack_v(c.cache.v_pool)), (c.cache.k_scale, c.cache.v_scale)):
        assert ((gs.double() - sc).abs() <= 1e-6 * sc).all()
        off = (got - pool).abs()
        assert (off <= (pool.abs() * 2.0 ** -4).clamp(min=2.0 ** -10) * (1 + 1e-5) + slack).all(), off.max()
    return want


SHAPES = [([1], [0]), ([1], [4103]), ([16], [0]), ([17], [15]), ([33, 0, 1, 5], [0, 0, 31, 250]), ([3, 64, 130], [7, 16, 1])]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,kv,page", [(256, 4, 64), (128, 3, 48), (64, 5, 16)])
@pytest.mark.parametrize("rows,old", SHAPES)
def test_append_matches_the_definition(cuda, rows, old, hd, kv, page, typ):
    c = Case(cuda, rows, old, kv=kv, hd=hd, page=page, seed=len(rows) + hd)
    check_append(c, c.randn(kv * hd, typ), c.randn(kv * hd, typ), freqs(cuda, hd // 4))


@pytest.mark.parametrize("pdim", [0, 8, 64, 128])
@pytest.mark.parametrize("pos", [0, 1000, 131000, 1000000])
def test_append_rotates_at_any_position(cuda, pdim, pos):
    c = Case(cuda, [40], [pos], hd=128, page=1024, seed=pdim)
    check_append(c, c.randn(256, "f32"), c.randn(256, "f32"), freqs(cuda, pdim))


@pytest.mark.parametrize("shift,pad", [(0, 4), (1, 0), (2, 2), (3, 1)])
@pytest.mark.parametrize("typ", ["f32", "f16"])
def test_append_takes_strided_and_unaligned_rows(cuda, shift, pad, typ):
    import torch

    c = Case(cuda, [9, 30], [3, 0], kv=2, hd=128, seed=shift)
    wide = torch.randn(39, 512 + pad + shift, generator=c.g, device=cuda).to(ttype(typ))
    check_append(c, wide[:, shift:shift + 256], wide[:, shift + 256:shift + 512], freqs(cuda, 32))


def test_append_token_by_token_keeps_every_row(cuda):
    """Scales grow inside a block: each step follows the definition, and after all of them every value is
    within the roundings it went through."""
    import torch

    from spk import paged

    kv, hd, n = 2, 64, 40
    g = torch.Generator(device=cuda)
    g.manual_seed(5)
    x = torch.randn(n, kv * hd, generator=g, device=cuda) * torch.linspace(0.1, 8, n, device=cuda)[:, None]
    cache = paged.PagedCache(3, 16, kv, hd, device=cuda)
    row0 = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
    length = torch.zeros(1, dtype=torch.int32, device=cuda)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=cuda)
    b = paged.PagedBatch(cache, row0, length, table, rows=1, heads=kv)
    for i in range(n):
        length.fill_(i + 1)     # the batch follows what its arrays hold
        b.append(x[i:i + 1], x[i:i + 1])
    k, v = cache.values()
    for got in (k, v):
        seq = got[[2, 0, 1]].transpose(0, 1).reshape(kv, 48, hd)[:, :n].transpose(0, 1).reshape(n, -1).double()
        # a row is rounded once and again whenever a later row of its block raised the scale: at most 16 times
        top = x.abs().reshape(n, kv, hd).amax(-1)
        for i in range(n):
            blk = top[i // 16 * 16:(i // 16 + 1) * 16].amax(0)
            lim = 16 * (x[i].abs().double() * 2.0 ** -4).clamp(min=float(blk.max()) / 448 * 2.0 ** -10)
            assert ((seq[i] - x[i].double()).abs() <= lim * 1.01).all()


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_append_every_step_of_a_block_follows_the_definition(cuda, typ):
    """40 single tokens of growing size: after each one the block's new and earlier rows are one rounding of what the
    definition makes of the bytes before it."""
    import torch

    c = Case(cuda, [1], [39], kv=2, hd=64, page=16, seed=21)
    for i in range(40):
        c.len = [i + 1]
        c.kv_len.fill_(i + 1)
        size = 0.1 * 1.15 ** i if i % 5 else 0.01
        check_append(c, c.randn(128, typ, scale=size), c.randn(128, typ, scale=size), freqs(cuda, 32))
    assert (c.cache.k_scale[c.table[0][:3]] > 0).all() and torch.isfinite(c.cache.values()[0][c.table[0][:3]]).all()


def test_append_many_sequences_and_long_runs(cuda):
    """More blocks than a CTA takes at once, several head groups, 700 sequences of one row."""
    c = Case(cuda, [6000], [5], kv=6, hd=128, page=64, seed=2)
    check_append(c, c.randn(768, "bf16"), c.randn(768, "bf16"), freqs(cuda, 128))
    c = Case(cuda, [1] * 700, [i % 50 for i in range(700)], kv=2, hd=64, page=16, seed=3)
    check_append(c, c.randn(128, "f16"), c.randn(128, "f16"), freqs(cuda, 16))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_append_poisons_the_block_of_a_value_that_is_no_number(cuda, bad):
    import torch

    c = Case(cuda, [40], [0], kv=2, hd=64, page=16, seed=1)
    k, v = c.randn(128, "f32"), c.randn(128, "f32")
    k[20, 70] = bad     # block 1 of head 1
    v[33, 3] = bad      # block 2 of head 0
    c.batch.append(k, v)
    assert check_errors() == 0
    pg = c.table[0]
    ks = torch.stack([c.cache.k_scale[p, :, 0] for p in pg]).isfinite()
    vs = torch.stack([c.cache.v_scale[p, :, 0] for p in pg]).isfinite()
    assert ks.tolist() == [[True, True], [True, False], [True, True]]
    assert vs.tolist() == [[True, True], [True, True], [False, True]]
    for pool in (c.cache.k_pool, c.cache.v_pool):
        assert pool[pg].float().isfinite().all()     # never a stored byte


def test_append_leaves_other_pages_alone_and_reports_bad_batches(cuda):
    import torch

    import spk

    c = Case(cuda, [20, 20], [0, 0], kv=2, hd=64, page=16, seed=4)
    before = c.cache.k_pool.clone().view(torch.uint8)
    c.batch.append(c.randn(128, "f32"), c.randn(128, "f32"))
    now = c.cache.k_pool.view(torch.uint8)
    held = [p for row in c.table for p in row if p >= 0]
    other = [p for p in range(c.cache.pages) if p not in held]
    assert torch.equal(before[other], now[other])
    for spoil in ("page", "rows", "length"):
        c = Case(cuda, [20, 20], [0, 0], kv=2, hd=64, page=16, seed=4)
        if spoil == "page":
            c.tab[1, 1] = c.cache.pages
        elif spoil == "rows":
            c.row0[2] = 41
        else:
            c.kv_len[0] = 4000
        c.batch.append(c.randn(128, "f32"), c.randn(128, "f32"))
        assert check_errors() == -1 and "index" in spk.last_error(), spoil
        assert check_errors() == 0


# --------------------------------------------------------------------------------------- attention

def want_attention(c, q, freq=None, window=0, gate=None, scale=None):
    import torch

    k = unpack_k(c.cache.k_pool) * c.cache.k_scale.double().repeat_interleave(16, -1)[..., None]
    v = unpack_v(c.cache.v_pool) * c.cache.v_scale.double().repeat_interleave(16, -1)[..., None]
    group = c.heads // c.kv
    out = torch.zeros(sum(c.rows), c.heads, c.hd, dtype=torch.float64, device=c.dev)
    at = 0
    for s, (n, L) in enumerate(zip(c.rows, c.len)):
        if n == 0:
            continue
        pg = [p for p in c.table[s] if p >= 0]
        ks, vs = (x[pg].transpose(0, 1).reshape(c.kv, -1, c.hd)[:, :L] for x in (k, v))
        qs = rope(q[at:at + n].double().reshape(n, c.heads, c.hd), list(range(L - n, L)), freq)
        i, j = torch.arange(L - n, L, device=c.dev)[:, None], torch.arange(L, device=c.dev)
        hide = j > i
        if window:
            hide = hide | (j <= i - window)
        for h in range(c.heads):
            w = qs[:, h] @ ks[h // group].T * (scale or c.hd ** -0.5)
            out[at:at + n, h] = torch.softmax(w.masked_fill(hide, float("-inf")), -1) @ vs[h // group]
        at += n
    if gate is not None:
        out *= torch.sigmoid(gate.double())[..., None]
    return out.reshape(sum(c.rows), -1)


def check_attention(c, typ, q=None, tol=None, **kw):
    q = c.randn(c.heads * c.hd, typ) if q is None else q
    want = want_attention(c, q, **kw)
    for _ in range(2):      # the workspace is left ready
        got = c.batch.attention(q, **kw).double()
        assert check_errors() == 0
        err = ((got - want).norm() / want.norm()).item()
        assert err < (tol or TOL[typ]), err
    return got


LENGTHS = [([1], [0]), ([1], [14]), ([1], [15]), ([1], [16]), ([1], [126]), ([1], [127]), ([1], [128]), ([1], [5000]),
           ([5], [0]), ([8], [500]), ([2, 0, 1, 7], [3, 0, 300, 120]), ([150], [0]), ([70], [333])]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,kv,group,page", [(256, 4, 4, 64), (128, 2, 8, 32), (64, 3, 1, 16), (128, 1, 5, 48)])
@pytest.mark.parametrize("rows,old", LENGTHS)
def test_attention_matches_the_definition(cuda, rows, old, hd, kv, group, page, typ):
    c = Case(cuda, rows, old, kv=kv, hd=hd, page=page, heads=kv * group, seed=hd + group + len(rows))
    gate = c.randn(c.heads, typ)
    check_attention(c, typ, freq=freqs(cuda, hd // 4), gate=gate)


@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 128, 129, 400, 100000])
@pytest.mark.parametrize("typ,rows", [("f32", [1, 3]), ("bf16", [90, 2]), ("f16", [8, 40])])
def test_attention_window(cuda, window, typ, rows):
    c = Case(cuda, rows, [600, 130], kv=2, hd=128, heads=8, page=32, seed=window)
    check_attention(c, typ, window=window, freq=freqs(cuda, 128))


# On average 9, 21, 30, 170 and 290 rows of a sequence per KV head: a tile of every width, whole and cut.
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,group,page", [(64, 2, 16), (128, 4, 32), (256, 1, 128)])
@pytest.mark.parametrize("mean", [9, 21, 30, 170, 290])
@pytest.mark.parametrize("window", [0, 131])
def test_attention_tiles_of_every_width(cuda, window, mean, hd, group, page, typ):
    n = max(1, mean // group)
    c = Case(cuda, [2 * n - 1, 1], [260, 1000], kv=2, hd=hd, heads=2 * group, page=page, seed=mean + hd)
    check_attention(c, typ, window=window, freq=freqs(cuda, hd // 2), gate=c.randn(c.heads, typ))


@pytest.mark.parametrize("rows", [[1], [12], [60], [300]])
def test_attention_poison_under_every_width(cuda, rows):
    """A poisoned block is NaN for the rows that see it and nothing to the rows before it."""
    import torch

    c = Case(cuda, rows, [40], kv=1, hd=64, heads=2, page=16, seed=2)
    q = c.randn(c.heads * 64, "bf16")
    clean = c.batch.attention(q).clone()
    last = (c.len[0] - 1) // 16                       # the block of the last token
    c.cache.v_scale[c.table[0][last], 0, 0] = float("nan")
    got = c.batch.attention(q)
    assert check_errors() == 0
    sees = torch.arange(c.len[0] - rows[0], c.len[0], device=cuda) >= 16 * last
    assert torch.isnan(got[sees]).all() and torch.equal(got[~sees], clean[~sees])


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_attention_with_scales_far_apart(cuda, typ):
    """Block scales over 13 orders of magnitude, some of the smallest allowed: no weight is lost under
    another block's scale."""
    import torch

    c = Case(cuda, [1, 6], [900, 300], kv=2, hd=128, heads=8, page=32, seed=9)
    for s in (c.cache.v_scale,):
        s.copy_(torch.pow(10.0, torch.randint(-9, 4, s.shape, generator=c.g, device=cuda).float()))
    check_attention(c, typ)
    if typ != "f16":     # which has no value that small
        c.cache.v_scale.fill_(2.0 ** -100)
        check_attention(c, typ)


@pytest.mark.parametrize("size", [1e-18, 1e-3, 300.0])
@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_attention_takes_queries_of_any_size(cuda, typ, size):
    """Tiny ones weigh every token alike; large ones pick one token."""
    c = Case(cuda, [1, 9], [200, 60], kv=2, hd=128, heads=8, page=32, seed=8)
    q = c.randn(c.heads * c.hd, typ, scale=size)
    # scores up to ~3000 move a weight by the query's rounding (2^-21 f32, 2^-14 three terms) times that
    check_attention(c, typ, q=q, tol=max(TOL[typ], 3e3 * 2.0 ** -19 if size > 1 else 0))


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mean", [2, 9, 30, 290])
@pytest.mark.parametrize("size", [3e4, 1e8, 2.0 ** 123])
def test_attention_rows_of_mixed_size(cuda, size, mean, typ):
    """A row is held as exactly beside rows of any other size as alone: TOL for the ordinary rows, each on its
    own, whose bits do not change when the others (a later token, another head) are ordinary, too; a row so large
    that one key has all of its weight gets that key's value."""
    import torch

    if typ == "f16" and size > 65504:
        pytest.skip("past the type's range")
    n = max(1, mean // 2)
    c = Case(cuda, [n, n], [70, 300], kv=1, hd=128, heads=2, page=32, seed=mean)
    q = c.randn(256, typ)
    plain = c.batch.attention(q, freq=freqs(cuda, 64)).clone()
    large = torch.zeros(2 * n, 2, dtype=torch.bool, device=cuda)
    large[n - 1, 1] = large[2 * n - 1, 0] = large[n // 2, 0] = True
    big = q.reshape(-1, 2, 128).clone()
    big[large] = (big[large].double() * (size if typ != "f16" else 4000)).to(big.dtype)
    assert big.isfinite().all()
    got = c.batch.attention(big.reshape(q.shape), freq=freqs(cuda, 64))
    assert check_errors() == 0
    assert torch.equal(got.reshape(-1, 2, 128)[~large], plain.reshape(-1, 2, 128)[~large])
    want = want_attention(c, q, freq=freqs(cuda, 64)).reshape(-1, 2, 128)[~large]
    err = (got.reshape(-1, 2, 128)[~large].double() - want).norm(dim=-1) / want.norm(dim=-1)
    assert (err < TOL[typ]).all(), err.max()
    sure = want_attention(c, big.reshape(q.shape), freq=freqs(cuda, 64)).reshape(-1, 2, 128)[large]
    gap = want_attention(c, big.reshape(q.shape), freq=freqs(cuda, 64), scale=128 ** -0.5 * 0.97).reshape(-1, 2, 128)[large]
    one = (sure == gap).all(-1)      # one key has all of it, and would with scores 3 % nearer to each other
    err = (got.reshape(-1, 2, 128)[large].double() - sure).norm(dim=-1) / sure.norm(dim=-1)
    assert one.any() and (err[one] < TOL[typ]).all(), err


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 12, 40, 300])
@pytest.mark.parametrize("n,mass", [(8000, 0.9), (32768, 0.9), (131072, 0.9), (131072, 0.99)])
def test_attention_small_weights_count(cuda, n, mass, rows, typ):
    """A first token with nearly all of the weight and a value of 0, as models park attention: the output is
    what the other keys' weights, down to 2^-24 of the first one's, make of their values. 152 sequences over
    the same pages, so that a CTA has the whole context of a group under one reference.

    Bound. The values have a mean of half their spread, so the output is about (1 - mass) / 2 of the spread. All weights lie
    above half of the last term's smallest byte (2^-28 of the first token's for bf16, 2^-31 f16, 2^-37 f32), so their
    errors are roundings, as likely up as down, and add as sqrt(n): TOL, as elsewhere."""
    import torch

    from spk import paged

    hd, page, nseq = 64, 128, 152
    g = torch.Generator(device=cuda)
    g.manual_seed(n + rows)
    pages = -(-n // page)
    cache = paged.PagedCache(pages, page, 1, hd, device=cuda)
    k = torch.randn(pages, 1, page, hd, generator=g, device=cuda) * 50
    v = torch.randn(pages, 1, page, hd, generator=g, device=cuda) * 80 + 40
    k[..., 0] = 0
    k[0, 0, :16], v[0, 0, 0] = 0, 0
    k[0, 0, 0, 0] = 400
    cache.k_pool.copy_(pack_k(k.clamp(-440, 440).to(torch.float16)).to(torch.float8_e4m3fn))
    cache.v_pool.copy_(pack_v(v.clamp(-440, 440).to(torch.float16)).to(torch.float8_e4m3fn))
    cache.k_scale.fill_(0.01)
    cache.v_scale.fill_(0.01)
    # the others' weights average e^(1/8): scores of spread 1/2
    first = np.log(mass / (1 - mass) * n) + 0.125
    cache.k_scale[0, 0, 0] = first * hd ** 0.5 / 4 / float(cache.k_pool[0, 0, 0, 0, 0, 0].float())
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    row0, kv_len = i32(np.arange(nseq + 1) * rows), i32([n] * nseq)
    table = torch.arange(pages, dtype=torch.int32, device=cuda).repeat(nseq, 1)
    q = torch.randn(nseq * rows, hd, generator=g, device=cuda).to(ttype(typ))
    q[:, 0] = 4
    b = paged.PagedBatch(cache, row0, kv_len, table, rows=nseq * rows, heads=1)
    got = b.attention(q)
    assert check_errors() == 0
    kk = (unpack_k(cache.k_pool)[:, 0] * cache.k_scale[:, 0].double().repeat_interleave(16, -1)[..., None]).reshape(-1, hd)[:n]
    vv = (unpack_v(cache.v_pool)[:, 0] * 0.01).reshape(-1, hd)[:n]
    hide = torch.arange(n, device=cuda)[None] > torch.arange(n - rows, n, device=cuda)[:, None]
    for s in (0, 77, nseq - 1):
        at = slice(s * rows, (s + 1) * rows)
        w = torch.softmax((q[at].double() @ kk.T / hd ** 0.5).masked_fill(hide, float("-inf")), -1)
        assert abs(w[:, 0].mean().item() - mass) < 0.05
        want = w @ vv
        err = ((got[at].double() - want).norm() / want.norm()).item()
        assert err < TOL[typ], err


def test_attention_ignores_what_no_row_sees(cuda):
    """NaN bytes and scales in pages that are not the sequence's and behind its last block, NaN bytes behind
    its last token in that block, and a poisoned block that only other rows see."""
    import torch

    for typ, rows in (("f32", [1, 2]), ("bf16", [40, 1]), ("f16", [1, 9])):
        c = Case(cuda, rows, [100, 37], kv=2, hd=64, heads=4, page=64, seed=6)
        q = c.randn(c.heads * c.hd, typ)
        want = want_attention(c, q)
        kb, vb = c.cache.k_pool.view(torch.uint8), c.cache.v_pool.view(torch.uint8)
        held = {p for row in c.table for p in row if p >= 0}
        for p in range(c.cache.pages):
            if p not in held:
                kb[p], vb[p] = 0x7f, 0x7f
                c.cache.k_scale[p], c.cache.v_scale[p] = float("nan"), float("inf")
        for s, L in enumerate(c.len):
            pg, o = c.table[s][(L - 1) // 64], (L - 1) % 64
            for t in range(o + 1, 64):
                kb[pg, :, t // 8, :, t % 8] = 0x7f
                vb[pg, :, t // 16, :, ORDER.index(t % 16)] = 0xff
            c.cache.k_scale[pg, :, o // 16 + 1:] = float("nan")
            c.cache.v_scale[pg, :, o // 16 + 1:] = float("nan")
        got = c.batch.attention(q).double()
        assert check_errors() == 0
        assert ((got - want).norm() / want.norm()).item() < TOL[typ]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_attention_poisoned_block_reaches_only_the_rows_that_see_it(cuda, typ):
    import torch

    c = Case(cuda, [120], [20], kv=2, hd=64, heads=4, page=16, seed=3)
    q = c.randn(c.heads * c.hd, typ)
    for window in (0, 16):
        want = want_attention(c, q, window=window)
        c.cache.v_scale[c.table[0][4], 0] = float("nan")      # tokens 64 .. 79 of KV head 0 (heads 0, 1)
        got = c.batch.attention(q, window=window).double().reshape(120, 4, 64)
        c.cache.v_scale[c.table[0][4], 0] = 0.01
        pos = torch.arange(20, 140)
        sees = (pos >= 64) & ((pos - window < 79) if window else torch.ones(120, dtype=torch.bool))
        assert got[sees][:, :2].isnan().all()
        rest = want.reshape(120, 4, 64)
        # the rows before the block, and the other KV head's
        for a, b in ((got[~sees], rest[~sees]), (got[:, 2:], rest[:, 2:])):
            assert a.isfinite().all()
        c.cache.v_scale[c.table[0][4], 0] = 0.01


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_attention_beside_a_poisoned_block_is_what_it_is_without(cuda, which, typ):
    """The rows before a poisoned block, those whose window has left it, and the other KV head's: the same values."""
    import torch

    c = Case(cuda, [120], [20], kv=2, hd=64, heads=4, page=16, seed=3)
    q = c.randn(c.heads * c.hd, typ)
    scale, at = getattr(c.cache, which), (c.table[0][4], 0)       # tokens 64 .. 79 of KV head 0 (heads 0, 1)
    good = scale[at].clone()
    for window in (0, 16):
        want = want_attention(c, q, window=window).reshape(120, 4, 64)
        for bad in (float("nan"), float("inf")):
            scale[at] = bad
            got = c.batch.attention(q, window=window).double().reshape(120, 4, 64)
            scale[at] = good
            assert check_errors() == 0
            pos = torch.arange(20, 140, device=cuda)
            sees = (pos >= 64) & ((pos - window < 79) if window else torch.ones_like(pos, dtype=torch.bool))
            if bad != bad:
                assert got[sees][:, :2].isnan().all()
            assert (~sees).sum() > 40
            for a, b in ((got[~sees], want[~sees]), (got[:, 2:], want[:, 2:])):
                assert (((a - b).norm(dim=-1) / b.norm(dim=-1)) < 4 * TOL[typ]).all()
                assert ((a - b).norm() / b.norm()).item() < TOL[typ]


def test_attention_nan_query_stays_in_its_row(cuda):
    for typ, rows in (("f32", [1]), ("bf16", [50])):
        c = Case(cuda, rows, [70], kv=1, hd=128, heads=4, page=32, seed=2)
        q = c.randn(512, typ)
        want = want_attention(c, q)
        for bad in (float("nan"), float("inf")):
            p = q.clone()
            p[0, 128 + 5] = bad       # row 0, head 1
            got = c.batch.attention(p).double().reshape(-1, 4, 128)
            assert got[0, 1].isnan().all()
            got[0, 1] = want.reshape(-1, 4, 128)[0, 1]
            assert ((got.reshape(-1, 512) - want).norm() / want.norm()).item() < TOL[typ]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_attention_strides(cuda, typ):
    """Rows of q, the gate and the output are views of wider, unaligned matrices."""
    import torch

    c = Case(cuda, [3, 20], [40, 7], kv=2, hd=64, heads=4, page=16, seed=7)
    wide = torch.randn(23, 261, generator=c.g, device=cuda).to(ttype(typ))
    gates = torch.randn(23, 9, generator=c.g, device=cuda).to(ttype(typ))
    out = torch.full((23, 300), 7.0, device=cuda).to(ttype(typ))
    q, gate = wide[:, 3:259], gates[:, 2:6]
    c.batch.attention(q, out[:, 5:261], gate=gate, scale=0.2)
    want = want_attention(c, q, gate=gate, scale=0.2)
    assert ((out[:, 5:261].double() - want).norm() / want.norm()).item() < TOL[typ]
    assert (out[:, :5] == 7).all() and (out[:, 261:] == 7).all()


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_attention_many_sequences(cuda, typ):
    """Hundreds of sequences, most of them short, some without a row: several to a CTA."""
    rng = np.random.default_rng(3)
    rows = rng.integers(0, 4, 700).tolist()
    old = (np.exp(rng.uniform(0, 6, 700))).astype(int).tolist()
    c = Case(cuda, rows, old, kv=2, hd=64, heads=4, page=16, seed=1)
    check_attention(c, typ, window=0)


def test_attention_line_of_work_of_many_heads_a_kv_head(cuda):
    """Thousands of heads on one KV head: 375467 row tiles of 24 columns, 24 / 4096 tokens each. Their lengths add up to
    less than 32 bits only if a tile is not taken to be a token longer than the one before it."""
    import torch

    heads, n, hd = 4096, 2200, 64
    c = Case(cuda, [n], [0], kv=1, hd=hd, heads=heads, page=64, seed=14)
    q = c.randn(heads * hd, "f32")
    out = torch.full_like(q, float("nan"))
    c.batch.attention(q, out)
    assert check_errors() == 0 and out.isfinite().all()
    pg = c.table[0]
    k, v = ((u[pg, 0] * s[pg, 0].double().repeat_interleave(16, -1)[..., None]).reshape(-1, hd)[:n]
            for u, s in ((unpack_k(c.cache.k_pool), c.cache.k_scale), (unpack_v(c.cache.v_pool), c.cache.v_scale)))
    for i in (0, 1, 700, 1500, n - 1):
        want = torch.softmax(q[i].reshape(heads, hd).double() @ k[:i + 1].T / 8, -1) @ v[:i + 1]
        got = out[i].reshape(heads, hd).double()
        assert ((got - want).norm() / want.norm()).item() < TOL["f32"], i


def test_attention_rows_that_see_nothing_are_zero_and_bad_batches_reported(cuda):
    import spk

    c = Case(cuda, [4, 3], [0, 30], kv=2, hd=64, heads=4, page=16, seed=5)
    q = c.randn(256, "f32")
    c.kv_len[0] = 2        # rows at positions -2 .. 1: the first two see nothing
    c.len[0] = 2
    out = c.batch.attention(q)
    assert check_errors() == 0
    assert (out[:2] == 0).all() and out[2:].abs().sum(-1).min() > 0
    for spoil in ("page", "rows", "length"):
        c = Case(cuda, [4, 3], [0, 30], kv=2, hd=64, heads=4, page=16, seed=5)
        if spoil == "page":
            c.tab[1, 1] = -1
        elif spoil == "rows":
            c.row0[2] = 8
        else:
            c.kv_len[1] = 100000
        c.batch.attention(c.randn(256, "f32"))
        assert check_errors() == -1 and "index" in spk.last_error(), spoil
        assert check_errors() == 0


def test_frequencies_are_f32_side_by_side_on_the_rows_device(cuda):
    """Anything else would be read past its end or as other numbers."""
    import torch

    import spk

    c = Case(cuda, [2, 1], [5, 30], kv=2, hd=64, heads=4, page=16, seed=3)
    q, k, v, good = c.randn(256, "f32"), c.randn(128, "f32"), c.randn(128, "f32"), freqs(cuda, 32)
    before = c.cache.k_pool.view(torch.uint8).clone()
    wide = torch.zeros(16, 2, device=cuda)
    wide[:, 0] = good
    for bad in (good.double(), good.half(), good.bfloat16(), good.int(), wide[:, 0], good.flip(0)[::2], good.cpu(), freqs(cuda, 64)[:31],
                freqs(cuda, 128)):
        for call in (lambda: c.batch.append(k, v, freq=bad), lambda: c.batch.attention(q, freq=bad)):
            with pytest.raises(spk.SpkError):
                call()
    torch.cuda.synchronize()
    assert torch.equal(before, c.cache.k_pool.view(torch.uint8))
    check_append(c, k, v, wide[:, 0].contiguous())
    check_attention(c, "f32", q=q, freq=good)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [[1], [300]])
def test_attention_of_scores_that_are_all_far_below_zero(cuda, rows, typ):
    """Every key the same and every query its opposite, of any size: the mean of the values seen, in one part or in many."""
    import torch

    c = Case(cuda, rows, [20000], kv=1, hd=64, heads=1, page=64, seed=5)
    c.cache.k_pool.copy_(c.cache.k_pool[0, 0, 0, :, :1].expand_as(c.cache.k_pool))
    c.cache.k_scale.fill_(0.01)
    c.cache.v_scale.fill_(0.01)
    q = -unpack_k(c.cache.k_pool[:1])[0, 0, :1].expand(rows[0], 64)
    v = (unpack_v(c.cache.v_pool)[:, 0] * 0.01)[c.table[0]].reshape(-1, 64)
    mean = (v.cumsum(0) / torch.arange(1, len(v) + 1, device=cuda)[:, None])[20000:20000 + rows[0]]
    for size in (1e-3, 1e25, 1e33):
        got = c.batch.attention((q * size).to(ttype(typ))).double()
        assert check_errors() == 0
        assert ((got - mean).norm() / mean.norm()).item() < TOL[typ], size


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,old", [([1], [40000]), ([9, 1, 30], [3000, 500, 9000]), ([400], [2000])])
def test_attention_repeats_itself_bit_for_bit(cuda, rows, old, typ):
    """Parts of a group are joined in the CTAs' order, whichever comes last."""
    import torch

    c = Case(cuda, rows, old, kv=2, hd=128, heads=8, page=64, seed=len(rows))
    q = c.randn(c.heads * c.hd, typ)
    first = c.batch.attention(q, freq=freqs(cuda, 64)).clone()
    for _ in range(20):
        assert torch.equal(c.batch.attention(q, freq=freqs(cuda, 64)), first)
    assert check_errors() == 0


def test_calls_without_rows(cuda):
    import torch

    from spk import paged, score

    c = Case(cuda, [3, 2], [5, 30], kv=2, hd=64, heads=4, page=16, seed=3)
    s = torch.cuda.Stream()
    none = paged.PagedBatch(c.cache, torch.zeros(3, dtype=torch.int32, device=cuda), c.kv_len, c.tab, rows=0, heads=4)
    before = c.cache.k_pool.view(torch.uint8).clone()
    e = lambda w: torch.empty(0, w, device=cuda)  # noqa: E731
    for stream in (None, s):
        none.append(e(128), e(128), stream=stream)
        assert none.attention(e(256), stream=stream).shape == (0, 256)
        lp = score.LogProbs(0, 100, 3, device=cuda)
        logp, ent, ids, best = lp(e(100), torch.empty(0, dtype=torch.int32, device=cuda), stream=stream)
        assert logp.numel() == 0 and ids.shape == (0, 3)
    torch.cuda.synchronize()
    assert check_errors() == 0 and torch.equal(before, c.cache.k_pool.view(torch.uint8))


def test_append_then_attention_is_attention_over_the_rounded_rows(cuda):
    """The two together, over pages as they come, against attention in 64 bits over what the cache holds."""
    c = Case(cuda, [60, 1, 9], [10, 200, 0], kv=4, hd=256, heads=16, page=32, seed=11)
    f = freqs(cuda, 64, 5e6)
    qkv = c.randn(24 * 256, "bf16")
    q, k, v = qkv[:, :4096], qkv[:, 4096:5120], qkv[:, 5120:]
    c.batch.append(k, v, freq=f)
    check_attention(c, "bf16", q=q, freq=f)


def test_on_a_stream_and_in_a_graph(cuda):
    """Calls go to torch's current stream; a captured graph follows the batch's arrays."""
    import torch

    c = Case(cuda, [1, 1], [40, 99], kv=2, hd=128, heads=8, page=64, seed=12)
    c.table = [[0, 1, 2], [3, 4, 5]]
    c.tab = torch.tensor(c.table, dtype=torch.int32, device=cuda)
    from spk import paged

    c.cache = paged.PagedCache(6, 64, 2, 128, device=cuda)
    for t in (c.cache.k_pool, c.cache.v_pool):
        t.view(torch.uint8).zero_()
    c.cache.k_scale.fill_(0.01)
    c.cache.v_scale.fill_(0.01)
    c.batch = paged.PagedBatch(c.cache, c.row0, c.kv_len, c.tab, rows=2, heads=8)
    f, qkv, out = freqs(cuda, 128), c.randn(12 * 128, "f32"), torch.empty(2, 1024, device=cuda)
    q, k, v = qkv[:, :1024], qkv[:, 1024:1280], qkv[:, 1280:]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.batch.append(k, v, freq=f)
        c.batch.attention(q, out, freq=f)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.batch.append(k, v, freq=f)
            c.batch.attention(q, out, freq=f)
    torch.cuda.synchronize()
    for step in range(4):
        c.kv_len += 1
        c.len = [n + 1 for n in c.len]
        qkv.copy_(torch.randn(qkv.shape, generator=c.g, device=cuda))
        g.replay()
        torch.cuda.synchronize()
        want = want_attention(c, q, freq=f)
        assert ((out.double() - want).norm() / want.norm()).item() < TOL["f32"]
    assert check_errors() == 0


def test_a_given_stream_is_ordered_with_the_objects_own_buffers(cuda):
    """Calls on a stream of their own while the current one is busy: the output does not take memory that the
    current stream still reads, the workspace's zeroing and the pool's earlier owner are waited for, and what is
    dropped after the call is not handed out again before the call has read it."""
    import torch

    from spk import paged

    kv, hd, n = 2, 128, 3000
    g = torch.Generator(device=cuda)
    g.manual_seed(6)
    q, k, v = (torch.randn(n, w * hd, generator=g, device=cuda) for w in (8, 2, 2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    row0, kv_len, table = i32([0, n]), i32([n]), torch.arange(47, dtype=torch.int32, device=cuda)[None].contiguous()
    cache = paged.PagedCache(47, 64, kv, hd, device=cuda)
    batch = paged.PagedBatch(cache, row0, kv_len, table, rows=n, heads=8)
    batch.append(k, v)
    want = batch.attention(q).clone()
    pools = [t.view(torch.uint8).clone() for t in (cache.k_pool, cache.v_pool)]
    busy = lambda: torch.cuda._sleep(100_000_000)   # noqa: E731  (some 50 ms)
    s = torch.cuda.Stream()
    for _ in range(3):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        # memory that the current stream reads late and that is free for its next owner
        old = [torch.full((n, 8 * hd), 7.0, device=cuda), torch.full_like(pools[0], 9), torch.full_like(pools[1], 9),
               torch.full_like(batch.workspace, 255)]
        busy()
        kept = [t.clone() for t in old]
        del old
        c2 = paged.PagedCache(47, 64, kv, hd, device=cuda)
        b2 = paged.PagedBatch(c2, row0, kv_len, table, rows=n, heads=8)
        b2.append(k, v, stream=s)
        out = b2.attention(q, stream=s)
        torch.cuda.synchronize()
        assert all((t == x).all() for t, x in zip(kept, (7.0, 9, 9, 255)))
        assert torch.equal(out, want)
        assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(pools, (c2.k_pool, c2.v_pool)))
    # dropped after the call, which comes late
    args = [t.clone() for t in (q, k, v, row0, kv_len, table)]
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        busy()
    b3 = paged.PagedBatch(cache, *args[3:], rows=n, heads=8)
    b3.append(args[1], args[2], stream=s)
    out = b3.attention(args[0], stream=s)
    shapes = [(t.shape, t.dtype) for t in args] + [(b3.workspace.shape, torch.uint8)]
    del args, b3
    junk = [torch.full(sh, 99, dtype=dt, device=cuda) for sh, dt in shapes for _ in range(2)]
    torch.cuda.synchronize()
    assert torch.equal(out, want) and check_errors() == 0
    del junk


def test_offsets_past_32_bits(cuda):
    """Pages whose bytes lie past 4 GiB of the pool."""
    import torch

    from spk import paged

    pages, page, kv, hd = 9300, 128, 8, 512 // 2
    cache = paged.PagedCache(pages, page, kv, hd, device=cuda)       # 2.4 GB of 2^31 + each
    assert cache.k_pool.numel() > 2 ** 31
    c = Case(cuda, [130], [0], kv=kv, hd=hd, heads=8, page=page, seed=13)
    c.cache, c.table = cache, [[pages - 1, 2, pages - 2]]
    c.tab = torch.tensor(c.table, dtype=torch.int32, device=cuda)
    c.batch = paged.PagedBatch(cache, c.row0, c.kv_len, c.tab, rows=130, heads=8)
    k, v, q = c.randn(kv * hd, "bf16"), c.randn(kv * hd, "bf16"), c.randn(8 * hd, "bf16")
    c.batch.append(k, v)
    got = c.batch.attention(q).double().reshape(130, 8, hd)
    assert check_errors() == 0
    kk, vv = (torch.cat([p[pages - 1].cpu(), p[2].cpu()], 1).double()[:, :130].to(cuda)
              for p in (unpack_pages(cache, "k", c.table[0][:2]), unpack_pages(cache, "v", c.table[0][:2])))
    for h in range(8):
        w = q[:, h * hd:(h + 1) * hd].double() @ kk[h].T / 16
        w = w.masked_fill(torch.ones(130, 130, device=cuda).triu(1).bool(), float("-inf"))
        want = torch.softmax(w, -1) @ vv[h]
        assert ((got[:, h] - want).norm() / want.norm()).item() < TOL["bf16"]


def test_offsets_past_2_to_the_32(cuda):
    """Pages whose bytes lie past 2^32 of the pool, rows whose elements lie past 2^31 of their matrix."""
    import torch

    from spk import paged

    pages, page, kv, hd, n, ld = 17000, 128, 8, 256, 3, 2 ** 30 + 24
    cache = paged.PagedCache(pages, page, kv, hd, device=cuda)
    assert (pages - 2) * kv * page * hd > 2 ** 32 and 2 * ld > 2 ** 31
    c = Case(cuda, [n], [127], kv=kv, hd=hd, heads=kv, page=page, seed=15)
    c.cache, c.table = cache, [[pages - 1, pages - 2]]
    c.tab = torch.tensor(c.table, dtype=torch.int32, device=cuda)
    store = torch.empty(n * ld, dtype=torch.bfloat16, device=cuda)
    row = lambda o, w: store[o:].as_strided((n, w), (ld, 1))  # noqa: E731
    q, k, v, out = row(0, kv * hd), row(2048, kv * hd), row(4096, kv * hd), row(6144, kv * hd)
    c.rows = [127]
    c.len = [127]
    first = paged.PagedBatch(cache, torch.tensor([0, 127], dtype=torch.int32, device=cuda),
                             torch.tensor([127], dtype=torch.int32, device=cuda), c.tab, rows=127, heads=kv)
    kk, vv = c.randn(kv * hd, "bf16"), c.randn(kv * hd, "bf16")
    first.append(kk, vv)
    for t in (q, k, v):
        t.copy_(torch.randn(n, kv * hd, generator=c.g, device=cuda))
    b = paged.PagedBatch(cache, c.row0, c.kv_len, c.tab, rows=n, heads=kv)
    b.append(k, v)
    b.attention(q, out)
    assert check_errors() == 0
    for name, rows in (("k", torch.cat([kk, k])), ("v", torch.cat([vv, v]))):
        got = unpack_pages(cache, name, c.table[0])
        got = torch.cat([got[p] for p in c.table[0]], 1)[:, :130].transpose(0, 1).reshape(130, -1)
        assert ((got - rows.double()).norm() / rows.double().norm()).item() < 2 ** -4
        kk, vv = (got, vv) if name == "k" else (kk, got)
    w = torch.einsum("ihd,jhd->hij", q.double().reshape(n, kv, hd), kk.reshape(130, kv, hd)) / 16
    w = w.masked_fill(torch.arange(130, device=cuda)[None] > torch.arange(127, 130, device=cuda)[:, None], float("-inf"))
    want = torch.einsum("hij,jhd->ihd", torch.softmax(w, -1), vv.reshape(130, kv, hd)).reshape(n, -1)
    assert ((out.double() - want).norm() / want.norm()).item() < TOL["bf16"]


def unpack_pages(cache, name, pages):
    """{page: values [kv][tokens][hd]} of some pages."""
    out = {}
    for p in pages:
        if name == "k":
            out[p] = unpack_k(cache.k_pool[p:p + 1])[0] * cache.k_scale[p].double().repeat_interleave(16, -1)[..., None]
        else:
            out[p] = unpack_v(cache.v_pool[p:p + 1])[0] * cache.v_scale[p].double().repeat_interleave(16, -1)[..., None]
    return out
