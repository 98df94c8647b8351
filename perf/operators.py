"""The batched serving operators as workloads: their cases, inputs, plain forms and definitions.

Three operators that one served or scored batch runs after each other:

  append     new keys (rotated on the way) and values go into the pages of an 8-bit cache with one
             scale per 16-token block and KV head
  attention  causal grouped-query attention of each sequence's new rows over its pages
  logprobs   log probability of a given token, entropy and best alternatives of each row of logits

Cache bytes (e4m3). A page holds `page` tokens per KV head. Keys [page/8][hd/16][8 tokens][16 dims];
values [page/16][hd][16 tokens], the tokens of a block in the order ORDER. Token p of sequence s lies
in page table[s][p // page] at p % page.
"""
import os
import random
import sys

import torch

own = False

BLOCK = 16
ORDER = [0, 1, 8, 9, 2, 3, 10, 11, 4, 5, 12, 13, 6, 7, 14, 15]   # the tokens of a value block, as they lie
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -100
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------ cases

def listed():
    # `ctx`: cached tokens of the longest sequence before the call, `new`: rows of the longest one in
    # the call; `ragged`: the others are shorter, some empty. The decoder's own heads: 16 over 4 of 256,
    # window 512, rotation over 64 (full layers) or 256 dims (sliding ones), 131072 tokens.
    dec = {"heads": 16, "kv": 4, "hd": 256}
    gqa8 = {"heads": 32, "kv": 4, "hd": 128}
    return [
        # one decode step of one sequence: the call is latency
        {"name": "append-1-token", "op": "append", **dec, "type": "f32", "nseq": 1, "new": 1, "ctx": 4103, "ragged": False, "page": 64, "pdim": 64},
        # one decode step of a full batch, heads of 128
        {"name": "append-batch-step", "op": "append", **gqa8, "type": "f16", "nseq": 96, "new": 1, "ctx": 6000, "ragged": True, "page": 32, "pdim": 128},
        # prompts of mixed lengths that arrive together
        {"name": "append-prompts", "op": "append", **dec, "type": "f32", "nseq": 13, "new": 1501, "ctx": 700, "ragged": True, "page": 64, "pdim": 256},
        # one long prompt in one call
        {"name": "append-long-prompt", "op": "append", **dec, "type": "bf16", "nseq": 1, "new": 16384, "ctx": 0, "ragged": False, "page": 128, "pdim": 64},
        # one decode step of one sequence on a sliding layer: the smallest call
        {"name": "attn-window-step", "op": "attention", **dec, "type": "f32", "nseq": 1, "new": 1, "ctx": 4103, "ragged": False, "page": 64, "pdim": 256, "window": 512, "gate": True},
        # one decode step of one sequence at the decoder's full context
        {"name": "attn-long-step", "op": "attention", **dec, "type": "f32", "nseq": 1, "new": 1, "ctx": 131071, "ragged": False, "page": 128, "pdim": 64, "window": 0, "gate": True},
        # one decode step of a batch with lengths from a few tokens to 9000
        {"name": "attn-batch-step", "op": "attention", **dec, "type": "bf16", "nseq": 64, "new": 1, "ctx": 9000, "ragged": True, "page": 64, "pdim": 64, "window": 0, "gate": True},
        # drafted tokens of a batch verified at once (an anchor and 7 proposals each)
        {"name": "attn-verify", "op": "attention", **gqa8, "type": "f16", "nseq": 24, "new": 8, "ctx": 5000, "ragged": True, "page": 32, "pdim": 128, "window": 0, "gate": False},
        # a chunk of a long prompt over what is cached
        {"name": "attn-prompt-chunk", "op": "attention", **dec, "type": "bf16", "nseq": 1, "new": 2048, "ctx": 6144, "ragged": False, "page": 128, "pdim": 64, "window": 0, "gate": True},
        # one generated token with its alternatives
        {"name": "logprobs-1-row", "op": "logprobs", "type": "f32", "rows": 1, "vocab": 131072, "top": 20, "pad": 0},
        # a scored batch over an odd vocabulary, rows padded
        {"name": "logprobs-odd", "op": "logprobs", "type": "f16", "rows": 61, "vocab": 50021, "top": 1, "pad": 11},
        # a scored prompt chunk
        {"name": "logprobs-prompt", "op": "logprobs", "type": "bf16", "rows": 1024, "vocab": 131072, "top": 5, "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "logprobs", "logprobs"])
    typ = rng.choice(["f32", "f16", "bf16"])
    if op == "logprobs":
        vocab = _log(rng, 1000, 131072)
        return {"op": op, "type": typ, "rows": _log(rng, 1, min(2048, 2 ** 27 // vocab)), "vocab": vocab,
                "top": rng.choice([0, 1, 2, 5, 8, 20]), "pad": rng.choice([0, 0, 1, 8])}
    hd = rng.choice([64, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 8])
    c = {"op": op, "heads": heads, "kv": kv, "hd": hd, "type": typ, "page": rng.choice([16, 32, 48, 64, 128]),
         "pdim": rng.choice([0, hd // 4, hd // 2, hd]), "ragged": rng.random() < 0.6}
    if op == "append":
        c["nseq"] = _log(rng, 1, 128)
        c["new"] = _log(rng, 1, max(2, min(16384, 2 ** 24 // (c["nseq"] * kv * hd))))
        c["ctx"] = rng.choice([0, _log(rng, 1, 30000)])
        return c
    kind = rng.choice(["step", "verify", "chunk"])
    c["window"] = rng.choice([0, 0, 0, _log(rng, 8, 2048)])
    c["gate"] = rng.random() < 0.5
    if kind == "chunk":
        c["nseq"] = _log(rng, 1, 8)
        c["new"] = _log(rng, 16, 2048 // c["nseq"])
        c["ctx"] = rng.choice([0, _log(rng, 1, 6144)])
        if c["nseq"] * c["new"] * heads * (c["new"] + c["ctx"]) * hd > 2048 * 16 * 8192 * 256:
            c["new"] = max(16, c["new"] // 4)
    else:
        c["nseq"] = _log(rng, 1, 64)
        c["new"] = 1 if kind == "step" else rng.randint(2, 8)
        c["ctx"] = _log(rng, 1, max(64, min(131000, 2 ** 29 // (c["nseq"] * kv * hd * 2 * c["new"]))))
    return c


def _lengths(case):
    """Rows in the call and cached tokens after it, of every sequence: by the case alone."""
    n, new, ctx = case["nseq"], case["new"], case["ctx"]
    if not case["ragged"]:
        return [new] * n, [ctx + new] * n
    r = random.Random(n * 1000003 + new * 1009 + ctx)
    rows = [new if s == 0 else (0 if s % 7 == 3 else _log(r, 1, new)) for s in range(n)]
    old = [ctx if s == 0 or ctx == 0 else (0 if s % 11 == 5 else _log(r, 1, ctx)) for s in range(n)]
    return rows, [a + b for a, b in zip(rows, old)]


def _seen(n, length, window):
    """Tokens that some row of a sequence sees, and (row, token) pairs that are seen."""
    if n == 0:
        return 0, 0
    first = length - n
    pairs = sum(min(p + 1, window) if window else p + 1 for p in range(first, length))
    return length - (max(0, first + 1 - window) if window else 0), pairs


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}
    rows, length = _lengths(case)
    kv, hd, heads = case["kv"], case["hd"], case["heads"]
    if case["op"] == "append":
        vals = 2 * sum(rows) * kv * hd
        blocks = sum((L + 15) // 16 - (L - n) // 16 for n, L in zip(rows, length) if n)
        return {"bytes": vals * (size + 1) + blocks * kv * 8, "flops": 6 * vals}
    seen = [_seen(n, L, case["window"]) for n, L in zip(rows, length)]
    cached = sum(s for s, _ in seen) * kv * 2 * (hd + 4 / BLOCK)
    return {"bytes": int(cached + 2 * sum(rows) * heads * hd * size + (sum(rows) * heads * size if case["gate"] else 0)),
            "flops": 4 * sum(p for _, p in seen) * heads * hd}


# ----------------------------------------------------------------------------------------- inputs

def _freq(pdim, dev):
    theta = 5e6 if pdim <= 64 else 1e4
    return (1.0 / torch.pow(torch.tensor(theta, dtype=torch.float32), torch.arange(0, pdim, 2, dtype=torch.float32) / pdim)).to(dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7919 + 17)
    t = TYPES[case["type"]]
    if case["op"] == "logprobs":
        # logits of a head: a broad background and a few likely tokens; some are masked out
        rows, vocab = case["rows"], case["vocab"]
        x = torch.empty(rows, vocab + case["pad"], dtype=t, device=dev)
        x.normal_(0, 2.5, generator=g)
        hot = torch.randint(0, vocab, (rows, 8), generator=g, device=dev)
        x.scatter_add_(1, hot, torch.rand(rows, 8, generator=g, device=dev).mul_(14).to(t))
        off = torch.randint(0, vocab, (rows, 16), generator=g, device=dev)
        x.scatter_(1, off, torch.full((rows, 16), float("-inf"), dtype=t, device=dev))
        target = torch.where(torch.rand(rows, generator=g, device=dev) < 0.7, hot[:, 0],
                             torch.randint(0, vocab, (rows,), generator=g, device=dev)).to(torch.int32)
        st = {"op": "logprobs", "logits": x[:, :vocab], "target": target, "top": case["top"]}
        if own:
            st["plan"] = _spk("score").LogProbs(rows, vocab, case["top"], device=dev)
        return st

    rows, length = _lengths(case)
    nseq, page, kv, hd, heads, pdim = case["nseq"], case["page"], case["kv"], case["hd"], case["heads"], case["pdim"]
    ntok = sum(rows)
    width = max(1, max((L + page - 1) // page for L in length))
    need = sum((L + page - 1) // page for L in length)
    pages = need + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((nseq, width), -1, dtype=torch.int32, device=dev)
    at = 0
    for s, L in enumerate(length):
        n = (L + page - 1) // page
        table[s, :n] = order[at:at + n]
        at += n
    st = {"op": case["op"], "heads": heads, "kv": kv, "hd": hd, "page": page, "ntok": ntok,
          "row0": torch.tensor([sum(rows[:s]) for s in range(nseq + 1)], dtype=torch.int32, device=dev),
          "kv_len": torch.tensor(length, dtype=torch.int32, device=dev), "table": table,
          "new": max(rows), "longest": max(length),
          "freq": _freq(pdim, dev) if pdim else None}
    # what is cached: rows of about unit size, kept in 8 bits under scales that differ by block
    shape = (pages, kv, page // 8, hd // 16, 8, 16), (pages, kv, page // BLOCK, hd, BLOCK)
    for name, sh in zip("kv", shape):
        st[name + "_pool"] = torch.empty(sh, device=dev, dtype=torch.float16).normal_(0, 90, generator=g).clamp_(-440, 440).to(torch.float8_e4m3fn)
        st[name + "_scale"] = torch.rand(pages, kv, page // BLOCK, generator=g, device=dev).mul_(0.02).add_(0.002)
    # the projections of a step come out side by side: q heads, then k, then v
    qkv = torch.empty(ntok, (heads + 2 * kv) * hd, dtype=t, device=dev).normal_(0, 1, generator=g)
    st["q"], st["k"], st["v"] = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kv) * hd], qkv[:, (heads + kv) * hd:]
    if case["op"] == "attention":
        st["window"] = case["window"]
        st["gate"] = torch.empty(ntok, heads, dtype=t, device=dev).normal_(0, 1, generator=g) if case["gate"] else None
        st["out"] = torch.empty(ntok, heads * hd, dtype=t, device=dev)
    if own:
        paged = _spk("paged")
        cache = paged.PagedCache(pages, page, kv, hd, device=dev)
        for name in ("k_pool", "v_pool", "k_scale", "v_scale"):
            getattr(cache, name).copy_(st[name])
            st[name] = getattr(cache, name)
        st["batch"] = paged.PagedBatch(cache, st["row0"], st["kv_len"], table, rows=ntok, heads=heads)
    return st


def _spk(name):
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spark-x2.6-4b-q6k_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import importlib

    return importlib.import_module("spk." + name)


def run(st):
    if own:
        if st["op"] == "logprobs":
            return st["plan"](st["logits"], st["target"])
        if st["op"] == "append":
            st["batch"].append(st["k"], st["v"], freq=st["freq"])
            return st["k_pool"], st["v_pool"], st["k_scale"], st["v_scale"]
        return st["batch"].attention(st["q"], st["out"], window=st["window"], freq=st["freq"], gate=st["gate"])
    return {"append": _append, "attention": _attention, "logprobs": _logprobs}[st["op"]](st)


# ------------------------------------------------------------------------------------ plain forms

def _places(st):
    """Sequence and position of every row."""
    row = torch.arange(st["ntok"], device=st["row0"].device)
    seq = torch.searchsorted(st["row0"][1:].long(), row, right=True)
    n = st["row0"][1:] - st["row0"][:-1]
    return seq, row - st["row0"][seq] + (st["kv_len"] - n)[seq]


def _rotate(x, pos, freq):
    """x [rows][heads][hd] in 32 bits; the angle is the 32-bit product of position and frequency."""
    if freq is None:
        return x
    h = freq.numel()
    ang = pos.float()[:, None] * freq
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)


def _append(st):
    kv, hd, page, dev = st["kv"], st["hd"], st["page"], st["row0"].device
    seq, pos = _places(st)
    place = torch.tensor([ORDER.index(i) for i in range(BLOCK)], device=dev)
    n = (st["row0"][1:] - st["row0"][:-1]).long()
    first, last = st["kv_len"].long() - n, st["kv_len"].long() - 1
    any_new = n > 0
    pg, off = st["table"][seq, pos // page].long(), pos % page
    # the first and the last block that each sequence touches
    firstc, lastc, every = first.clamp(max=st["table"].shape[1] * page - 1), last.clamp(min=0), torch.arange(n.numel(), device=dev)
    pf, of = st["table"][every, firstc // page].long().clamp(min=0), firstc % page
    pl, ol = st["table"][every, lastc // page].long().clamp(min=0), lastc % page
    r = torch.arange(BLOCK, device=dev)
    for name in "kv":
        x = st[name].float().view(-1, kv, hd)
        if name == "k":
            x = _rotate(x, pos, st["freq"])
        pool, scale = st[name + "_pool"], st[name + "_scale"]
        bytes_ = pool.view(torch.uint8)

        def rows_of(p, o):   # the 16 rows of the block at offset o of page p: indices
            if name == "k":
                t = (o // BLOCK * BLOCK)[:, None] + r
                return p[:, None], slice(None), t // 8, slice(None), t % 8
            return p[:, None], slice(None), (o // BLOCK)[:, None].expand(-1, BLOCK), slice(None), place.expand(p.numel(), -1)

        # scales: the largest value of the call's rows in a block, and what the block had
        flat = (pg * kv)[:, None] * (page // BLOCK) + torch.arange(kv, device=dev) * (page // BLOCK) + (off // BLOCK)[:, None]
        old = scale.clone().view(-1)
        top = torch.full_like(old, -1.0).scatter_reduce(0, flat.view(-1), x.abs().amax(-1).view(-1), "amax")
        new = torch.where(top < 0, old, (top / E4M3_MAX).clamp(min=SCALE_MIN))
        ff = (pf * kv)[:, None] * (page // BLOCK) + torch.arange(kv, device=dev) * (page // BLOCK) + (of // BLOCK)[:, None]
        part = (any_new & (of % BLOCK > 0))[:, None]
        new = new.scatter(0, ff.view(-1), torch.where(part, torch.maximum(new[ff], old[ff]), new[ff]).view(-1))
        # rows that the first block held: rounded again where its scale grew
        at = rows_of(pf, of)
        had = bytes_[at].view(torch.float8_e4m3fn).float().view(-1, BLOCK, kv, hd)
        grew = new[ff] > old[ff]
        ratio = torch.where(grew, old[ff] / new[ff], torch.ones_like(new[ff]))
        had = (had * ratio[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        keep = part[:, :, None, None] & (r < (of % BLOCK)[:, None])[:, :, None, None]
        now = bytes_[at]
        bytes_[at] = torch.where(keep, had, now.view(-1, BLOCK, kv, hd)).view_as(now)
        # the new rows
        q = (x * (1.0 / new[flat])[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        if name == "k":
            bytes_[pg, :, off // 8, :, off % 8] = q.view(-1, kv, hd // 16, 16)
        else:
            bytes_[pg, :, off // BLOCK, :, place[off % BLOCK]] = q
        # nothing after the last one
        at = rows_of(pl, ol)
        now = bytes_[at]
        drop = any_new[:, None, None, None] & (r > (ol % BLOCK)[:, None])[:, :, None, None]
        bytes_[at] = torch.where(drop, torch.zeros_like(now.view(-1, BLOCK, kv, hd)), now.view(-1, BLOCK, kv, hd)).view_as(now)
        scale.view(-1).copy_(new)
    return st["k_pool"], st["v_pool"], st["k_scale"], st["v_scale"]


def _cached(st, name, width):
    """[nseq][kv][width tokens][hd] in 32 bits."""
    kv, hd, page = st["kv"], st["hd"], st["page"]
    tab = st["table"].long().clamp(min=0)
    x = st[name + "_pool"].view(torch.uint8)[tab].view(torch.float8_e4m3fn).float()
    scale = st[name + "_scale"][tab]
    if name == "k":     # [nseq][pages][kv][page/8][hd/16][8][16]
        x = x.permute(0, 2, 1, 3, 5, 4, 6).reshape(tab.shape[0], kv, -1, hd)
    else:               # [nseq][pages][kv][page/16][hd][16]
        inv = torch.tensor([ORDER.index(i) for i in range(BLOCK)], device=x.device)
        x = x[..., inv].permute(0, 2, 1, 3, 5, 4).reshape(tab.shape[0], kv, -1, hd)
    x.view(*x.shape[:2], -1, BLOCK, hd).mul_(scale.permute(0, 2, 1, 3).reshape(tab.shape[0], kv, -1)[..., None, None])
    return x[:, :, :width]


def _attention(st):
    heads, kv, hd, nseq = st["heads"], st["kv"], st["hd"], st["kv_len"].numel()
    seq, pos = _places(st)
    k, v = _cached(st, "k", st["longest"]), _cached(st, "v", st["longest"])
    q = _rotate(st["q"].float().view(-1, heads, hd), pos, st["freq"])
    row = torch.arange(st["ntok"], device=q.device) - st["row0"][seq]
    qp = q.new_zeros(nseq, st["new"], heads, hd)
    qp[seq, row] = q
    at = torch.full((nseq, st["new"]), -1, dtype=torch.long, device=q.device)
    at[seq, row] = pos.long()
    j = torch.arange(st["longest"], device=q.device)
    see = j <= at[..., None]
    if st["window"]:
        see &= j > at[..., None] - st["window"]
    qp = qp.view(nseq, st["new"], kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(nseq, kv, -1, hd)
    s = torch.matmul(qp, k.transpose(-1, -2)).view(nseq, kv, heads // kv, st["new"], -1) * hd ** -0.5
    s.masked_fill_(~see[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    del s
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(nseq, kv, -1, p.shape[-1]), v).view(nseq, kv, heads // kv, st["new"], hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(nseq, st["new"], heads, hd)[seq, row]
    if st["gate"] is not None:
        o = o / (1 + torch.exp(-st["gate"].float()))[..., None]
    return o.reshape(st["ntok"], heads * hd).to(st["q"].dtype)


def _logprobs(st):
    x = st["logits"].float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(-1)
    lse = m[:, 0] + torch.log(total)
    got = x.gather(1, st["target"].long()[:, None])[:, 0] - lse
    ent = torch.log(total) - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(-1) / total
    best, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    top = st["top"]
    return got, ent, ids[:, :top].to(torch.int32), best[:, :top] - lse[:, None]


# ------------------------------------------------------------------------- definitions in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        x = st["logits"].double()
        lse = torch.logsumexp(x, -1)
        lp = x - lse[:, None]
        ent = torch.special.entr(lp.exp()).sum(-1)
        ids = torch.argsort(lp, dim=-1, descending=True, stable=True)[:, :case["top"]]
        return lp[torch.arange(case["rows"]), st["target"].long()], ent, ids.to(torch.int32), lp.gather(1, ids)

    rows, length = _lengths(case)
    kv, hd, page, heads = case["kv"], case["hd"], case["page"], case["heads"]
    table = st["table"].tolist()

    def turned(x, positions):    # x [n][heads][hd]; angles as the format has them: f32(position * frequency)
        if st["freq"] is None:
            return x
        h = st["freq"].numel()
        ang = (torch.tensor(positions, dtype=torch.float32, device=x.device)[:, None] * st["freq"][None]).double()
        z = torch.complex(x[..., :h], x[..., h:2 * h]) * torch.polar(torch.ones_like(ang), ang)[:, None]
        return torch.cat([z.real, z.imag, x[..., 2 * h:]], -1)

    def logical(name):           # the pool as [pages][kv][tokens][hd], in 64 bits
        p = st[name + "_pool"].double()
        if name == "k":
            return p.transpose(3, 4).reshape(p.shape[0], kv, page, hd)
        y = torch.empty(p.shape[0], kv, page // BLOCK, BLOCK, hd, dtype=torch.float64, device=p.device)
        for i, token in enumerate(ORDER):
            y[:, :, :, token] = p[..., i]
        return y.view(p.shape[0], kv, page, hd)

    if case["op"] == "append":
        out = []
        for name in "kv":
            p, sc = logical(name), st[name + "_scale"].double()
            x = st[name].double().reshape(-1, kv, hd)
            at = 0
            for s, (n, L) in enumerate(zip(rows, length)):
                new = x[at:at + n]
                at += n
                if n and name == "k":
                    new = turned(new, list(range(L - n, L)))
                first = L - n
                b = first // BLOCK * BLOCK
                while n and b < L:      # block by block: positions b .. b + 15
                    pg, o = table[s][b // page], b % page
                    lo, hi = max(b, first), min(b + BLOCK, L)
                    vals = new[lo - first:hi - first]
                    d = vals.abs().amax((0, 2)).div(E4M3_MAX).clamp(min=SCALE_MIN)
                    if lo > b:
                        was = sc[pg, :, o // BLOCK].clone()
                        d = torch.maximum(d, was)
                        p[pg, :, o:o + lo - b] *= (was / d)[:, None, None]
                    sc[pg, :, o // BLOCK] = d
                    p[pg, :, o + lo - b:o + hi - b] = (vals / d[None, :, None]).transpose(0, 1)
                    p[pg, :, o + hi - b:o + BLOCK] = 0
                    b += BLOCK
            if name == "k":
                p = p.view(-1, kv, page // 8, 8, hd // 16, 16).transpose(3, 4)
            else:
                p = p.view(-1, kv, page // BLOCK, BLOCK, hd)[:, :, :, ORDER].transpose(3, 4)
            out += [p.contiguous(), sc]
        return out[0], out[2], out[1], out[3]

    k, v = (logical(name).view(-1, kv, page // BLOCK, BLOCK, hd) * st[name + "_scale"].double()[..., None, None] for name in "kv")
    out, at = [], 0
    for s, (n, L) in enumerate(zip(rows, length)):
        if n == 0:
            continue
        take = torch.tensor(table[s][:(L + page - 1) // page], device=k.device)
        ks, vs = (c[take].view(len(take), kv, page, hd).transpose(0, 1).reshape(kv, -1, hd)[:, :L] for c in (k, v))
        q = turned(st["q"][at:at + n].double().reshape(n, heads, hd), list(range(L - n, L)))
        i, j = torch.arange(L - n, L, device=q.device)[:, None], torch.arange(L, device=q.device)
        hide = (j > i) | (j <= i - case["window"]) if case["window"] else j > i
        for h in range(heads):
            w = q[:, h] @ ks[h * kv // heads].T / hd ** 0.5
            w = torch.softmax(w.masked_fill(hide, float("-inf")), -1)
            out.append((s, h, w @ vs[h * kv // heads]))
        at += n
    o = torch.cat([torch.stack([y for t, _, y in out if t == s], 1) for s in sorted({t for t, _, _ in out})])
    if st["gate"] is not None:
        o = o * torch.sigmoid(st["gate"].double())[..., None]
    return o.reshape(st["ntok"], heads * hd)
