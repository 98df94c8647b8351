"""Scoring a batch of sequences over a paged cache in 8 or 4 bits: the decoder of spk.model for many
sequences at once, where DeviceModel runs one.

``PagedScorer`` holds the same weights (the VQ projections re-laid for the tensor-core GEMM, the tied
Q8_0 head in its tile layout) and, per layer, a ``PagedCache`` that all sequences share. ``feed`` takes
new tokens of any of them, in one call: every layer appends the rows' keys and values to the sequences'
pages with the rotation on the way (spk_paged_append), attends over the pages (spk_paged_attn, the gate
in its epilogue), and the head's logits end in each token's log probability, the entropy and the most
likely alternatives (spk_logprobs). With ``kv_bits=4`` the cache is a ``Paged4Cache`` (4.5 bits a value for 8.06, so nearly
twice the tokens in the same memory): one spk_paged4_append rotates queries and keys and rounds keys and values, and
spk_paged4_attn attends. A sequence may be continued by later calls, and dropped with
``release``. A call that raises leaves the sequences as they were, as long and on the same pages.

    python -m spk.serve [--layers N] [--sequences N] [--tokens N] [--kv-bits 8|4]    # synthetic weights
"""
from __future__ import annotations

import ctypes as C
from contextlib import contextmanager
from dataclasses import dataclass

import numpy as np

from . import SpkError, check, dev_bytes, lib
from .model import MATS, ModelConfig, mat_shapes, upload_container
from .paged import MAX_SEQ, PagedBatch, PagedCache, PageTable, rope_freq
from .paged4 import Paged4Batch, Paged4Cache
from .score import MAX_ROWS, MAX_TOP, LogProbs

GEMM_ROWS = 128     # rows of one spk_vq_lut_gemm call
HEAD_ROWS = 8       # rows of one spk_q80_tile_head call


@dataclass
class Scored:
    """What one call says about a sequence's new tokens: logp[i] of token i + 1 after token i (the last
    token's is None), and per token the entropy (nats) and alternatives of what follows it."""

    logp: list
    entropy: list
    alternatives: list      # per token: [(id, logp), ...], most likely first


class _Matrix:
    """A VQ matrix re-laid for the batched GEMM (spk_vq_lut_pack)."""

    def __init__(self, buf: bytes, device):
        import torch

        L = lib()
        M, keep = upload_container(buf, device)
        n = L.spk_vq_lut_bytes(M.dim, M.nc, M.rows, M.cols, M.v3)
        if not n:
            raise SpkError(f"a {M.rows} x {M.cols} matrix of {M.nc} codes is not one the batched GEMM takes")
        self.geometry = (M.dim, M.nc, M.rows, M.cols, M.v3)
        self.rows, self.cols = M.rows, M.cols
        self.words = [torch.zeros(n, dtype=torch.uint8, device=device) for _ in range(M.nstages)]
        for s, w in enumerate(self.words):
            check(L.spk_vq_lut_pack(M.stages[s], *self.geometry, w.data_ptr(), None))
        torch.cuda.synchronize(device)      # the payload may go now
        self.ptrs = (C.c_void_p * M.nstages)(*[w.data_ptr() for w in self.words])
        self.scratch = torch.zeros(L.spk_vq_lut_gemm_scratch_bytes(M.rows, M.cols, GEMM_ROWS), dtype=torch.uint8, device=device)

    def __call__(self, x, out, norm=None, eps: float = 0.0, accumulate: bool = False):
        """out (=, +=) W RMSNorm?(x) for the rows of x (f32)."""
        import torch

        L, s = lib(), torch.cuda.current_stream(x.device).cuda_stream
        for r in range(0, x.shape[0], GEMM_ROWS):
            n = min(GEMM_ROWS, x.shape[0] - r)
            check(L.spk_vq_lut_gemm(self.ptrs, len(self.words), *self.geometry, n, x[r].data_ptr(), x.stride(0),
                                    None if norm is None else norm.data_ptr(), eps, out[r].data_ptr(), out.stride(0),
                                    int(accumulate), self.scratch.data_ptr(), s))
        return out


class PagedScorer:
    def __init__(self, cfg: ModelConfig, weights: dict, pages: int, page_tokens: int = 64, device="cuda:0", kv_bits: int = 8):
        import torch

        if kv_bits not in (8, 4):
            raise SpkError(f"a cache of {kv_bits} bits (8 or 4)")
        self.kv_bits = kv_bits
        self.cfg, self.device = cfg, torch.device(device)
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(self.device)  # noqa: E731
        shapes = mat_shapes(cfg)
        self.layers = []
        for Lw in weights["layers"]:
            mats = {n: _Matrix(Lw[n], self.device) for n in MATS}
            for n in MATS:
                if (mats[n].rows, mats[n].cols) != shapes[n]:
                    raise SpkError(f"{n} is {mats[n].rows} x {mats[n].cols}, the configuration says {shapes[n]}")
            self.layers.append((mats, put(Lw["in_norm"]), put(Lw["post_norm"])))
        self.norm = put(weights["norm"])
        L = lib()
        row = cfg.hidden // 32 * 34
        self.embed = dev_bytes(weights["embed"], self.device)
        self._embed_rows = self.embed[:cfg.vocab * row].view(cfg.vocab, row)
        n = L.spk_q80_tile_bytes(cfg.vocab, cfg.hidden)
        if not n:
            raise SpkError(f"a {cfg.vocab} x {cfg.hidden} head has no tile layout")
        self.head = torch.zeros(n, dtype=torch.uint8, device=self.device)
        check(L.spk_q80_tile(self.embed.data_ptr(), cfg.vocab, cfg.hidden, self.head.data_ptr(), None))
        self.head_scratch = torch.zeros(L.spk_q80_tile_scratch_bytes(), dtype=torch.uint8, device=self.device)
        dims = lambda part: int(cfg.head_dim * part)  # noqa: E731
        self.freq = {1: rope_freq(cfg.rope_theta_full, dims(cfg.rope_partial_full), self.device),
                     0: rope_freq(cfg.rope_theta_slide, dims(cfg.rope_partial_slide), self.device)}
        cache = PagedCache if kv_bits == 8 else Paged4Cache
        self.caches = [cache(pages, page_tokens, cfg.kv_heads, cfg.head_dim, self.device) for _ in range(cfg.layers)]
        self.table = PageTable(pages, page_tokens)
        self.len: dict = {}
        torch.cuda.synchronize(self.device)

    def release(self, seq) -> None:
        """Forgets a sequence; its pages serve others."""
        self.table.release(seq)
        self.len.pop(seq, None)

    def _check(self, new: dict, rows_most=None, top: int = 0) -> list:
        """The sequences of a call that have tokens; raises where the call cannot be done. Changes nothing."""
        cfg, seqs = self.cfg, [s for s in new if len(new[s])]
        if not 0 <= top <= min(MAX_TOP, cfg.vocab):
            raise SpkError(f"{top} alternatives (0 to {min(MAX_TOP, cfg.vocab)})")
        if len(seqs) > MAX_SEQ:
            raise SpkError(f"{len(seqs)} sequences in a call (up to {MAX_SEQ})")
        rows = sum(len(new[s]) for s in seqs)
        if rows_most is not None and rows > rows_most:
            raise SpkError(f"{rows} tokens in a call (up to {rows_most})")
        for s in seqs:
            if not all(0 <= t < cfg.vocab for t in new[s]):
                raise SpkError(f"sequence {s}: a token id outside the vocabulary of {cfg.vocab}")
        return seqs

    @contextmanager
    def _kept(self, seqs):
        """The sequences' lengths and pages as they were, if what follows raises. Rows that it appended are written
        over by the next call; a block that holds earlier tokens, too, may keep a larger scale from them."""
        was = {s: (self.len.get(s), len(self.table.held.get(s, ()))) for s in seqs}
        try:
            yield
        except BaseException:
            for s in reversed(seqs):
                n, pages = was[s]
                self.table.trim(s, pages)
                if n is None:
                    self.len.pop(s, None)
                else:
                    self.len[s] = n
            raise

    def forward(self, new: dict):
        """Rows of new tokens {sequence: [ids]} through the decoder: logits [rows][vocab] (f32), the
        sequences in the order given. Their keys and values stay in the cache."""
        seqs = self._check(new)
        with self._kept(seqs):
            return self._forward(new, seqs)

    def _forward(self, new: dict, seqs: list):
        import torch

        cfg, dev = self.cfg, self.device
        rows = sum(len(new[s]) for s in seqs)
        if not rows:
            return torch.empty(0, cfg.vocab, device=dev)
        for s in seqs:
            self.table.reserve(s, self.len.get(s, 0) + len(new[s]))
        for s in seqs:
            self.len[s] = self.len.get(s, 0) + len(new[s])
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        row0 = i32(np.concatenate([[0], np.cumsum([len(new[s]) for s in seqs])]).tolist())
        kv_len, table = i32([self.len[s] for s in seqs]), self.table.rows(seqs, dev)
        L, st = lib(), torch.cuda.current_stream(dev).cuda_stream
        ids = torch.tensor([t for s in seqs for t in new[s]], device=dev)
        h = torch.empty(rows, cfg.hidden, device=dev)
        picked = self._embed_rows[ids].contiguous()
        check(L.spk_q80_dequant(picked.data_ptr(), rows * cfg.hidden // 32, h.data_ptr(), st))
        new_ = lambda width: torch.empty(rows, width, device=dev)  # noqa: E731
        qkv, gate, att = new_(cfg.q_dim + 2 * cfg.kv_dim), new_(cfg.heads), new_(cfg.q_dim)
        ga, up, logits = new_(cfg.inter), new_(cfg.inter), new_(cfg.vocab)
        batch = (PagedBatch if self.kv_bits == 8 else Paged4Batch)(self.caches[0], row0, kv_len, table, rows=rows, heads=cfg.heads)
        for (m, in_norm, post_norm), cache, full in zip(self.layers, self.caches, cfg.full):
            batch.use(cache)
            freq = self.freq[int(bool(full))]
            m["qkv"](h, qkv, in_norm, cfg.eps)
            m["attn_gate"](h, gate, in_norm, cfg.eps)
            q, k, v = qkv[:, :cfg.q_dim], qkv[:, cfg.q_dim:cfg.q_dim + cfg.kv_dim], qkv[:, cfg.q_dim + cfg.kv_dim:]
            window = 0 if full else cfg.window
            if self.kv_bits == 8:
                batch.append(k, v, freq=freq)
                batch.attention(q, att, window=window, freq=freq, gate=gate)
            else:
                batch.append(k, v, freq=freq, q=q, q_out=q)
                batch.attention(q, att, window=window, gate=gate)
            m["out"](att, h, accumulate=True)
            m["gate"](h, ga, post_norm, cfg.eps)
            m["up"](h, up, post_norm, cfg.eps)
            m["down"](torch.nn.functional.gelu(ga).mul_(up), h, accumulate=True)     # erf form, model.rs:253-258
        for r in range(0, rows, HEAD_ROWS):
            n = min(HEAD_ROWS, rows - r)
            check(L.spk_q80_tile_head(self.head.data_ptr(), cfg.vocab, cfg.hidden, n, h[r].data_ptr(), h.stride(0),
                                      self.norm.data_ptr(), cfg.eps, logits[r].data_ptr(), logits.stride(0), None,
                                      self.head_scratch.data_ptr(), st))
        return logits

    def feed(self, new: dict, top: int = 0) -> dict:
        """Scores new tokens {sequence: [ids]}: {sequence: Scored}. Synchronizes. The first token of a sequence's
        later part is not scored: its distribution was the last row of the part before."""
        import torch

        seqs = self._check(new, MAX_ROWS, top)
        target = torch.tensor([t for s in seqs for t in list(new[s][1:]) + [-1]], dtype=torch.int32, device=self.device)
        lp = LogProbs(len(target), self.cfg.vocab, top, device=self.device)
        with self._kept(seqs):
            logits = self._forward(new, seqs)
            logp, ent, ids, best = [t.tolist() for t in lp(logits, target)] if len(target) else ([], [], [], [])
            check(lib().spk_check_device_error(), "feed")
        out, r = {s: Scored([], [], []) for s in new}, 0
        for s in seqs:
            n = len(new[s])
            out[s] = Scored(logp[r:r + n - 1] + [None], ent[r:r + n], [list(zip(a, b)) for a, b in zip(ids[r:r + n], best[r:r + n])])
            r += n
        return out


def main() -> None:
    import argparse
    import math
    import time

    import torch

    from .model import small_config, synth_weights

    ap = argparse.ArgumentParser(description="Scores random sequences with a synthetic model over the paged cache.")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--sequences", type=int, default=12)
    ap.add_argument("--tokens", type=int, default=200, help="of the longest sequence")
    ap.add_argument("--kv-bits", type=int, default=8, choices=(8, 4), help="of the cache")
    a = ap.parse_args()
    cfg = small_config(layers=a.layers)
    rng = np.random.default_rng(0)
    seqs = {i: rng.integers(0, cfg.vocab, max(2, a.tokens * (i + 1) // a.sequences)).tolist() for i in range(a.sequences)}
    scorer = PagedScorer(cfg, synth_weights(cfg, seed=1, exact_q80=True), pages=sum(len(t) // 32 + 1 for t in seqs.values()), page_tokens=32, kv_bits=a.kv_bits)
    scorer.feed(seqs)
    for s in seqs:
        scorer.release(s)
    torch.cuda.synchronize()
    t = time.perf_counter()
    got = scorer.feed(seqs, top=3)
    t = time.perf_counter() - t
    for s, r in got.items():
        nll = [-x for x in r.logp if x is not None]
        print(f"sequence {s}: {len(seqs[s])} tokens, perplexity {math.exp(sum(nll) / len(nll)):.1f}, next "
              + ", ".join(f"{i} ({p:.2f})" for i, p in r.alternatives[-1]))
    n = sum(len(x) for x in seqs.values())
    print(f"{n} tokens in {1e3 * t:.1f} ms")


if __name__ == "__main__":
    main()
