"""spk.serve.PagedScorer over the paged 4-bit cache against the CPU oracle's decoder.

Bound. The oracle's cache is f32; here keys and values are e2m1 under scales of 4 significant bits, off by 9.5 % of a value
(rms, of normal values in groups of 16), 3.7 times what the 8-bit cache's e4m3 is off by, so the bounds are 3.7 times those of its test: logits of a
4-layer model within 30 % (relative norm), a log probability within 1.1. The same rows through the 8-bit cache differ from these by
no more than both bounds."""
import numpy as np
import pytest

import oracle
from spk.model import small_config, synth_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(cuda):
    from spk.serve import PagedScorer

    cfg = small_config()
    W = synth_weights(cfg, seed=3, exact_q80=True)
    layers = [{"in_norm": L["in_norm"], "post_norm": L["post_norm"],
               **{n: oracle.decode(L[n]) for n in ("qkv", "attn_gate", "out", "gate", "up", "down")}} for L in W["layers"]]
    embed = oracle.q80_dequant(W["embed"], cfg.vocab, cfg.hidden)
    ref = oracle.Model(cfg.as_oracle(), layers, embed, W["norm"], 200)
    return cfg, ref, PagedScorer(cfg, W, pages=40, page_tokens=16, device=cuda, kv_bits=4)


def want(ref, ids):
    """Logits after every token of a sequence, by the oracle one token at a time."""
    return np.stack([ref.forward(t, p).copy() for p, t in enumerate(ids)])


def test_a_batch_of_sequences_is_near_the_oracle(model):
    cfg, ref, sc = model
    rng = np.random.default_rng(1)
    seqs = {"a": rng.integers(0, cfg.vocab, 150).tolist(), "b": [7], "c": rng.integers(0, cfg.vocab, 33).tolist(),
            "d": [], "e": rng.integers(0, cfg.vocab, 16).tolist()}
    logits = sc.forward(seqs).cpu().numpy().astype(np.float64)
    at = 0
    for s, ids in seqs.items():
        if not ids:
            continue
        w = want(ref, ids).astype(np.float64)
        g = logits[at:at + len(ids)]
        at += len(ids)
        assert np.linalg.norm(g - w) / np.linalg.norm(w) < 0.3, s
    for s in seqs:
        sc.release(s)


def test_calls_continue_and_scores_are_near(model):
    """A sequence fed in parts reads what the parts before left, token for token the same cache as in one call."""
    cfg, ref, sc = model
    rng = np.random.default_rng(2)
    seqs = {"a": rng.integers(0, cfg.vocab, 60).tolist(), "b": rng.integers(0, cfg.vocab, 21).tolist()}
    whole = sc.forward(seqs).cpu().numpy()
    whole = {"a": whole[:60], "b": whole[60:]}
    for s in seqs:
        sc.release(s)
    parts = {s: [] for s in seqs}
    for part in (slice(0, 1), slice(1, 18), slice(18, 19), slice(19, 60)):
        new = {s: ids[part] for s, ids in seqs.items()}
        got, at = sc.forward(new).cpu().numpy(), 0
        for s in seqs:
            parts[s].append(got[at:at + len(new[s])])
            at += len(new[s])
    for s in seqs:
        assert np.linalg.norm(np.concatenate(parts[s]) - whole[s]) / np.linalg.norm(whole[s]) < 0.02, s
        sc.release(s)
    for s, r in sc.feed(seqs, top=3).items():
        full = want(ref, seqs[s]).astype(np.float64)
        p = full - np.log(np.exp(full).sum(-1, keepdims=True))
        assert all(abs(x - p[i][seqs[s][i + 1]]) < 1.1 for i, x in enumerate(r.logp[:-1]))
        sc.release(s)


def test_what_it_refuses(model, cuda):
    import spk
    from spk.serve import PagedScorer

    cfg, _, sc = model
    with pytest.raises(spk.SpkError):
        PagedScorer(cfg, {}, pages=4, kv_bits=3)
    with pytest.raises(spk.SpkError):
        sc.forward({"x": [0] * 16 * 41})
    assert "x" not in sc.len and len(sc.table.free) == 40


def test_the_command(cuda, capsys, monkeypatch):
    import sys

    from spk import serve

    monkeypatch.setattr(sys, "argv", ["serve", "--layers", "2", "--sequences", "3", "--tokens", "40", "--kv-bits", "4"])
    serve.main()
    assert "perplexity" in capsys.readouterr().out
