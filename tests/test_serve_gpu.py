"""spk.serve.PagedScorer (the decoder over the paged 8-bit cache) against the CPU oracle's decoder.

Bound. The oracle's cache is f32; here keys and values are e4m3, off by 2.6 % of a value (rms). A layer's
attention output is off by about that, and it is one of two terms a layer adds to the residual, so the
logits of a 4-layer model stay within 8 % (relative norm); a log probability within the difference that
makes to logits of unit spread, 0.3."""
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
    return cfg, ref, PagedScorer(cfg, W, pages=40, page_tokens=16, device=cuda)


def want(ref, ids):
    """Logits after every token of a sequence, by the oracle one token at a time."""
    return np.stack([ref.forward(t, p).copy() for p, t in enumerate(ids)])


def test_a_batch_of_sequences_matches_the_oracle(model):
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
        assert np.linalg.norm(g - w) / np.linalg.norm(w) < 0.08, s
    for s in seqs:
        sc.release(s)


def test_scores_are_the_log_probabilities_and_calls_continue(model):
    cfg, ref, sc = model
    rng = np.random.default_rng(2)
    seqs = {"a": rng.integers(0, cfg.vocab, 60).tolist(), "b": rng.integers(0, cfg.vocab, 21).tolist()}
    full = {s: want(ref, ids) for s, ids in seqs.items()}
    got = {s: [] for s in seqs}
    for part in (slice(0, 1), slice(1, 18), slice(18, 19), slice(19, 60)):     # a token, a run, a token, the rest
        for s, r in sc.feed({s: ids[part] for s, ids in seqs.items()}, top=4).items():
            got[s].append(r)
    for s, ids in seqs.items():
        lse = np.log(np.exp(full[s].astype(np.float64)).sum(-1))
        ent = [e for r in got[s] for e in r.entropy]
        alts = [x for r in got[s] for x in r.alternatives]
        logp = [x for r in got[s] for x in r.logp]
        assert len(ent) == len(alts) == len(logp) == len(ids)
        for i in range(len(ids)):
            p = full[s][i].astype(np.float64) - lse[i]
            assert abs(ent[i] + (np.exp(p) * p).sum()) < 0.3
            assert [a[1] for a in alts[i]] == sorted((a[1] for a in alts[i]), reverse=True)
            assert all(abs(v - p[t]) < 0.3 for t, v in alts[i])
            if logp[i] is not None:
                assert abs(logp[i] - p[ids[i + 1]]) < 0.3
        assert sum(x is None for x in logp) == sum(bool(r.logp) for r in got[s])
    for s in seqs:
        sc.release(s)


def test_what_it_refuses(model):
    import spk

    cfg, _, sc = model
    with pytest.raises(spk.SpkError):
        sc.feed({"x": [cfg.vocab]})
    with pytest.raises(spk.SpkError):
        sc.feed({"x": [1] * 641})        # 41 pages of 16, 40 there
    sc.release("x")
    assert sc.feed({}) == {}


def test_a_call_that_fails_leaves_the_sequences_as_they_were(model):
    """Refused before anything is appended, or failed under way (no memory, a wait that ran out): the same tokens fed
    afterwards are scored as by a scorer that never saw the failure. Scores are compared as they are: a block's scale
    is that of its rows, and the tokens that come again are the same."""
    from unittest import mock

    import spk
    from spk import serve

    cfg, _, sc = model
    rng = np.random.default_rng(4)
    a, b = rng.integers(0, cfg.vocab, 50).tolist(), rng.integers(0, cfg.vocab, 20).tolist()
    parts = [{"a": a[:20]}, {"a": a[20:], "b": b}]
    fresh = [sc.feed(p, top=3) for p in parts]
    for s in "ab":
        sc.release(s)

    def state():
        return dict(sc.len), {s: list(p) for s, p in sc.table.held.items()}, list(sc.table.free)

    def refuses(new, **kw):
        was = state()
        with pytest.raises((spk.SpkError, MemoryError)):
            sc.feed(new, **kw)
        assert state() == was

    got = []
    for p in parts:
        refuses(p, top=33)
        refuses(p, top=-1)
        refuses({**p, "x": [cfg.vocab]})
        refuses({**p, "x": [1] * 640})                           # pages for some of them
        refuses({**p, **{i: [1] for i in range(1024)}})          # more sequences than a call takes
        refuses({**p, "x": [1] * 65536})                         # more rows than log probabilities are of
        for what in ("PagedBatch.attention", "LogProbs.__call__"):
            with mock.patch.object(getattr(serve, what.split(".")[0]), what.split(".")[1], side_effect=MemoryError):
                refuses(p, top=3)
        with mock.patch.object(serve, "lib", lambda: mock.Mock(wraps=spk.lib(), spk_check_device_error=lambda: -1)):
            refuses(p, top=3)
        got.append(sc.feed(p, top=3))
    assert got == fresh
    for s in "ab":
        sc.release(s)


def test_it_runs_as_a_command(cuda, capsys):
    import sys
    from unittest import mock

    from spk import serve

    with mock.patch.object(sys, "argv", ["serve", "--layers", "4", "--sequences", "3", "--tokens", "40"]):
        serve.main()
    out = capsys.readouterr().out
    assert out.count("perplexity") == 3 and "tokens in" in out
