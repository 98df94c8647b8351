"""spk_logprobs against log-softmax in 64 bits.

Bounds. Sums of 2^t with t in f32 (|t| up to ~200: off by 2^-17 at most for what counts, |t| < 20: 2^-19)
and an exponential good to 2^-22: a log sum is off by about 1e-6, a log probability by that and the f32
rounding of (x - m) - log S: 2e-6 + 2^-22 |logp|. Entropy is a weighted mean of such terms: 4e-6 + 1e-6 H."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def ttype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def check(x, target, top, dev):
    import torch

    from spk import score

    rows, vocab = x.shape
    lp = score.LogProbs(rows, vocab, top, device=dev)
    d = x.double()
    want = torch.log_softmax(d, -1)
    p = want.exp()
    H = -(torch.where(p == 0, torch.zeros_like(p), p * want)).sum(-1)     # NaN where there is no distribution
    order = torch.sort(torch.where(d.isnan(), torch.full_like(d, float("-inf")), d), dim=-1, descending=True, stable=True)[1][:, :top]
    for _ in range(2):      # the workspace is left ready
        logp, ent, ids, best = lp(x, target)
        t = target.long().clamp(0, vocab - 1)
        w = torch.where(target < 0, torch.zeros(rows, dtype=torch.float64, device=dev), want.gather(1, t[:, None])[:, 0])
        for got, ref, lim in ((logp, w, 2e-6), (ent, H, 4e-6), (best, want.gather(1, order), 2e-6)):
            got = got.double()
            same = (got == ref) | (got.isnan() & ref.isnan())
            assert (same | ((got - ref).abs() <= lim + 1e-6 * ref.abs())).all(), (got - ref).abs().max()
        assert torch.equal(ids.long(), order)
    return logp


def rand(dev, rows, vocab, typ, seed=0, pad=0, shift=0, scale=3.0):
    import torch

    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    x = (torch.randn(rows, vocab + pad + shift, generator=g, device=dev) * scale).to(ttype(typ))
    t = torch.randint(0, vocab, (rows,), generator=g, device=dev).int()
    return x[:, shift:shift + vocab], t


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 7, 7), (3, 33, 32), (5, 1000, 5), (1, 131072, 20), (2, 4096, 0), (40, 50021, 3),
                                            (1, 131071, 32), (300, 9999, 8), (1500, 700, 2)])
def test_matches_log_softmax(cuda, rows, vocab, top, typ):
    x, t = rand(cuda, rows, vocab, typ, seed=rows + vocab)
    check(x, t, top, cuda)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift,pad", [(1, 0), (3, 2), (7, 8), (0, 1)])
def test_unaligned_rows(cuda, typ, shift, pad):
    for rows, vocab in ((1, 20001), (9, 4097), (200, 2050)):
        x, t = rand(cuda, rows, vocab, typ, seed=shift, pad=pad, shift=shift)
        check(x, t, 6, cuda)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_ties_go_to_the_lower_index(cuda, typ):
    import torch

    for rows, vocab in ((1, 50000), (700, 5000)):
        x, t = rand(cuda, rows, vocab, typ, seed=4)
        x = x.round().clamp(-3, 3)          # seven values
        check(x.contiguous(), t, 32, cuda)
        check(torch.zeros_like(x), t, 32, cuda)
        z = torch.zeros_like(x)
        z[:, ::2] = -0.0                    # no order between the zeros
        check(z, t, 32, cuda)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("order", ["up", "down"])
def test_sorted_rows(cuda, typ, order):
    """Every value beats (or none does) what came before it."""
    import torch

    x = torch.linspace(-20, 20, 30000, device=cuda).repeat(3, 1)
    x = (x if order == "up" else x.flip(1)).to(ttype(typ)).contiguous()
    check(x, torch.tensor([0, 29999, 77], dtype=torch.int32, device=cuda), 20, cuda)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_masked_tokens(cuda, typ):
    """-inf and the type's lowest value in places, in all places but one, in all."""
    import torch

    low = torch.finfo(ttype(typ)).min
    for mask in (float("-inf"), low):
        for rows, vocab in ((6, 9000), (1, 70000), (400, 300)):
            x, t = rand(cuda, rows, vocab, typ, seed=5)
            x = x.contiguous()
            x[:, vocab // 3:] = mask
            if rows > 3:
                x[1] = mask
                x[1, 17] = 2.0
                if mask == low:
                    x[2] = mask             # a distribution all the same: the uniform one
                x[3, :100] = mask
            check(x, t, 5, cuda)
    if typ == "f32":                         # references at the edge of f32
        for big in (3e38, -3e38):
            x, t = rand(cuda, 2, 5000, typ, seed=6)
            check((x + big).contiguous(), t, 4, cuda)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_rows_without_a_distribution(cuda, typ):
    import torch

    for rows, vocab in ((8, 3000), (8, 100000)):
        x, t = rand(cuda, rows, vocab, typ, seed=7)
        x = x.contiguous()
        x[1, 5] = float("nan")
        x[3] = float("-inf")
        x[4, vocab - 1] = float("inf")
        x[6, 0] = float("nan")
        x[6, 1:] = float("-inf")
        logp = check(x, t, 4, cuda)
        assert logp.isnan().tolist() == [False, True, False, True, True, False, True, False]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [900, 9000, 70000])
def test_alternatives_of_rows_with_many_nan(cuda, typ, vocab):
    """A NaN ranks as -inf, however many lie side by side; the order of the rest stays."""
    x, t = rand(cuda, 4, vocab, typ, seed=vocab)
    x[0, :vocab // 2] = float("nan")
    x[1, ::2] = float("nan")
    x[2, 40:] = float("nan")
    x[3] = float("nan")
    check(x, t, 20, cuda)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift", [0, 1, 3, 5])
@pytest.mark.parametrize("vocab,left", [(900, 0), (900, 3), (9000, 7), (70000, 2)])
def test_alternatives_of_rows_with_few_tokens_left(cuda, vocab, left, shift, typ):
    """Fewer tokens that can come than alternatives asked for, in rows of any alignment: the masked ones
    follow in their order, each once."""
    x, t = rand(cuda, 5, vocab, typ, seed=vocab + left, shift=shift, pad=3)
    x[:, :vocab - left] = float("-inf")
    check(x, t, 20, cuda)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("offset", [1e2, -1e3, 1e4, -1e4, 6e4, -6e4, 1e6, -1e9, 1e30, -1e30])
def test_logits_far_from_zero(cuda, offset, typ):
    """A constant added to a row changes nothing but the values' own rounding, and a row masked whole by any
    finite value is the uniform distribution: the bounds above hold as they are, since x - m is exact near the
    maximum."""
    import torch

    if not np.isfinite(float(torch.tensor(offset).to(ttype(typ)))):
        pytest.skip("past the type's range")
    for rows, vocab in ((1, 30000), (5, 4097), (900, 700)):
        x, t = rand(cuda, rows, vocab, "f32", seed=rows)
        x = (x.double() + offset).to(ttype(typ))
        x[0] = offset
        if rows > 1:
            x[1] = offset
            x[1, vocab // 2:] = 3.0         # masked by the offset (or the other way round)
        x = x.contiguous()
        assert x.isfinite().all()
        check(x, t, 6, cuda)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_rows_past_2_to_the_31(cuda, typ):
    """Rows whose elements lie past 2^31 of their matrix, and past 2^32 of its bytes."""
    import torch

    ld, rows, vocab = 2 ** 30 + 17, 3, 9001
    x = torch.empty(2 * ld + vocab, dtype=ttype(typ), device=cuda).as_strided((rows, vocab), (ld, 1))
    y, t = rand(cuda, rows, vocab, typ, seed=9)
    x.copy_(y)
    check(x, t, 5, cuda)


def test_targets(cuda):
    import torch

    import spk
    from spk import score

    x, t = rand(cuda, 5, 100, "f32")
    t[1], t[3] = -1, -7
    logp = check(x, t, 2, cuda)
    assert logp[1] == 0 and logp[3] == 0
    t[2] = 100
    lp = score.LogProbs(5, 100, 0, device=cuda)
    logp = lp(x, t)[0]
    assert logp[2].isnan() and not logp[0].isnan()
    assert spk.lib().spk_check_device_error() == -1 and spk.lib().spk_check_device_error() == 0


def test_a_workspace_serves_calls_of_fewer_rows(cuda):
    """One workspace of 128 rows, for 20, 128, 1 and 128 of them, each cut over several CTAs."""
    import torch

    import spk

    x, t = rand(cuda, 128, 60000, "f32", seed=8)
    x = x.contiguous()
    L = spk.lib()
    ws = torch.zeros(L.spk_logprobs_workspace_bytes(128, 60000), dtype=torch.uint8, device=cuda)
    want = torch.log_softmax(x.double(), -1)
    for rows in (20, 128, 1, 128):
        logp = torch.full((rows,), 7.0, device=cuda)
        ids, best = torch.full((rows, 2), -1, dtype=torch.int32, device=cuda), torch.zeros(rows, 2, device=cuda)
        spk.check(L.spk_logprobs(x.data_ptr(), 0, rows, 60000, 60000, t.data_ptr(), logp.data_ptr(), None, 2, ids.data_ptr(),
                                 best.data_ptr(), ws.data_ptr(), None))
        torch.cuda.synchronize()
        w = want[:rows].gather(1, t[:rows].long()[:, None])[:, 0]
        assert ((logp.double() - w).abs() <= 2e-6 + 1e-6 * w.abs()).all(), rows
        assert torch.equal(ids.long(), want[:rows].topk(2)[1]), rows


def test_optional_outputs_and_streams(cuda):
    import torch

    import spk

    x, t = rand(cuda, 3, 5000, "bf16")
    x = x.contiguous()
    L = spk.lib()
    ws = torch.zeros(L.spk_logprobs_workspace_bytes(3, 5000), dtype=torch.uint8, device=cuda)
    ent = torch.empty(3, device=cuda)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    spk.check(L.spk_logprobs(x.data_ptr(), 2, 3, 5000, 5000, None, None, ent.data_ptr(), 0, None, None, ws.data_ptr(), s.cuda_stream))
    s.synchronize()
    w = torch.log_softmax(x.double(), -1)
    assert np.allclose(ent.cpu(), -(w.exp() * w).sum(-1).cpu(), atol=1e-5)


def test_a_given_stream_is_ordered_with_the_objects_own_buffers(cuda):
    """A first call on another stream than the object's, which is still busy with its zeroing; logits dropped after
    the call; then a call that is captured."""
    import torch

    from spk import score

    x, t = rand(cuda, 3, 60000, "f32", seed=2)
    x = x.contiguous()
    want = torch.log_softmax(x.double(), -1).gather(1, t.long()[:, None])[:, 0]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    junk = torch.full((score.LogProbs(3, 60000, 2, device=cuda).workspace.numel(),), 255, dtype=torch.uint8, device=cuda)
    del junk
    torch.cuda._sleep(100_000_000)
    lp = score.LogProbs(3, 60000, 2, device=cuda)
    mine = x.clone()
    s.wait_stream(torch.cuda.current_stream())      # the logits are the caller's to order
    logp = lp(mine, t, stream=s)[0]
    del mine
    junk = torch.zeros_like(x)
    torch.cuda.synchronize()
    assert ((logp.double() - want).abs() < 2e-5).all()
    lp = score.LogProbs(3, 60000, 2, device=cuda)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lp(x, t)
    lp.logp.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert ((lp.logp.double() - want).abs() < 2e-5).all() and junk.sum() == 0
