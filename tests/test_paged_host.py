"""The paged cache's host side: what the entry points refuse (no device work is reached), the page
table's book-keeping, the layout's constants."""
import ctypes as C
import os

import pytest

import spk
from spk import paged, score

needs_lib = pytest.mark.skipif(not os.path.exists(spk.LIB_PATH), reason="libspk.so not built")
P = 1 << 20   # a non-null pointer that is never followed: every call below is refused first


def pool(**kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, pages=8, page_tokens=32, kv_heads=2, head_dim=128)
    d.update(kw)
    return paged._Pool(*[d[f] for f, _ in paged._Pool._fields_])


def batch(**kw):
    d = dict(nseq=2, rows=3, row0=P, kv_len=P, table=P, max_pages=4)
    d.update(kw)
    return paged._Batch(*[d[f] for f, _ in paged._Batch._fields_])


BAD_POOLS = [dict(k=None), dict(v_scale=None), dict(head_dim=96), dict(head_dim=0), dict(pages=0), dict(kv_heads=0),
             dict(page_tokens=8), dict(page_tokens=40), dict(k=P + 8), dict(k_scale=P + 2)]
BAD_BATCHES = [dict(nseq=0), dict(nseq=paged.MAX_SEQ + 1), dict(rows=-1), dict(max_pages=0), dict(row0=None),
               dict(kv_len=None), dict(table=None)]


@needs_lib
@pytest.mark.parametrize("bad", BAD_POOLS + BAD_BATCHES)
def test_bad_pools_and_batches_are_refused(bad):
    L = spk.lib()
    p = pool(**{k: v for k, v in bad.items() if k in dict(paged._Pool._fields_)})
    b = batch(**{k: v for k, v in bad.items() if k in dict(paged._Batch._fields_)})
    a = paged._Attn(q=P, ldq=512, type=0, heads=4, out=P, ldout=512, workspace=P)
    assert L.spk_paged_append(C.addressof(p), C.addressof(b), P, 256, P, 256, 0, None, 0, None) == -1
    assert "spk_paged_append" in spk.last_error()
    assert L.spk_paged_attn(C.addressof(p), C.addressof(b), C.addressof(a), None) == -1
    assert "spk_paged_attn" in spk.last_error()


@needs_lib
@pytest.mark.parametrize("kw", [dict(type=3), dict(type=-1), dict(pdim=12, freq=P), dict(pdim=256, freq=P), dict(pdim=-8, freq=P),
                                dict(pdim=64), dict(k=None), dict(v=None), dict(ldk=255), dict(ldv=100), dict(k=P + 2),
                                dict(v=P + 1, type=1)])
def test_append_refuses(kw):
    d = dict(k=P, ldk=256, v=P, ldv=256, type=0, freq=None, pdim=0)
    d.update(kw)
    p, b = pool(), batch()
    assert spk.lib().spk_paged_append(C.addressof(p), C.addressof(b), d["k"], d["ldk"], d["v"], d["ldv"], d["type"],
                                      d["freq"], d["pdim"], None) == -1
    assert spk.last_error()


@needs_lib
@pytest.mark.parametrize("kw", [dict(type=7), dict(heads=3), dict(heads=0), dict(pdim=4, freq=P), dict(pdim=64), dict(window=-1),
                                dict(q=None), dict(out=None), dict(workspace=None), dict(ldq=511), dict(ldout=10),
                                dict(gate=P, ldgate=3), dict(q=P + 2), dict(out=P + 1), dict(workspace=P + 8)])
def test_attention_refuses(kw):
    d = dict(q=P, ldq=512, type=0, heads=4, out=P, ldout=512, workspace=P)
    d.update(kw)
    p, b, a = pool(), batch(), paged._Attn(**d)
    assert spk.lib().spk_paged_attn(C.addressof(p), C.addressof(b), C.addressof(a), None) == -1
    assert spk.last_error()


@needs_lib
def test_unaligned_frequencies_are_refused():
    p, b = pool(), batch()
    a = paged._Attn(q=P, ldq=512, type=0, heads=4, out=P, ldout=512, workspace=P, freq=P + 2, pdim=64)
    assert spk.lib().spk_paged_append(C.addressof(p), C.addressof(b), P, 256, P, 256, 0, P + 1, 64, None) == -1
    assert spk.lib().spk_paged_attn(C.addressof(p), C.addressof(b), C.addressof(a), None) == -1


@needs_lib
def test_attention_refuses_a_batch_past_its_line_of_work():
    """Row tiles times blocks of the longest table has to fit 32 bits."""
    p = pool(pages=1 << 20, page_tokens=1024, kv_heads=64)
    b = batch(rows=1 << 20, max_pages=1 << 15)
    a = paged._Attn(q=P, ldq=64 * 128, type=1, heads=64, out=P, ldout=64 * 128, workspace=P)
    assert spk.lib().spk_paged_attn(C.addressof(p), C.addressof(b), C.addressof(a), None) == -1
    assert "too much" in spk.last_error()


@needs_lib
def test_attention_refuses_many_heads_past_the_line_of_work():
    """480000 row tiles of less than a token over a table of 80000 tokens: 2.4e9 blocks."""
    p = pool(pages=2000, page_tokens=64, kv_heads=1, head_dim=64)
    b = batch(nseq=1, rows=90000, max_pages=1250)
    a = paged._Attn(q=P, ldq=128 * 64, type=0, heads=128, out=P, ldout=128 * 64, workspace=P)
    assert spk.lib().spk_paged_attn(C.addressof(p), C.addressof(b), C.addressof(a), None) == -1
    assert "too much" in spk.last_error()


@needs_lib
def test_no_rows_is_a_call_that_does_nothing():
    p, b = pool(), batch(rows=0)
    a = paged._Attn(type=0, heads=4)
    assert spk.lib().spk_paged_append(C.addressof(p), C.addressof(b), None, 0, None, 0, 0, None, 0, None) == 0
    assert spk.lib().spk_paged_attn(C.addressof(p), C.addressof(b), C.addressof(a), None) == 0
    assert spk.lib().spk_logprobs(None, 0, 0, 10, 10, None, None, None, 0, None, None, None, None) == 0


@needs_lib
@pytest.mark.parametrize("kw", [dict(type=3), dict(rows=-1), dict(rows=70000), dict(vocab=0), dict(top=33), dict(top=-1),
                                dict(top=11), dict(logits=None), dict(workspace=None), dict(target=None), dict(ids=None),
                                dict(best=None), dict(logits=P + 2), dict(ld=9), dict(workspace=P + 4)])
def test_logprobs_refuses(kw):
    d = dict(logits=P, type=0, rows=2, vocab=10, ld=10, target=P, logp=P, entropy=P, top=4, ids=P, best=P, workspace=P)
    d.update(kw)
    assert spk.lib().spk_logprobs(*[d[k] for k in ("logits", "type", "rows", "vocab", "ld", "target", "logp", "entropy", "top",
                                                   "ids", "best", "workspace")], None) == -1
    assert spk.last_error()


@needs_lib
def test_workspace_sizes():
    L = spk.lib()
    assert L.spk_paged_attn_workspace_bytes(96) == 0
    assert L.spk_logprobs_workspace_bytes(0, 5) == 0
    assert L.spk_logprobs_workspace_bytes(3, 100) < L.spk_logprobs_workspace_bytes(300, 100)


@needs_lib
def test_logprobs_workspace_is_no_larger_than_its_parts():
    """Rows past the CTAs that run side by side are not split: a workspace does not grow with them."""
    size = spk.lib().spk_logprobs_workspace_bytes
    assert all(size(n, 131072) <= size(n + 1, 131072) for n in range(1, 2000))
    assert size(65535, 131072) == size(1000, 10) < 300000


def test_value_order_is_a_permutation_with_its_inverse():
    assert sorted(paged.ORDER) == list(range(paged.BLOCK))
    place = [4 * ((i & 7) >> 1) + (i & 1) + 2 * (i >> 3) for i in range(paged.BLOCK)]
    assert [paged.ORDER[place[i]] for i in range(paged.BLOCK)] == list(range(paged.BLOCK))


def test_page_table_hands_out_and_takes_back():
    t = paged.PageTable(5, 16)
    assert t.reserve("a", 17) == [0, 1]
    assert t.reserve("b", 1) == [2]
    assert t.reserve("a", 32) == [0, 1]
    assert t.reserve("a", 33) == [0, 1, 3]
    with pytest.raises(spk.SpkError):
        t.reserve("c", 33)
    rows = t.rows(["b", "a", "z"], device="cpu")
    assert rows.tolist() == [[2, -1, -1], [0, 1, 3], [-1, -1, -1]]
    t.release("a")
    t.release("nobody")
    assert t.reserve("c", 49) == [0, 1, 3, 4]


def test_page_table_after_a_refusal_and_a_trim():
    t = paged.PageTable(4, 16)
    t.reserve("a", 20)
    was = list(t.free), {s: list(p) for s, p in t.held.items()}
    with pytest.raises(spk.SpkError):
        t.reserve("b", 33)
    assert (t.free, t.held) == was       # not even an empty entry
    t.reserve("a", 50)
    t.trim("a", 2)
    t.trim("nobody", 0)
    assert t.held["a"] == [0, 1] and t.reserve("c", 16)
    t.trim("c", 0)
    assert "c" not in t.held


@pytest.mark.parametrize("kw", [dict(head_dim=80), dict(page_tokens=24), dict(pages=0), dict(kv_heads=0)])
def test_cache_refuses(kw):
    d = dict(pages=4, page_tokens=32, kv_heads=2, head_dim=64, device="cpu")
    d.update(kw)
    with pytest.raises(spk.SpkError):
        paged.PagedCache(**d)


def test_python_checks_of_rows():
    import torch

    c = paged.PagedCache(4, 32, 2, 64, device="cpu")
    with pytest.raises(spk.SpkError):
        paged.PagedBatch(c, torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32), 1, 2)
    with pytest.raises(spk.SpkError):
        paged._rows(torch.zeros(3, 4), 3, 5, "k")
    with pytest.raises(spk.SpkError):
        paged._rows(torch.zeros(4, 3).T, 3, 4, "k")
    with pytest.raises(spk.SpkError):
        paged._rows(torch.zeros(3, 4), 3, 4, "k")      # on the host
    with pytest.raises(spk.SpkError):
        paged.type_of(torch.zeros(1, dtype=torch.float64))
    with pytest.raises(spk.SpkError):
        score.LogProbs(3, 10, top=11, device="cpu")


def test_rows_of_another_device_than_the_pool_are_refused():
    """The pool's, the batch's and the rows' addresses go to one device, whichever tensor is looked at first."""
    from unittest import mock

    import torch

    def rows(device):
        t = mock.Mock(shape=(3, 128), dtype=torch.float32, is_cuda=True, device=torch.device(device))
        t.stride.return_value, t.get_device.return_value = (128, 1), t.device.index
        return t

    pool = torch.device("cuda:0")
    assert paged._rows(rows("cuda:0"), 3, 128, "k", on=pool) == 128
    with pytest.raises(spk.SpkError):
        paged._rows(rows("cuda:1"), 3, 128, "k", on=pool)
    b = mock.Mock(spec=paged.PagedBatch, cache=mock.Mock(kv_heads=2, head_dim=64, device=pool), rows=3, heads=2, _a=paged._Attn())
    with pytest.raises(spk.SpkError, match="pool"):
        paged.PagedBatch.append(b, rows("cuda:1"), rows("cuda:1"))
    with pytest.raises(spk.SpkError, match="pool"):
        paged.PagedBatch.attention(b, rows("cuda:1"), rows("cuda:1"))
