"""The 4-bit cache's host side: what the entry points refuse (no device work is reached), its layout's sizes."""
import ctypes as C
import os

import pytest

import spk
from spk import paged, paged4

needs_lib = pytest.mark.skipif(not os.path.exists(spk.LIB_PATH), reason="libspk.so not built")
P = 1 << 20   # a non-null pointer that is never followed: every call below is refused first


def fill(struct, d, kw):
    return struct(**{**d, **kw})


def pool(**kw):
    return fill(paged4._Pool4, dict(k=P, v=P, k_scale=P, v_scale=P, pages=8, page_tokens=32, kv_heads=2, head_dim=128), kw)


def batch(**kw):
    return fill(paged._Batch, dict(nseq=2, rows=3, row0=P, kv_len=P, table=P, max_pages=4), kw)


def append_args(**kw):
    return fill(paged4._Append4, dict(q=P, ldq=512, q_out=P, ldq_out=512, k=P, v=P, ldk=256, ldv=256, type=0, heads=4, eps=1e-6), kw)


def read_args(**kw):
    return fill(paged4._Read4, dict(type=0, k=P, v=P, ldk=256, ldv=256, k_scale=P, v_scale=P, ldk_scale=16, ldv_scale=16), kw)


def attn_args(**kw):
    return fill(paged4._Attn4, dict(q=P, ldq=512, type=0, heads=4, out=P, ldout=512, workspace=P), kw)


def call(name, p, b, a):
    return getattr(spk.lib(), name)(p and C.addressof(p), b and C.addressof(b), a and C.addressof(a), None)


ALL = [("spk_paged4_append", append_args), ("spk_paged4_read", read_args), ("spk_paged4_attn", attn_args)]


@needs_lib
@pytest.mark.parametrize("name,args", ALL)
@pytest.mark.parametrize("bad", [dict(k=None), dict(v_scale=None), dict(head_dim=96), dict(head_dim=0), dict(pages=0), dict(kv_heads=0),
                                 dict(page_tokens=8), dict(page_tokens=40), dict(v=P + 8), dict(k_scale=P + 4)])
def test_bad_pools_are_refused(name, args, bad):
    assert call(name, pool(**bad), batch(), args()) == -1
    assert name in spk.last_error()


@needs_lib
@pytest.mark.parametrize("name,args", ALL)
@pytest.mark.parametrize("bad", [dict(nseq=0), dict(nseq=paged.MAX_SEQ + 1), dict(rows=-1), dict(max_pages=0), dict(row0=None),
                                 dict(kv_len=None), dict(table=None)])
def test_bad_batches_are_refused(name, args, bad):
    assert call(name, pool(), batch(**bad), args()) == -1
    assert name in spk.last_error()


@needs_lib
@pytest.mark.parametrize("name,args", ALL)
def test_null_structs_are_refused(name, args):
    for p, b, a in ((None, batch(), args()), (pool(), None, args()), (pool(), batch(), None)):
        assert call(name, p, b, a) == -1


@needs_lib
@pytest.mark.parametrize("kw", [dict(type=3), dict(type=-1), dict(heads=-1), dict(heads=70000, ldq=1 << 24, ldq_out=1 << 24), dict(pdim=8, freq=P),
                                dict(pdim=144, freq=P), dict(pdim=-16, freq=P), dict(pdim=64), dict(pdim=64, freq=P + 2), dict(q_norm=P + 4),
                                dict(k_norm=P + 8), dict(k_norm=P, eps=-1.0), dict(q_norm=P, eps=float("nan")), dict(k=None), dict(v=None),
                                dict(q=None), dict(q_out=None), dict(ldk=255), dict(ldv=0), dict(ldq=511), dict(ldq_out=100), dict(k=P + 2),
                                dict(q=P + 1, type=1), dict(q_out=P + 1, type=2)])
def test_append_refuses(kw):
    assert call("spk_paged4_append", pool(), batch(), append_args(**kw)) == -1
    assert "spk_paged4_append" in spk.last_error()


@needs_lib
@pytest.mark.parametrize("kw", [dict(type=4), dict(type=-1), dict(k=None, v=None), dict(ldk=255), dict(ldv=-256), dict(k=P + 2), dict(v=P + 1, type=1),
                                dict(type=3, k_scale=None), dict(type=3, v_scale=P + 1), dict(type=3, ldk_scale=15), dict(type=3, ldk=10)])
def test_read_refuses(kw):
    assert call("spk_paged4_read", pool(), batch(), read_args(**kw)) == -1
    assert "spk_paged4_read" in spk.last_error()


@needs_lib
@pytest.mark.parametrize("kw", [dict(type=7), dict(heads=3), dict(heads=0), dict(window=-1), dict(q=None), dict(out=None), dict(workspace=None),
                                dict(ldq=511), dict(ldout=10), dict(gate=P, ldgate=3), dict(q=P + 2), dict(out=P + 1), dict(gate=P + 2, ldgate=4),
                                dict(workspace=P + 8)])
def test_attention_refuses(kw):
    assert call("spk_paged4_attn", pool(), batch(), attn_args(**kw)) == -1
    assert "spk_paged4_attn" in spk.last_error()


@needs_lib
def test_attention_refuses_a_batch_past_its_line_of_work():
    """Row tiles times blocks of the longest table has to fit 32 bits."""
    p = pool(pages=1 << 20, page_tokens=1024, kv_heads=64)
    b = batch(rows=1 << 20, max_pages=1 << 15)
    assert call("spk_paged4_attn", p, b, attn_args(type=1, heads=64, ldq=64 * 128, ldout=64 * 128)) == -1
    assert "too much" in spk.last_error()


@needs_lib
def test_attention_refuses_many_sequences_past_the_line_of_work():
    """1024 sequences of few rows over tables of 2^22 tokens, 64 KV heads: 1024 x 2^18 blocks x 64."""
    p = pool(pages=1 << 20, page_tokens=1024, kv_heads=64)
    b = batch(nseq=1024, rows=1024, max_pages=1 << 12)
    assert call("spk_paged4_attn", p, b, attn_args(type=1, heads=64, ldq=64 * 128, ldout=64 * 128)) == -1
    assert "too much" in spk.last_error()


@needs_lib
def test_no_rows_is_a_call_that_does_nothing():
    b = batch(rows=0)
    assert call("spk_paged4_append", pool(), b, paged4._Append4()) == 0
    assert call("spk_paged4_read", pool(), b, paged4._Read4()) == 0
    assert call("spk_paged4_attn", pool(), b, paged4._Attn4(heads=4)) == 0


@needs_lib
def test_workspace_sizes():
    L = spk.lib()
    assert L.spk_paged4_attn_workspace_bytes(96) == 0


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(pages=0), dict(page_tokens=24), dict(kv_heads=0)])
def test_caches_that_are_refused(kw):
    with pytest.raises(spk.SpkError):
        paged4.Paged4Cache(**{**dict(pages=4, page_tokens=16, kv_heads=2, head_dim=64, device="cpu"), **kw})


def test_a_value_takes_four_and_a_half_bits():
    c = paged4.Paged4Cache(3, 32, 2, 128, device="cpu")
    assert 8 * sum(t.numel() for t in (c.k_pool, c.v_pool, c.k_scale, c.v_scale)) == 4.5 * 2 * 3 * 32 * 2 * 128


def test_values_of_every_code_and_scale():
    import torch

    c = paged4.Paged4Cache(1, 16, 1, 64, device="cpu")
    c.k_pool.copy_(torch.arange(512).to(torch.uint8).reshape(1, 1, 16, 32))
    c.v_pool.fill_(0xf7)
    c.k_scale.fill_(120)                  # 1.0
    c.v_scale.copy_(torch.arange(8, 72).to(torch.uint8).reshape(1, 1, 16, 4))
    k, v = c.values()
    have = [0, .5, 1, 1.5, 2, 3, 4, 6]
    have += [-x for x in have]
    assert k.flatten().tolist() == [have[x] for b in range(512) for x in (b & 15, b >> 4 & 15)]
    d = [(1 + (b & 7) / 8) * 2.0 ** ((b >> 3) - 15) for b in range(8, 72)]
    assert v.flatten().tolist() == [s * x for s in d for _ in range(8) for x in (6.0, -6.0)]
