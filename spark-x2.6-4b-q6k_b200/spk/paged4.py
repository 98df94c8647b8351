"""Batched serving over the paged 4-bit cache: spk_paged4_append, spk_paged4_attn and spk_paged4_read.

What spk.paged is for 8 bits, in 4.5 bits a value (the layout is include/spk.h's, spk_kv4_pool): codes of 4 bits under one
scale byte per 16 values of a head's row. ``Paged4Cache`` owns one layer's pool, ``Paged4Batch`` is the set of rows that a
call works on; ``spk.paged.PageTable`` hands out the pages of both kinds.

    cache = Paged4Cache(pages, 64, kv_heads, head_dim)
    batch = Paged4Batch(cache, row0, kv_len, table, rows=n, heads=heads)
    q = batch.append(k, v, freq=freq, q=q, q_norm=wq, k_norm=wk)   # norms, rotation, rounding: one pass
    batch.attention(q, out, gate=g)                                # q as append left it
    k, v = batch.read(dtype=torch.bfloat16)                        # the same rows as the cache has them

Queries are normalised and rotated once, beside the keys, where the 8-bit cache's attention rotates them itself.
Streams, ownership and lifetimes are spk.paged's.
"""
from __future__ import annotations

import ctypes as C
import struct

from . import SpkError, check, lib
from .paged import BLOCK, Owned, PagedBatch, _angles, _attend, _rows, lent, stream_of, type_of

GROUP = 16          # values that share a scale


class _Pool4(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("pages", C.c_int), ("page_tokens", C.c_int), ("kv_heads", C.c_int), ("head_dim", C.c_int)]


class _Append4(C.Structure):
    _fields_ = [("q", C.c_void_p), ("ldq", C.c_longlong), ("q_out", C.c_void_p), ("ldq_out", C.c_longlong),
                ("k", C.c_void_p), ("v", C.c_void_p), ("ldk", C.c_longlong), ("ldv", C.c_longlong),
                ("type", C.c_int), ("heads", C.c_int), ("q_norm", C.c_void_p), ("k_norm", C.c_void_p), ("eps", C.c_float),
                ("freq", C.c_void_p), ("pdim", C.c_int), ("interleaved", C.c_int)]


class _Read4(C.Structure):
    _fields_ = [("type", C.c_int), ("k", C.c_void_p), ("v", C.c_void_p), ("ldk", C.c_longlong), ("ldv", C.c_longlong),
                ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("ldk_scale", C.c_longlong), ("ldv_scale", C.c_longlong)]


class _Attn4(C.Structure):
    _fields_ = [("q", C.c_void_p), ("ldq", C.c_longlong), ("type", C.c_int), ("heads", C.c_int), ("window", C.c_int),
                ("scale", C.c_float), ("gate", C.c_void_p), ("ldgate", C.c_longlong), ("out", C.c_void_p),
                ("ldout", C.c_longlong), ("workspace", C.c_void_p)]


PARTS = 3           # spk_paged4_read's type: codes and scales apart

# The arguments' fields in one go: a step's calls take less time than setting them one by one.
_APPEND, _READ = struct.Struct("@PqPqPPqqiiPPfPii"), struct.Struct("@iPPqqPPqq")


def _stride(t, shape, like, what: str):
    """_rows() of a row matrix that has to be like `like` (type and device), without its words where all is well."""
    if t.shape == shape and t.dtype == like.dtype and t.get_device() == like.get_device() >= 0:
        ld, one = t.stride()
        if one == 1:
            return ld
    return _rows(t, *shape, what, like)


class Paged4Cache:
    """One layer's keys and values of every sequence. Needs no initial contents."""

    def __init__(self, pages: int, page_tokens: int, kv_heads: int, head_dim: int, device="cuda"):
        import torch

        if head_dim not in (64, 128, 256):
            raise SpkError(f"head_dim {head_dim} (64, 128 or 256)")
        if pages < 1 or kv_heads < 1 or page_tokens < BLOCK or page_tokens % BLOCK:
            raise SpkError(f"{pages} pages of {page_tokens} tokens (a multiple of {BLOCK}), {kv_heads} KV heads")
        self.pages, self.page_tokens, self.kv_heads, self.head_dim = pages, page_tokens, kv_heads, head_dim
        self.k_pool = torch.empty(pages, kv_heads, page_tokens, head_dim // 2, dtype=torch.uint8, device=device)
        self.v_pool = torch.empty_like(self.k_pool)
        self.k_scale = torch.empty(pages, kv_heads, page_tokens, head_dim // GROUP, dtype=torch.uint8, device=device)
        self.v_scale = torch.empty_like(self.k_scale)
        self.device = self.k_pool.device
        self.owned = Owned(self.k_pool, self.v_pool, self.k_scale, self.v_scale)
        self._c = _Pool4(self.k_pool.data_ptr(), self.v_pool.data_ptr(), self.k_scale.data_ptr(),
                         self.v_scale.data_ptr(), pages, page_tokens, kv_heads, head_dim)

    def values(self):
        """The keys and values that the pool stands for, f32 [pages][kv_heads][page_tokens][head_dim]
        (for inspection and tests; torch operations, a copy)."""
        import torch

        have = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device=self.device)
        have = torch.cat([have, -have])

        def wide(pool, scale):
            x = torch.stack([have[(pool & 15).int()], have[(pool >> 4).int()]], -1).flatten(-2)
            return x * (scale.to(torch.int16) << 7).view(torch.float16).float().repeat_interleave(GROUP, -1)

        return wide(self.k_pool, self.k_scale), wide(self.v_pool, self.v_scale)


class Paged4Batch(PagedBatch):
    """The rows of a call over a 4-bit pool: PagedBatch's arguments, checks and limits. `rows` may be more than row0[nseq] (a padded buffer,
    a captured graph): the rows behind it are left as they are."""

    _cache = Paged4Cache

    def _bind(self) -> None:
        import torch

        L = lib()
        with torch.cuda.device(self.cache.device):
            self.workspace = torch.zeros(L.spk_paged4_attn_workspace_bytes(self.cache.head_dim), dtype=torch.uint8,
                                         device=self.cache.device)
        self._a = _Attn4(heads=self.heads, workspace=self.workspace.data_ptr())
        self._append, self._attn, self._read = L.spk_paged4_append, L.spk_paged4_attn, L.spk_paged4_read
        self._ap, self._rd = (C.c_char * C.sizeof(_Append4))(), (C.c_char * C.sizeof(_Read4))()
        self._ap_p, self._rd_p = C.addressof(self._ap), C.addressof(self._rd)
        wide, self._f32 = self.cache.kv_heads * self.cache.head_dim, torch.float32
        self._parts = [(wide, torch.float8_e4m3fn), (wide // GROUP, torch.float16)] * 2
        self._kv_shape, self._q_shape = (torch.Size((self.rows, w)) for w in (wide, self.heads * self.cache.head_dim))
        self._sc_shape, self._e4m3, self._f16 = torch.Size((self.rows, wide // GROUP)), torch.float8_e4m3fn, torch.float16
        self._index = self.cache.device.index

    def append(self, k, v, freq=None, q=None, q_out=None, q_norm=None, k_norm=None, eps: float = 1e-6, interleaved: bool = False,
               stream=None):
        """Rows k, v [rows][kv_heads * head_dim] into the pages, and queries q [rows][heads * head_dim] to q_out (made when not
        given, returned; q itself for in place). q_norm, k_norm: f32 [head_dim], the weights of an RMS norm of each head.
        freq: the rotation of the first 2 * len(freq) dims, pairs half of that apart or, `interleaved`, side by side."""
        c = self.cache
        if k.get_device() != self._index:
            _rows(k, *self._kv_shape, "k", on=c.device)
        ldk, ldv = _stride(k, self._kv_shape, k, "k"), _stride(v, self._kv_shape, k, "v")
        at_q = at_out = ldq = ldo = heads = 0
        if q is not None:
            ldq = _stride(q, self._q_shape, k, "q")
            if q_out is None:
                import torch

                with torch.cuda.stream(stream):      # None: the current one
                    q_out = torch.empty(self._q_shape, dtype=q.dtype, device=q.device)
            ldo = _stride(q_out, self._q_shape, k, "q_out")
            at_q, at_out, heads = q.data_ptr(), q_out.data_ptr(), self.heads
        elif q_out is not None or q_norm is not None:
            raise SpkError("q_out and q_norm go with q")
        at_f, pdim = _angles(freq, k)
        _APPEND.pack_into(self._ap, 0, at_q, ldq, at_out, ldo, k.data_ptr(), v.data_ptr(), ldk, ldv, type_of(k), heads,
                          self._norm(q_norm, "q_norm"), self._norm(k_norm, "k_norm"), eps, at_f or 0, pdim, interleaved)
        raw = stream_of(k, stream)
        c.owned.use(raw, stream)
        check(self._append(self._pool_p, self._batch_p, self._ap_p, raw))
        if stream is not None:
            lent(stream, k, v, q, q_out, q_norm, k_norm, freq, *self._keep)
        return q_out

    def _norm(self, w, name: str):
        """The address of a norm's weights."""
        if w is None:
            return 0
        c = self.cache
        if w.dtype != self._f32 or w.shape != (c.head_dim,) or not w.is_contiguous() or w.device != c.device:
            raise SpkError(f"{name} is f32 [{c.head_dim}] on {c.device}; got {w.dtype} {list(w.shape)} on {w.device}")
        return w.data_ptr()

    def attention(self, q, out=None, window: int = 0, gate=None, scale: float = 0.0, stream=None):
        """out [rows][heads * head_dim] (made when not given): attention of the rows, which have been appended, over their
        sequences; q as append returns it, `gate` [rows][heads] goes through a sigmoid, `window` 0 sees every
        earlier token, `scale` 0 is 1 / sqrt(head_dim)."""
        return _attend(self, q, out, window, gate, scale, stream)

    def read(self, k=None, v=None, dtype=None, stream=None):
        """The rows' keys and values as the cache has them, (k, v) [rows][kv_heads * head_dim]: into k and v where given, else
        new rows of `dtype` (bf16 when not given)."""
        c = self.cache
        if k is None or v is None:
            import torch

            given = v if k is None else k
            if given is not None:
                dtype = given.dtype
            with torch.cuda.stream(stream):
                new = [torch.empty(self.rows, c.kv_heads * c.head_dim, dtype=dtype or torch.bfloat16, device=c.device) if t is None else t
                       for t in (k, v)]
            k, v = new
        if k.get_device() != self._index:
            _rows(k, *self._kv_shape, "k", on=c.device)
        _READ.pack_into(self._rd, 0, type_of(k), k.data_ptr(), v.data_ptr(), _stride(k, self._kv_shape, k, "k"), _stride(v, self._kv_shape, k, "v"), 0, 0, 0, 0)
        self._read_rows(stream, k, v)
        return k, v

    def parts(self, out=None, stream=None):
        """The rows as the cache has them, apart: [k codes, k scales, v codes, v scales], codes e4m3
        [rows][kv_heads * head_dim], scales f16 [rows][kv_heads * head_dim / 16]. out: four such tensors."""
        if out is None:
            import torch

            with torch.cuda.stream(stream):
                out = [torch.empty(self.rows, w, dtype=t, device=self.cache.device) for w, t in self._parts]
        k, ks, v, vs = out
        if k.dtype != self._e4m3 or ks.dtype != self._f16:
            raise SpkError(f"codes are {self._e4m3}, scales {self._f16}; got {k.dtype} and {ks.dtype}")
        if k.get_device() != self._index or ks.get_device() != self._index:
            _rows(k, *self._kv_shape, "k codes", on=self.cache.device)
            _rows(ks, *self._sc_shape, "k scales", on=self.cache.device)
        _READ.pack_into(self._rd, 0, PARTS, k.data_ptr(), v.data_ptr(), _stride(k, self._kv_shape, k, "k codes"), _stride(v, self._kv_shape, k, "v codes"),
                        ks.data_ptr(), vs.data_ptr(), _stride(ks, self._sc_shape, ks, "k scales"), _stride(vs, self._sc_shape, ks, "v scales"))
        self._read_rows(stream, *out)
        return out

    def _read_rows(self, stream, *out) -> None:
        raw = stream_of(out[0], stream)
        self.cache.owned.use(raw, stream)
        check(self._read(self._pool_p, self._batch_p, self._rd_p, raw))
        if stream is not None:
            lent(stream, *out, *self._keep)
