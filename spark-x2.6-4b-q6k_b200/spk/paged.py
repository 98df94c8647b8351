"""Batched serving over the paged 8-bit cache: spk_paged_append and spk_paged_attn.

``PagedCache`` owns one layer's pool (e4m3 bytes, one f32 scale per 16-token block and KV head;
the layout is include/spk.h's, spk_kv_pool). ``PagedBatch`` is the set of rows that a call works
on: which rows belong to which sequence, how long the sequences are and where their pages lie, as
device arrays that the kernels read, so a batch can be kept (and captured in a CUDA graph) while
their contents move. ``PageTable`` hands out pages.

    cache = PagedCache(pages, 64, kv_heads, head_dim)
    batch = PagedBatch(cache, row0, kv_len, table, rows=n, heads=heads)
    batch.append(k, v, freq=freq)                  # rows into the pages, keys rotated on the way
    batch.attention(q, out, freq=freq, gate=g)     # causal attention over them

Calls go to torch's current stream unless a stream is given, and do not synchronize. What an object
here makes for itself may be used on any stream. Tensors that are handed in are ordered with a given
stream by the caller, as between any two streams; they may be dropped after the call. Output that a
call makes belongs to the call's stream.
"""
from __future__ import annotations

import ctypes as C

from . import SpkError, check, lib, ptr

BLOCK = 16          # tokens that share a scale
MAX_SEQ = 1024
ORDER = [2 * (b // 4) + b % 2 + 8 * (b // 2 % 2) for b in range(BLOCK)]   # the tokens of a value block, as they lie


class _Pool(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("pages", C.c_int), ("page_tokens", C.c_int), ("kv_heads", C.c_int), ("head_dim", C.c_int)]


class _Batch(C.Structure):
    _fields_ = [("nseq", C.c_int), ("rows", C.c_int), ("row0", C.c_void_p), ("kv_len", C.c_void_p),
                ("table", C.c_void_p), ("max_pages", C.c_int)]


class _Attn(C.Structure):
    _fields_ = [("q", C.c_void_p), ("ldq", C.c_longlong), ("type", C.c_int), ("heads", C.c_int),
                ("freq", C.c_void_p), ("pdim", C.c_int), ("window", C.c_int), ("scale", C.c_float),
                ("gate", C.c_void_p), ("ldgate", C.c_longlong), ("out", C.c_void_p), ("ldout", C.c_longlong),
                ("workspace", C.c_void_p)]


_TYPES = None


def type_of(t) -> int:
    """0 f32, 1 f16, 2 bf16: the ABI's number of a tensor's type."""
    global _TYPES
    if _TYPES is None:
        import torch

        _TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    n = _TYPES.get(t.dtype)
    if n is None:
        raise SpkError(f"rows are f32, f16 or bf16; got {t.dtype}")
    return n


_cuda = None


def stream_of(t, stream) -> int:
    """The CUDA stream of a call on tensor t: the one given, else torch's current one. The library
    launches on the current device, which has to be the tensor's."""
    global _cuda
    if _cuda is None:
        import torch

        _cuda = (torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream)   # what torch.cuda's own calls wrap
    i = t.get_device()
    if _cuda[0]() != i:
        raise SpkError(f"the rows lie on cuda:{i}, the current device is cuda:{_cuda[0]()}")
    return stream.cuda_stream if stream is not None else _cuda[1](i)


class Owned:
    """Buffers that an object makes for itself, on the stream then current. A first call on another stream
    waits for what that one had before it, since the buffers' memory may be in use there until then or their
    zeroing on its way, and keeps them from being handed out again before the call is done with them. (A call that is
    being captured does neither: a capture begins when the device is idle, and the graph's owner keeps what it reads.)"""

    def __init__(self, *tensors):
        import torch

        self.tensors, self.seen, self.made = tensors, set(), None
        dev = tensors[0].device
        if dev.type == "cuda":
            with torch.cuda.device(dev):
                self.seen.add(torch.cuda.current_stream().cuda_stream)
                if not torch.cuda.is_current_stream_capturing():
                    self.made = torch.cuda.Event()
                    self.made.record()

    def use(self, raw: int, stream) -> None:
        """Before a launch on the stream `raw`, `stream` as it was given to the call."""
        if raw in self.seen:
            return
        import torch

        s = stream if stream is not None else torch.cuda.current_stream(self.tensors[0].device)
        with torch.cuda.stream(s):
            if torch.cuda.is_current_stream_capturing():
                return
        if self.made is not None:
            s.wait_event(self.made)
        for t in self.tensors:
            t.record_stream(s)
        self.seen.add(raw)


def lent(stream, *tensors) -> None:
    """Tensors handed in to a call on a stream of its own: not handed out again before it is done with them."""
    if stream is not None:
        for t in tensors:
            if t is not None:
                t.record_stream(stream)


def rope_freq(theta: float, pdim: int, device="cuda"):
    """1 / theta^(2i / pdim), the rotation's frequencies (model.rs:416-429), f32 on the device."""
    import numpy as np
    import torch

    i = np.arange(0, pdim, 2, dtype=np.float32)
    return torch.from_numpy((np.float32(1) / np.power(np.float32(theta), i / np.float32(pdim))).astype(np.float32)).to(device)


def _rows(t, rows: int, width: int, what: str, like=None, on=None):
    """A row matrix [rows][width] whose last axis is dense: its row stride in elements. `like`: rows of the same type
    and device; `on`: the device that it has to lie on."""
    if t.shape != (rows, width):
        raise SpkError(f"{what} is [{rows}, {width}]; got {list(t.shape)}")
    ld, one = t.stride()
    if one != 1 and width > 1:
        raise SpkError(f"{what}: the values of a row lie {one} apart")
    if not t.is_cuda:
        raise SpkError("libspk takes device buffers; got a host tensor")
    if like is not None and (t.dtype != like.dtype or t.get_device() != like.get_device()):
        raise SpkError(f"{what} is {t.dtype} on {t.device}, the other rows {like.dtype} on {like.device}")
    if on is not None and t.device != on:
        raise SpkError(f"{what} lies on {t.device}, the pool on {on}")
    return ld


def _angles(freq, t):
    """(address, rotated dims) of the frequencies for the rows t: the kernels read f32 values side by side."""
    if freq is None:
        return None, 0
    import torch

    if freq.dtype != torch.float32 or not freq.is_contiguous():
        raise SpkError(f"freq is f32, its values side by side; got {freq.dtype} with strides {freq.stride()}")
    if freq.get_device() != t.get_device():
        raise SpkError(f"freq lies on {freq.device}, the rows on {t.device}")
    return ptr(freq), 2 * freq.numel()


class PagedCache:
    """One layer's keys and values of every sequence. Needs no initial contents."""

    def __init__(self, pages: int, page_tokens: int, kv_heads: int, head_dim: int, device="cuda"):
        import torch

        if head_dim not in (64, 128, 256):
            raise SpkError(f"head_dim {head_dim} (64, 128 or 256)")
        if pages < 1 or kv_heads < 1 or page_tokens < BLOCK or page_tokens % BLOCK:
            raise SpkError(f"{pages} pages of {page_tokens} tokens (a multiple of {BLOCK}), {kv_heads} KV heads")
        self.pages, self.page_tokens, self.kv_heads, self.head_dim = pages, page_tokens, kv_heads, head_dim
        f8 = torch.float8_e4m3fn
        self.k_pool = torch.empty(pages, kv_heads, page_tokens // 8, head_dim // 16, 8, 16, dtype=f8, device=device)
        self.v_pool = torch.empty(pages, kv_heads, page_tokens // BLOCK, head_dim, BLOCK, dtype=f8, device=device)
        self.k_scale = torch.empty(pages, kv_heads, page_tokens // BLOCK, device=device)
        self.v_scale = torch.empty_like(self.k_scale)
        self.device = self.k_pool.device
        self.owned = Owned(self.k_pool, self.v_pool, self.k_scale, self.v_scale)
        self._c = _Pool(self.k_pool.data_ptr(), self.v_pool.data_ptr(), self.k_scale.data_ptr(),
                        self.v_scale.data_ptr(), pages, page_tokens, kv_heads, head_dim)

    def values(self):
        """The keys and values that the pool stands for, f32 [pages][kv_heads][page_tokens][head_dim]
        (for inspection and tests; torch operations, a copy)."""
        import torch

        P, H, T, D = self.pages, self.kv_heads, self.page_tokens, self.head_dim
        inv = torch.tensor([ORDER.index(i) for i in range(BLOCK)], device=self.device)
        k = self.k_pool.float().transpose(3, 4).reshape(P, H, T // BLOCK, BLOCK, D)
        v = self.v_pool.float()[..., inv].transpose(3, 4)
        return ((k * self.k_scale[..., None, None]).reshape(P, H, T, D),
                (v * self.v_scale[..., None, None]).reshape(P, H, T, D))


class PageTable:
    """Which pages the sequences of a pool hold (host). Pages are handed out lowest first."""

    def __init__(self, pages: int, page_tokens: int):
        self.page_tokens = page_tokens
        self.free = list(range(pages))[::-1]
        self.held: dict = {}

    def reserve(self, seq, tokens: int) -> list:
        """The pages of sequence `seq` for `tokens` tokens, more of them when it needs more."""
        need = -(-tokens // self.page_tokens) - len(self.held.get(seq, ()))
        if need > len(self.free):
            raise SpkError(f"sequence {seq} needs {need} more pages, {len(self.free)} are free")
        have = self.held.setdefault(seq, [])
        for _ in range(need):
            have.append(self.free.pop())
        return have

    def trim(self, seq, pages: int) -> None:
        """Gives back the pages of `seq` past the first `pages`, the last one first."""
        have = self.held.get(seq, [])
        while len(have) > pages:
            self.free.append(have.pop())
        if not have:
            self.held.pop(seq, None)

    def release(self, seq) -> None:
        self.free += self.held.pop(seq, [])[::-1]

    def rows(self, seqs, device="cuda"):
        """int32 [len(seqs)][most pages] for PagedBatch, -1 where a sequence has fewer."""
        import torch

        width = max([1] + [len(self.held.get(s, [])) for s in seqs])
        return torch.tensor([self.held.get(s, []) + [-1] * (width - len(self.held.get(s, []))) for s in seqs],
                            dtype=torch.int32, device=device)


class PagedBatch:
    """The rows of a call over a pool. row0 int32 [nseq + 1], kv_len int32 [nseq] (the call's rows
    counted), table int32 [nseq][max_pages], on the pool's device; `rows` = row0[nseq]. Holds the
    attention's workspace: calls of one batch must not overlap on the GPU."""

    def __init__(self, cache: PagedCache, row0, kv_len, table, rows: int, heads: int):
        import torch

        nseq = kv_len.numel()
        for t, n, what in ((row0, nseq + 1, "row0"), (kv_len, nseq, "kv_len"), (table, None, "table")):
            if t.dtype != torch.int32 or not t.is_contiguous() or t.device != cache.device or (n and t.numel() != n):
                raise SpkError(f"{what}: {t.dtype} {list(t.shape)} on {t.device}")
        if table.dim() != 2 or table.shape[0] != nseq or not 1 <= nseq <= MAX_SEQ:
            raise SpkError(f"a table of {list(table.shape)} for {nseq} sequences (1 to {MAX_SEQ})")
        if heads < 1 or heads % cache.kv_heads:
            raise SpkError(f"{heads} heads over {cache.kv_heads} KV heads")
        self.cache, self.rows, self.heads = cache, rows, heads
        self._keep = (row0, kv_len, table)
        self._b = _Batch(nseq, rows, row0.data_ptr(), kv_len.data_ptr(), table.data_ptr(), table.shape[1])
        L = lib()
        with torch.cuda.device(cache.device):
            self.workspace = torch.zeros(L.spk_paged_attn_workspace_bytes(cache.head_dim), dtype=torch.uint8,
                                         device=cache.device)
        self.owned = Owned(self.workspace)
        self._a = _Attn(heads=heads, workspace=self.workspace.data_ptr())
        self._pool_p, self._batch_p, self._attn_p = C.addressof(cache._c), C.addressof(self._b), C.addressof(self._a)
        self._append, self._attn = L.spk_paged_append, L.spk_paged_attn

    def use(self, cache: PagedCache) -> None:
        """Turns the batch to another layer's pool of the same geometry (the page table is the layers' own)."""
        c = self.cache
        if (cache.pages, cache.page_tokens, cache.kv_heads, cache.head_dim, cache.device) != (
                c.pages, c.page_tokens, c.kv_heads, c.head_dim, c.device):
            raise SpkError("a pool of another geometry")
        self.cache, self._pool_p = cache, C.addressof(cache._c)

    def append(self, k, v, freq=None, stream=None) -> None:
        """Rows k, v [rows][kv_heads * head_dim] (views of a wider matrix are fine) into the pages;
        keys are rotated over their first 2 * len(freq) dims when freq is given."""
        width = self.cache.kv_heads * self.cache.head_dim
        ldk, ldv = _rows(k, self.rows, width, "k", on=self.cache.device), _rows(v, self.rows, width, "v", k)
        f, pdim = _angles(freq, k)
        typ, raw = type_of(k), stream_of(k, stream)
        self.cache.owned.use(raw, stream)
        check(self._append(self._pool_p, self._batch_p, k.data_ptr(), ldk, v.data_ptr(), ldv, typ, f, pdim, raw))
        lent(stream, k, v, freq, *self._keep)

    def attention(self, q, out=None, window: int = 0, freq=None, gate=None, scale: float = 0.0, stream=None):
        """out [rows][heads * head_dim] (made when not given): attention of the rows, which have been
        appended, over their sequences; q is rotated when freq is given, `gate` [rows][heads] goes
        through a sigmoid, `window` 0 sees every earlier token, `scale` 0 is 1 / sqrt(head_dim)."""
        width = self.heads * self.cache.head_dim
        a = self._a
        a.ldq = _rows(q, self.rows, width, "q", on=self.cache.device)
        if out is None:
            import torch

            with torch.cuda.stream(stream):      # None: the current one
                out = torch.empty(self.rows, width, dtype=q.dtype, device=q.device)
        a.ldout = _rows(out, self.rows, width, "out", q)
        a.q, a.out, a.type, a.window, a.scale = q.data_ptr(), out.data_ptr(), type_of(q), window, scale
        a.gate = None
        if gate is not None:
            a.ldgate = _rows(gate, self.rows, self.heads, "gate", q)
            a.gate = gate.data_ptr()
        a.freq, a.pdim = _angles(freq, q)
        raw = stream_of(q, stream)
        self.cache.owned.use(raw, stream)
        self.owned.use(raw, stream)
        check(self._attn(self._pool_p, self._batch_p, self._attn_p, raw))
        lent(stream, q, out, gate, freq, *self._keep)
        return out
