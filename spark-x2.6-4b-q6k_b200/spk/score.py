"""What logits say about given tokens: spk_logprobs.

``LogProbs`` keeps the buffers of a row count, vocabulary and number of alternatives:

    lp = LogProbs(rows, vocab, top=5)
    logp, entropy, ids, best = lp(logits, target)

logp[i] = log softmax(logits[i])[target[i]], entropy[i] in nats, ids / best [rows][top] the most
likely tokens and their log probabilities, ties to the lower id. The buffers are the object's own
and are written again by its next call; calls may be on any stream, one after the other.
"""
from __future__ import annotations

from . import SpkError, check, lib
from .paged import Owned, _rows, lent, stream_of, type_of

MAX_TOP = 32
MAX_ROWS = 65535    # of a call


class LogProbs:
    def __init__(self, rows: int, vocab: int, top: int = 0, device="cuda"):
        import torch

        if not 0 <= rows <= MAX_ROWS or vocab < 1 or not 0 <= top <= min(MAX_TOP, vocab):
            raise SpkError(f"{rows} rows of {vocab} with {top} alternatives (0 to {MAX_TOP})")
        self.rows, self.vocab, self.top = rows, vocab, top
        self.logp = torch.empty(rows, device=device)
        self.entropy = torch.empty(rows, device=device)
        self.ids = torch.empty(rows, top, dtype=torch.int32, device=device)
        self.best = torch.empty(rows, top, device=device)
        L = lib()
        self.workspace = torch.zeros(L.spk_logprobs_workspace_bytes(rows, vocab), dtype=torch.uint8, device=device)
        self.owned = Owned(self.logp, self.entropy, self.ids, self.best, self.workspace)
        self._fn = L.spk_logprobs
        self._out = (self.logp.data_ptr(), self.entropy.data_ptr(), top, self.ids.data_ptr(), self.best.data_ptr(),
                     self.workspace.data_ptr())

    def __call__(self, logits, target, stream=None):
        """logits [rows][vocab] f32, f16 or bf16 (rows may lie apart), target int32 [rows] (negative:
        no token, logp 0). Returns the object's (logp, entropy, ids, best)."""
        import torch

        ld = _rows(logits, self.rows, self.vocab, "logits")
        if target.dtype != torch.int32 or target.numel() != self.rows or not target.is_contiguous():
            raise SpkError(f"target is int32 [{self.rows}]; got {target.dtype} {list(target.shape)}")
        if target.device != logits.device or self.logp.device != logits.device:
            raise SpkError("logits, target and the object's buffers lie on different devices")
        typ, raw = type_of(logits), stream_of(logits, stream)
        self.owned.use(raw, stream)
        check(self._fn(logits.data_ptr(), typ, self.rows, self.vocab, ld, target.data_ptr(), *self._out, raw))
        lent(stream, logits, target)
        return self.logp, self.entropy, self.ids, self.best
