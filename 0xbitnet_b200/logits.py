"""Rules on the logits before a token is picked (host mirror over libobn's C ABI).

The reference samples one row (packages/rust/crates/oxbitnet/src/sampling.rs:4-77:
repetition penalty, temperature, top-k, draw). A server steers many rows at once: each has a
history with penalties of its own, biases on some ids and a grammar's mask. One call applies
them to all rows where the LM head left the logits, and gives each row's greedy token.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import LogitRulesStruct
from .attention import _call


class LogitRules:
    """The rules of a batch of rows; every part is optional, and each is a CUDA tensor that
    the caller may rewrite in place between calls (a captured graph reads it anew).

    repetition, frequency, presence: f32 [rows]. history: int32 [rows, cap] (or [cap], shared)
    with history_lens int32 [rows]: once for each occurrence of an id a positive logit is
    divided and another one multiplied by repetition, and frequency is subtracted; presence
    is subtracted once. bias_ids int32 and bias_values f32 [rows, cap] (or [cap]) with
    bias_lens: added; the same id twice adds both. mask: int32 [rows, ceil(vocab / 32)] (or
    one row for all): bit v % 32 of word v // 32 set = token v allowed. Ids outside the
    vocabulary are ignored (pad with -1)."""

    def __init__(self, repetition=None, frequency=None, presence=None, history=None,
                 history_lens=None, bias_ids=None, bias_values=None, bias_lens=None, mask=None):
        self._kept = []     # the tensors whose addresses the struct holds
        self.index = None   # their device
        self.rows = None    # what the per-row tensors agree on
        self.mask_words = 0
        s = self._struct = LogitRulesStruct()
        self._address = ctypes.addressof(s)
        for name, t in (("repetition", repetition), ("frequency", frequency),
                        ("presence", presence)):
            setattr(s, name, self._vector(t, name, torch.float32))
        s.history, s.history_ld, s.history_cap = self._list(history, "history", torch.int32)
        s.history_lens = self._vector(history_lens, "history_lens", torch.int32)
        if (bias_ids is None) != (bias_values is None):
            raise ValueError("bias_ids and bias_values go together")
        if bias_ids is not None and bias_values.shape != bias_ids.shape:
            raise ValueError("bias_ids and bias_values must have one shape")
        s.bias_ids, s.bias_ld, s.bias_cap = self._list(bias_ids, "bias_ids", torch.int32)
        s.bias_values = self._list(bias_values, "bias_values", torch.float32)[0]
        s.bias_lens = self._vector(bias_lens, "bias_lens", torch.int32)
        s.mask, s.mask_ld, self.mask_words = self._list(mask, "mask", torch.int32)
        if mask is not None and not self.mask_words:
            raise ValueError("mask holds no words")

    def _take(self, t, name, dtype):
        if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dtype
                and t.is_contiguous()):
            raise TypeError(f"{name} must be a contiguous {dtype} CUDA tensor")
        if self.index is None:
            self.index = t.get_device()
        elif t.get_device() != self.index:
            raise ValueError(f"{name} is on {t.device}, other rules on cuda:{self.index}")
        self._kept.append(t)

    def _agree(self, rows, name):
        if self.rows is not None and rows != self.rows:
            raise ValueError(f"{name} has {rows} rows, other rules {self.rows}")
        self.rows = rows

    def _vector(self, t, name, dtype):
        if t is None:
            return None
        self._take(t, name, dtype)
        self._agree(t.numel(), name)
        return t.data_ptr()

    def _list(self, t, name, dtype):
        """(address, ld, cap) of a list for each row, or of one for all rows."""
        if t is None:
            return None, 0, 0
        self._take(t, name, dtype)
        if t.dim() not in (1, 2):
            raise ValueError(f"{name} must be [rows, cap] or [cap]")
        if t.dim() == 1 or t.shape[0] == 1:
            return t.data_ptr(), 0, t.shape[-1]
        self._agree(t.shape[0], name)
        return t.data_ptr(), t.shape[1], t.shape[1]


def logits_process(logits: torch.Tensor, rules: LogitRules, out: torch.Tensor | None = None,
                   token: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """logits [rows, vocab] f32 -> (the logits under the rules, each row's greedy token int32
    [rows], -1 where nothing is allowed). out may be logits itself."""
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dim() == 2
            and logits.dtype == torch.float32 and logits.is_contiguous()):
        raise TypeError("logits must be a contiguous torch.float32 CUDA tensor [rows, vocab]")
    rows, vocab = logits.shape
    index = logits.get_device()
    if rules.index is not None and rules.index != index:
        raise ValueError(f"logits are on {logits.device}, the rules on cuda:{rules.index}")
    if rules.rows is not None and rules.rows != rows:
        raise ValueError(f"the rules are for {rules.rows} rows, the logits have {rows}")
    if rules.mask_words and rules.mask_words < -(-vocab // 32):
        raise ValueError(f"the mask has {rules.mask_words} words a row, {vocab} ids need "
                         f"{-(-vocab // 32)}")
    if out is None:
        out = torch.empty_like(logits)
    elif not (out.shape == logits.shape and out.dtype is torch.float32 and out.is_contiguous()
              and out.is_cuda and out.get_device() == index):
        raise TypeError("out must be like logits")
    if token is None:
        token = torch.empty(rows, dtype=torch.int32, device=logits.device)
    elif not (token.numel() == rows and token.dtype is torch.int32 and token.is_contiguous()
              and token.is_cuda and token.get_device() == index):
        raise TypeError("token must be a contiguous int32 tensor [rows] beside the logits")
    _call("obn_logits_process", index, logits.data_ptr(), rows, vocab, rules._address,
          out.data_ptr(), token.data_ptr())
    return out, token
