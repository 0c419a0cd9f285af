"""Decoding rules on logits: penalties for tokens already emitted, biases (hotwords) and masks of allowed tokens (grammars).

The reference's searches take the argmax of the raw logits (src/rnnt/model.py:152-153,
src/rnnt/beam_searcher.py:91-93).  :class:`LogitRules` changes what they choose from:
``rnnt_amd.row_argmax(x, rules)`` and ``row_max_logp(x, rules)`` apply the rules on the way to the maximum, in one pass
over the logits; :func:`process_logits` writes the changed logits for a caller that samples or searches itself;
``greedy_decode`` and ``greedy_search_batch`` take ``rules=`` and keep the history.  Entry points ``rnnt_row_rules`` and
``rnnt_process_logits`` (include/rnnt_mi355.h) through the compiled binding.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, List, Optional, Union

import torch

from . import _torch_binding

_MAX_HISTORY = 65535   # the kernels' counters have 16 bits


def pack_allowed(mask: torch.Tensor) -> torch.Tensor:
    """Bool ``[..., V]`` -> int32 ``[..., (V + 31) // 32]``: token ``v`` in bit ``v % 32`` of word ``v // 32``."""
    if mask.dtype is not torch.bool or mask.dim() < 1 or mask.shape[-1] < 1:
        raise ValueError("mask must be a torch.bool tensor [..., V]")
    words = (mask.shape[-1] + 31) // 32
    bits = torch.zeros(*mask.shape[:-1], words * 32, dtype=torch.int64, device=mask.device)
    bits[..., :mask.shape[-1]] = mask
    word = (bits.view(*mask.shape[:-1], words, 32) << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)


@dataclass
class LogitRules:
    """What is done to a row of logits ``x`` before the maximum is taken, in this order, in fp32:

    ``c`` = how often a token stands in the row's history; where ``c > 0``: ``x / repetition_penalty`` if ``x > 0`` else
    ``x * repetition_penalty``; ``- frequency_penalty * c``; ``- presence_penalty`` where ``c > 0``; ``+ bias``; ``-inf``
    where not allowed, whatever ``x`` holds there.

    Attributes:
        bias: fp32 ``[V]`` (all rows) or ``[contexts, V]``.
        allowed: int32 words of one bit per token (:func:`pack_allowed`), ``[words]`` or ``[contexts, words]``.  For
            ``greedy_decode`` / ``greedy_search_batch`` also a callable: tokens emitted so far -> ``[words]``.  A row whose
            mask allows nothing gives token 0 with a NaN score.
        history: int32 ``[contexts, n]`` tokens (at most 65535), of which the first ``history_lens[c]`` (int32
            ``[contexts]``, clamped to ``[0, n]``; None: all) count; tokens outside ``[0, V)`` are ignored.

    Rows belong to contexts in order, ``rows / contexts`` each: the frames of one utterance's window share its context.
    """

    bias: Optional[torch.Tensor] = None
    allowed: Union[torch.Tensor, Callable[[List[int]], torch.Tensor], None] = None
    history: Optional[torch.Tensor] = None
    history_lens: Optional[torch.Tensor] = None
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0

    def _args(self):
        if callable(self.allowed):
            raise TypeError("a callable `allowed` is for greedy_decode and greedy_search_batch; pass its words here")
        return (self.bias, self.allowed, self.history, self.history_lens, float(self.repetition_penalty),
                float(self.presence_penalty), float(self.frequency_penalty))


def _check(rules) -> LogitRules:
    if not isinstance(rules, LogitRules):
        raise TypeError("rules must be a rnnt_amd.LogitRules")
    return rules


def process_logits(x: torch.Tensor, rules: LogitRules, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x[R, V]`` under ``rules``, computed in fp32 and rounded once to ``x``'s type (fp32, bf16 or fp16).  ``out`` may be
    ``x`` itself.  No backward: what requires grad (``out`` too) is refused in grad mode."""
    return _torch_binding.load().process_logits(x, *_check(rules)._args(), out)


class HistoryRules:
    """``rules`` as a greedy search uses them: the history of every utterance grows with what it emits.  It is kept, counted and
    limited to 65535 tokens only where a penalty may look at it (neutral penalties change no logit, whatever was emitted) or a history
    is given."""

    def __init__(self, rules: LogitRules, batch: int, vocab: int, most: int, device):
        self.rules, self.device = _check(rules), device
        self.tokens: List[List[int]] = [[] for _ in range(batch)]
        words = (vocab + 31) // 32

        def rows(t, width, name):
            if t is None:
                return None
            if t.dim() not in (1, 2) or t.shape[-1] != width or (t.dim() == 2 and t.shape[0] != batch):
                raise ValueError(f"rules.{name} must be [{width}] or [{batch}, {width}], got {list(t.shape)}")
            return t.to(device)

        self.bias = rows(rules.bias, vocab, "bias")
        self.grammar = rules.allowed if callable(rules.allowed) else None
        if self.grammar is None:
            self.allowed = rows(rules.allowed, words, "allowed")
        else:
            self.allowed = torch.empty(batch, words, dtype=torch.int32, device=device)
            for b in range(batch):
                self._ask(b)
        before = 0 if rules.history is None else rules.history.shape[-1]
        if rules.history is not None and (rules.history.dim() != 2 or rules.history.shape[0] != batch):
            raise ValueError(f"rules.history must be [{batch}, n]")
        if rules.history_lens is not None and (rules.history is None or rules.history_lens.shape != (batch,)):
            raise ValueError(f"rules.history_lens must be [{batch}], beside a history")
        for name in ("history", "history_lens"):
            if getattr(rules, name) is not None and getattr(rules, name).dtype is not torch.int32:
                raise TypeError(f"rules.{name} must be torch.int32")
        if rules.history is not None and before + most > _MAX_HISTORY:
            raise ValueError("the history (with one token per frame) is longer than 65535 tokens")
        self.before = before
        self.history = None
        if rules.history is None and (rules.repetition_penalty, rules.presence_penalty, rules.frequency_penalty) == (1, 0, 0):
            return
        # -1: no token.  (room for as many emissions as can be counted: `most` frames may be more, and emit far less)
        self.history = torch.full((batch, min(before + most, _MAX_HISTORY)), -1, dtype=torch.int32, device=device)
        if before:
            self.history[:, :before] = rules.history
            if rules.history_lens is not None:
                late = torch.arange(before, device=device) >= rules.history_lens.to(device)[:, None]
                self.history[:, :before].masked_fill_(late, -1)

    def _ask(self, b: int) -> None:
        words = self.grammar(list(self.tokens[b]))
        if words.dtype is not torch.int32 or words.shape != self.allowed.shape[1:]:
            raise ValueError(f"rules.allowed(tokens) must return int32 [{self.allowed.shape[1]}]")
        self.allowed[b] = words.to(self.allowed.device)

    def emit(self, utterances: List[int], tokens: List[int]) -> None:
        if self.history is not None:
            where = [self.before + len(self.tokens[b]) for b in utterances]
            if max(where) >= _MAX_HISTORY:
                raise ValueError("the history is longer than 65535 tokens: its counts have 16 bits")
            device = self.history.device
            self.history[torch.tensor(utterances, device=device), torch.tensor(where, device=device)] = torch.tensor(
                tokens, dtype=torch.int32, device=device)
        for b, t in zip(utterances, tokens):
            self.tokens[b].append(t)
            if self.grammar is not None:
                self._ask(b)

    def of(self, utterances: List[int]) -> LogitRules:
        """The rules of these utterances' rows."""
        r = self.rules
        longest = self.before + max(len(self.tokens[b]) for b in utterances)
        every = len(utterances) == len(self.tokens)
        sel = None if every else torch.tensor(utterances, device=self.device)

        def pick(t):
            return t if t is None or t.dim() == 1 or every else t.index_select(0, sel)

        return LogitRules(pick(self.bias), pick(self.allowed), None if self.history is None else pick(self.history)[:, :longest],
                          None, r.repetition_penalty,
                          r.presence_penalty, r.frequency_penalty)
