"""Rules of requests on their next token's logits (logit_rules.hip): penalties for
repeated tokens, biases and sets of allowed tokens.

:class:`LogitRules` holds them by request slot; :func:`adjust_logits` applies them to a
step's logits, :func:`append_tokens` records what was sampled.  Both stay on the device, so
that a decode step with rules can be captured and replayed.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import numpy as np
import torch

import polyrl_amd.ops as _ops
from . import ref

MOST_TOKENS = (1 << 19) - 1      # of a history
MOST_BIASES = (1 << 12) - 1      # of a slot
MOST_ROWS = 1 << 14              # whose tokens are recorded at a time (one block does)


def token_words(tokens, vocab: int) -> np.ndarray:
    """Token ids as the bits of ceil(vocab / 32) int32 words."""
    try:
        ids = np.asarray(list(tokens), dtype=np.int64)
    except OverflowError:
        raise ValueError("token ids outside of the vocabulary") from None
    if ids.size and (ids.min() < 0 or ids.max() >= vocab):
        raise ValueError("token ids outside of the vocabulary")
    bits = np.zeros((vocab + 31) // 32 * 32, dtype=np.uint8)
    bits[ids] = 1
    return np.packbits(bits, bitorder="little").view(np.int32)


def in_32_bits(v: float) -> float:
    """v as the kernels see it: what fp32 does not hold is infinite or 0."""
    try:
        with np.errstate(over="ignore", under="ignore"):
            return float(np.float32(v))
    except OverflowError:                # a whole number beyond all floats
        return math.inf if v > 0 else -math.inf


class LogitRules:
    """Rules of ``slots`` requests over a vocabulary: tensors by slot, which a program
    may also write itself.

    history (slots, capacity) int32   prompt, then output tokens
    prompt_len, total_len (slots)     int32: how many are the prompt's, how many in all
    repetition, frequency, presence   (slots) fp32
    bias_tokens, bias_values          (slots, biases) int32 (-1: none) and fp32; of a token
                                      named twice the last entry holds
    mask (slots, ceil(vocab/32))      int32, bit v % 32 of word v // 32: v is allowed
    masked (slots) int32              0: the slot's mask does not count
    """

    def __init__(self, slots: int, vocab: int, capacity: int, device,
                 biases: int = 0):
        if slots < 1 or vocab < 1 or not 0 <= capacity <= MOST_TOKENS \
                or not 0 <= biases <= MOST_BIASES:
            raise ValueError(
                f"LogitRules: a slot and a token at least, at most {MOST_TOKENS} "
                f"tokens of history and {MOST_BIASES} biases")
        i32 = dict(dtype=torch.int32, device=device)
        f32 = dict(dtype=torch.float32, device=device)
        self.slots, self.vocab, self.capacity = slots, vocab, capacity
        self.history = torch.full((slots, capacity), -1, **i32)
        self.prompt_len = torch.zeros(slots, **i32)
        self.total_len = torch.zeros(slots, **i32)
        self.repetition = torch.ones(slots, **f32)
        self.frequency = torch.zeros(slots, **f32)
        self.presence = torch.zeros(slots, **f32)
        self.bias_tokens = torch.full((slots, biases), -1, **i32)
        self.bias_values = torch.zeros(slots, biases, **f32)
        self.mask = torch.zeros(slots, (vocab + 31) // 32, **i32)
        self.masked = torch.zeros(slots, **i32)

    @property
    def biases(self) -> int:
        return self.bias_tokens.shape[1]

    def set(self, slot: int, prompt: Sequence[int] = (),
            output: Sequence[int] = (), repetition: float = 1.0,
            frequency: float = 0.0, presence: float = 0.0, bias=(),
            allowed=None):
        """A slot's rules and history anew.  ``bias``: (token, value) pairs or a dict;
        ``allowed``: token ids, or int32 words as of :func:`token_words`; None for all."""
        self._check(slot)
        for name, v in (("repetition", repetition), ("frequency", frequency),
                        ("presence", presence)):
            v = in_32_bits(v)
            if not math.isfinite(v) or name == "repetition" and v <= 0:
                raise ValueError(f"LogitRules: {name} {v}")
        words = np.asarray([*prompt, *output], dtype=np.int32)
        if len(words) > self.capacity:
            raise ValueError(f"LogitRules: {len(words)} tokens in a history "
                             f"of {self.capacity}")
        pairs = list(bias.items()) if isinstance(bias, dict) else list(bias)
        if len(pairs) > self.biases:
            raise ValueError(f"LogitRules: {len(pairs)} biases in {self.biases}")
        for t, v in pairs:
            if not 0 <= int(t) < self.vocab or math.isnan(in_32_bits(v)):
                raise ValueError(f"LogitRules: bias {v} of token {t}")
        self.allow(slot, allowed)
        if len(words):
            self.history[slot, :len(words)] = torch.from_numpy(words).to(
                self.history.device)
        self.prompt_len[slot] = len(prompt)
        self.total_len[slot] = len(words)
        self.repetition[slot] = in_32_bits(repetition)
        self.frequency[slot] = in_32_bits(frequency)
        self.presence[slot] = in_32_bits(presence)
        if self.biases:
            tokens = np.full(self.biases, -1, np.int32)
            values = np.zeros(self.biases, np.float32)
            for i, (t, v) in enumerate(pairs):
                tokens[i], values[i] = int(t), in_32_bits(v)
            dev = self.history.device
            self.bias_tokens[slot] = torch.from_numpy(tokens).to(dev)
            self.bias_values[slot] = torch.from_numpy(values).to(dev)

    def allow(self, slot: int, allowed=None):
        """The tokens that a slot's next one may be (as of :meth:`set`)."""
        self._check(slot)
        if allowed is None:
            self.masked[slot] = 0
            return
        if not (isinstance(allowed, np.ndarray) and allowed.dtype == np.int32):
            allowed = token_words(allowed, self.vocab)
        if allowed.shape != (self.mask.shape[1],):
            raise ValueError(f"LogitRules: {self.mask.shape[1]} words of "
                             "allowed tokens")
        self.mask[slot] = torch.from_numpy(
            np.ascontiguousarray(allowed)).to(self.mask.device)
        self.masked[slot] = 1

    def _check(self, slot: int):
        if not 0 <= slot < self.slots:
            raise ValueError(f"LogitRules: slot {slot} of {self.slots}")


def adjust_logits(logits: torch.Tensor, rules: LogitRules, rows: torch.Tensor,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """logits (N, V) bf16 or fp32, rows (N,) int32 every row's slot (one outside of the
    slots: the row stays as it is) -> logits under the rules, in their type:

        u = l / repetition where l > 0, else l * repetition, of tokens seen before
        u - frequency * (times in the output) - presence * (in the output) + bias

    and -inf for what is not allowed, in 32 bits, rounded once (no autograd).  ``out``: where
    they go, ``out=logits`` in place, else apart from it."""
    if logits.dim() != 2 or logits.shape[1] != rules.vocab:
        raise ValueError(f"adjust_logits: logits (N, {rules.vocab})")
    if rows.dtype != torch.int32 or rows.shape != logits.shape[:1]:
        raise ValueError("adjust_logits: rows (N,) int32")
    if torch.is_grad_enabled() and (
            logits.requires_grad or out is not None and out.requires_grad):
        raise RuntimeError("adjust_logits has no gradients: call it under "
                           "torch.no_grad()")
    if logits.is_cuda:
        ext = _ops._require_ext()
        if out is None:
            out = torch.empty(logits.shape, dtype=logits.dtype,
                              device=logits.device)
        ext.adjust_logits(out, logits, rows.contiguous(), rules.history,
                          rules.prompt_len, rules.total_len, rules.repetition,
                          rules.frequency, rules.presence, rules.bias_tokens,
                          rules.bias_values, rules.mask, rules.masked)
        return out
    if out is not None and ref.rows_overlap(out, logits) and (
            out.data_ptr() != logits.data_ptr() or out.stride() != logits.stride()):
        raise ValueError("adjust_logits: out is logits or apart from it")
    res = ref.adjust_logits(logits, rules, rows)
    return res if out is None else out.copy_(res)


def append_tokens(rules: LogitRules, rows: torch.Tensor,
                  tokens: torch.Tensor) -> None:
    """tokens (N,) int64 to the histories of slots ``rows`` (N,) int32, those of one slot in
    their order.  A full history stays as it is.  At most 16384 rows."""
    if rows.numel() > MOST_ROWS:
        raise ValueError(f"append_tokens: at most {MOST_ROWS} rows")
    if rows.dtype != torch.int32 or rows.dim() != 1 \
            or tokens.dtype != torch.int64 or tokens.shape != rows.shape:
        raise ValueError("append_tokens: rows (N,) int32, tokens (N,) int64")
    if rows.is_cuda:
        _ops._require_ext().append_tokens(rules.history, rules.total_len,
                                          rows.contiguous(), tokens.contiguous())
        return
    ref.append_tokens(rules, rows, tokens)
