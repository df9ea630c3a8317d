"""The engine's requests whose next token goes by rules: which slot of the rules' tables
(``ops.LogitRules``) each has, and what its tokens may be."""
from __future__ import annotations

import math
from typing import Dict, List, Optional

import numpy as np
import torch

import polyrl_amd.ops as ops
from ..ops.rules import MOST_BIASES, MOST_TOKENS, in_32_bits, token_words


def allowed_words(sp, output_ids, vocab: int) -> Optional[np.ndarray]:
    """Words of the tokens that may come next (``ops.token_words``), None for all."""
    words = None
    if len(sp.allowed_token_ids):
        words = token_words(sp.allowed_token_ids, vocab)
    if sp.token_mask is not None:
        now = sp.token_mask(list(output_ids))
        if now is not None:
            if not (isinstance(now, np.ndarray) and now.dtype == np.int32):
                now = token_words(now, vocab)
            if now.shape != ((vocab + 31) // 32,):
                raise ValueError("token_mask: words of another vocabulary")
            words = now if words is None else words & now
    return words


def leaves_a_token(words: Optional[np.ndarray], sp, vocab: int) -> bool:
    """Whether some token is allowed that no bias of -inf bans."""
    banned = [int(t) for t, v in dict(sp.logit_bias).items()
              if in_32_bits(v) == -math.inf]
    if words is None:
        return len(banned) < vocab
    bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:vocab]
    bits[banned] = 0
    return bool(bits.any())


class RequestRules:
    """Slots of ``ops.LogitRules`` by request id, made when the first request with rules is
    sampled and made larger when there are more of them than slots."""

    def __init__(self, vocab: int, capacity: int, slots: int, device):
        self.vocab, self.device = vocab, device
        self.capacity = min(capacity, MOST_TOKENS)
        self.first = slots
        self.table: Optional[ops.LogitRules] = None
        self._slots: Dict[str, int] = {}
        self._free: List[int] = []

    def check(self, sp, prompt_len: int) -> Optional[np.ndarray]:
        """What the first token may be (:func:`allowed_words`); ValueError for rules that no
        table could hold."""
        for name in ("repetition_penalty", "frequency_penalty",
                     "presence_penalty"):
            v = in_32_bits(getattr(sp, name))
            if not math.isfinite(v) or name[0] == "r" and v <= 0:
                raise ValueError(f"{name} {v}")
        bias = dict(sp.logit_bias)
        if len(bias) > MOST_BIASES:
            raise ValueError(f"more than {MOST_BIASES} biases")
        for t, v in bias.items():
            v = in_32_bits(v)
            if not 0 <= int(t) < self.vocab or math.isnan(v) or v == math.inf:
                raise ValueError(f"logit_bias {v} of token {t}")
        if prompt_len > self.capacity:
            raise ValueError(f"rules for a prompt of {prompt_len} tokens, more "
                             f"than {self.capacity}")
        try:
            words = allowed_words(sp, [], self.vocab)
        except ValueError:
            raise
        except Exception as e:               # the caller's token_mask
            raise ValueError(f"token_mask: {e!r}") from e
        if not leaves_a_token(words, sp, self.vocab):
            raise ValueError("rules that leave no token")
        # (kept until the first token is drawn: a mask may fill its words again)
        return None if words is None else words.copy()

    def rows(self, reqs) -> Optional[torch.Tensor]:
        """Slots of the requests on the device, -1 where one has no rules; None if none
        has."""
        if not any(r.sampling.has_rules for r in reqs):
            return None
        slots = [self._slot(r) if r.sampling.has_rules else -1 for r in reqs]
        return torch.tensor(slots, dtype=torch.int32, device=self.device)

    def advance(self, r) -> bool:
        """After a token of a request with a ``token_mask``: what may come next, or
        False if nothing may."""
        words = allowed_words(r.sampling, r.output_ids, self.vocab)
        if not leaves_a_token(words, r.sampling, self.vocab):
            return False
        self.table.allow(self._slots[r.rid], words)
        return True

    def release(self, rid: str) -> None:
        slot = self._slots.pop(rid, None)
        if slot is not None:
            self._free.append(slot)

    def _slot(self, r) -> int:
        slot = self._slots.get(r.rid)
        if slot is not None:
            return slot
        sp = r.sampling
        bias = dict(sp.logit_bias)
        if self.table is None or not self._free \
                or len(bias) > self.table.biases:
            self._enlarge(len(bias))
        slot = self._free[-1]
        self.table.set(slot, r.input_ids, r.output_ids,
                       repetition=sp.repetition_penalty,
                       frequency=sp.frequency_penalty,
                       presence=sp.presence_penalty, bias=bias,
                       allowed=r.first_words)
        self._free.pop()
        self._slots[r.rid] = slot
        return slot

    def _enlarge(self, biases: int) -> None:
        old = self.table
        slots = self.first if old is None else \
            old.slots if self._free else 2 * old.slots
        most = 0 if old is None else old.biases
        if biases > most:
            most = min(max(2 * most, biases), MOST_BIASES)
        new = ops.LogitRules(slots, self.vocab, self.capacity, self.device,
                             biases=most)
        n = 0
        if old is not None:
            n = old.slots
            for name, t in vars(old).items():
                if isinstance(t, torch.Tensor):
                    to = getattr(new, name)[:n]
                    (to[:, :t.shape[1]] if t.dim() == 2 else to).copy_(t)
        self._free.extend(range(n, slots))
        self.table = new
