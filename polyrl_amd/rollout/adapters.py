"""Low-rank adapters of the rollout engine: many at once, each request by its own.

The base weights stay as they are; every projection adds its adapters' part
(``ops.adapter_add``) to the rows of requests that name one.  The pool holds them in
buffers by slot, so that loading one into a free slot is a plain copy that captured decode
steps see.  With tensor parallelism a rank holds its share: rows of B where the
projection's rows are sharded, columns of A where its columns are, so that the all-reduce
behind the projection sums the adapters' part too.
"""
from __future__ import annotations

import math
import re
from typing import Dict, Iterable, List, Tuple

import torch

import polyrl_amd.ops as ops
from ..ops.rules import in_32_bits

# parts of the fused projections, in the order of their rows
PROJECTIONS = {"qkv": ("q", "k", "v"), "o": ("o",), "gate_up": ("gate", "up"),
               "down": ("down",)}
_OF = {part: (proj, i) for proj, parts in PROJECTIONS.items()
       for i, part in enumerate(parts)}
_NAME = re.compile(r"(?:^|\.)layers\.(\d+)\.(?:self_attn|mlp)\.([a-z]+)_proj\."
                   r"lora_([AB])(?:\.default)?(?:\.weight)?$")


class AdapterPool:
    """Adapters of an ``InferenceModel`` of the llama/qwen2 families."""

    def __init__(self, model, slots: int, rank: int):
        cfg, tp = model.cfg, model.tp.size
        if cfg.arch not in ("llama", "qwen2"):
            raise ValueError("adapters are for the llama and qwen2 families")
        if not 1 <= slots <= ops.adapters.MOST_ADAPTERS \
                or not 1 <= rank <= ops.adapters.MOST_RANK:
            raise ValueError(f"{slots} adapters of ranks up to {rank}")
        self.tp = model.tp
        self.slots, self.rank = slots, rank
        hq = cfg.num_attention_heads * cfg.head_dim // tp
        hk = cfg.num_key_value_heads * cfg.head_dim // tp
        h, ff = cfg.hidden_size, cfg.intermediate_size // tp
        self.widths = {"qkv": (hq, hk, hk), "o": (h,), "gate_up": (ff, ff),
                       "down": (h,)}
        inner = {"qkv": h, "o": hq, "gate_up": h, "down": ff}
        wide = -(-rank // 8) * 8          # rows of B in whole 16-byte words
        self.dtype = model.dtype
        new = dict(dtype=model.dtype, device=model.device)
        self.layers = [
            {proj: (torch.zeros(slots, len(w), wide, inner[proj], **new),
                    torch.zeros(slots, sum(w), wide, **new))
             for proj, w in self.widths.items()}
            for _ in range(cfg.num_hidden_layers)]
        self.scale = torch.ones(slots, device=model.device)
        self.ranks = {proj: torch.zeros(slots, dtype=torch.int32,
                                        device=model.device)
                      for proj in PROJECTIONS}
        self.names: Dict[str, int] = {}

    def index(self, names: Iterable[str]) -> List[int]:
        """Slots of requests' adapters, -1 for none."""
        return [self.names[n] if n else -1 for n in names]

    def plan(self, index: torch.Tensor):
        return ops.adapter_plan(index, self.slots)

    def add(self, layer: int, proj: str, y: torch.Tensor, x: torch.Tensor,
            plan) -> None:
        """y += every row's adapter of x, in place."""
        a, b = self.layers[layer][proj]
        ops.adapter_add(y, x, a, b, self.scale, plan, widths=self.widths[proj],
                        ranks=self.ranks[proj], out=y)

    @torch.no_grad()
    def load(self, name: str, state_dict: Dict[str, torch.Tensor],
             scaling: float) -> None:
        """``state_dict``: ``...layers.N.self_attn.q_proj.lora_A`` (r, in) and ``.lora_B``
        (out, r) of any of the seven projections, as ``models.lora.export_adapter`` and
        common adapter files name them.  A name that is there already is replaced."""
        parts = self._parts(state_dict)
        if not name or not math.isfinite(in_32_bits(scaling)):
            raise ValueError(f"adapter {name!r}: scaling {scaling}")
        slot = self.names.get(name)
        if slot is None:
            free = set(range(self.slots)) - set(self.names.values())
            if not free:
                raise RuntimeError(f"all {self.slots} adapter slots are taken")
            slot = min(free)
        # all that can be refused comes before the slot's first change: an adapter of this
        # name stays whole
        parts = {key: [t.to(device=self.scale.device, dtype=self.dtype) for t in pair]
                 for key, pair in parts.items()}
        for layer in self.layers:
            for a, b in layer.values():
                a[slot].zero_()
                b[slot].zero_()
        most = dict.fromkeys(PROJECTIONS, 0)
        for (li, part), (A, B) in parts.items():
            proj, i = _OF[part]
            a, b = self.layers[li][proj]
            at = sum(self.widths[proj][:i])
            r = A.shape[0]
            a[slot, i, :r].copy_(A)
            b[slot, at:at + self.widths[proj][i], :r].copy_(B)
            most[proj] = max(most[proj], r)
        self.scale[slot] = scaling
        for proj, r in most.items():
            self.ranks[proj][slot] = r
        self.names[name] = slot

    def unload(self, name: str) -> None:
        slot = self.names.pop(name)
        for ranks in self.ranks.values():
            ranks[slot] = 0

    def _parts(self, state_dict) -> Dict[Tuple[int, str], list]:
        """{(layer, part): (A, B)}, this rank's shares, all shapes checked."""
        parts: Dict[Tuple[int, str], list] = {}
        for key, t in state_dict.items():
            m = _NAME.search(key)
            if m is None or m[2] not in _OF or int(m[1]) >= len(self.layers):
                raise ValueError(f"no projection of this model: {key}")
            pair = parts.setdefault((int(m[1]), m[2]), [None, None])
            if pair[m[3] == "B"] is not None:
                raise ValueError(f"named twice: {key}")
            pair[m[3] == "B"] = t
        if not parts:
            raise ValueError("an adapter without tensors")
        n, at = self.tp.size, self.tp.rank
        for (li, part), (A, B) in parts.items():
            proj, i = _OF[part]
            width, k = self.widths[proj][i], self.layers[li][proj][0].shape[3]
            split_in = proj in ("o", "down")
            if A is None or B is None or A.dim() != 2 or B.dim() != 2 \
                    or A.shape[0] != B.shape[1] \
                    or not 1 <= A.shape[0] <= self.rank \
                    or A.shape[1] != (k * n if split_in else k) \
                    or B.shape[0] != (width if split_in else width * n):
                raise ValueError(
                    f"layer {li}, {part}_proj: A "
                    f"{None if A is None else tuple(A.shape)}, B "
                    f"{None if B is None else tuple(B.shape)}; ranks up to "
                    f"{self.rank}")
            if split_in:
                A = A[:, at * k:(at + 1) * k]
            else:
                B = B[at * width:(at + 1) * width]
            parts[li, part] = (A, B)
        return parts
