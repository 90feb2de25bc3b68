"""Device memory behind the cache manager's bookkeeping.

Layers with the same need share a group.  A paged group holds, for each of its layers,
keys and values as ``[pages, n_kv_heads, page_size, head_dim]`` in the compute dtype; one
page id is valid in every layer of its group.  Pages of a need without values have no value half.  A slot group holds ``[layers, slots, *shape]``
in the element type its need names, set to the need's initial value when a request starts.  A cache opened with an 8-bit type
(``cache_dtype``: "e4m3" or "int8") holds the pages of needs that allow it as codes, with float32 scales ``[pages, n_kv_heads,
page_size / block]`` beside them, blocks of EIGHT_BIT_BLOCK tokens (or of a page, if that is smaller).  The reference keeps one pool per attention layer in fp16
(gpu/cuda/paged_attention.cu:34-67) and conv states on the host between steps.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from .manager import PagedNeed, SlotNeed


_SLOT_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16, "int32": torch.int32}


EIGHT_BIT_DTYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
EIGHT_BIT_BLOCK = 16         # tokens of a scale: 4 bytes for each 16 * head_dim codes


def parse_cache_dtype(name: Optional[str]) -> Optional[torch.dtype]:
    """The torch type of a cache type's name; None for none (the compute dtype)."""
    if name is None or isinstance(name, torch.dtype) and name in EIGHT_BIT_DTYPES.values():
        return name
    if name not in EIGHT_BIT_DTYPES:
        raise ValueError(f"unknown cache type {name!r}; one of {sorted(EIGHT_BIT_DTYPES)}, or None for the compute dtype")
    return EIGHT_BIT_DTYPES[name]


def page_bytes(need: PagedNeed, page_size: int, dtype: torch.dtype, cache_dtype: Optional[torch.dtype] = None) -> int:
    """Device bytes of one page of one layer: keys and values, or codes and scales."""
    if cache_dtype is None or not need.eight_bit:
        return need.elements_per_token() * page_size * torch.empty((), dtype=dtype).element_size()
    return need.elements_per_token() * page_size + 2 * need.n_kv_heads * 4 * max(1, page_size // EIGHT_BIT_BLOCK)


@dataclass
class LayerCache:
    kind: str                 # "paged" | "slot" | "none"
    group: int = -1           # index among groups of its kind
    index: int = -1           # layer's index inside the group


class CacheStorage:
    def __init__(self, needs: Sequence[object], *, pages_per_group, page_size: int, max_requests: int,
                 dtype: torch.dtype, device, cache_dtype: Optional[torch.dtype] = None):
        """``needs`` maps a cache id to its PagedNeed / SlotNeed / None.  ``pages_per_group`` is
        an int (every paged group gets that many pages) or a callable ``need -> pages``.  ``cache_dtype``: an 8-bit
        type for the pages of needs that allow it."""
        self.page_size, self.dtype, self.device, self.cache_dtype = page_size, dtype, device, cache_dtype
        if cache_dtype is not None and page_size < 8:
            raise ValueError(f"a cache in 8 bits has pages of at least 8 tokens, got {page_size}")
        self.paged_needs: List[PagedNeed] = []
        self.slot_needs: List[SlotNeed] = []
        self.layers: Dict[int, LayerCache] = {}
        counts_p: List[int] = []
        counts_s: List[int] = []
        def place(need) -> LayerCache:
            if need is None:
                return LayerCache("none")
            if isinstance(need, PagedNeed):
                if need not in self.paged_needs:
                    self.paged_needs.append(need)
                    counts_p.append(0)
                g = self.paged_needs.index(need)
                counts_p[g] += 1
                return LayerCache("paged", g, counts_p[g] - 1)
            if isinstance(need, SlotNeed):
                if need not in self.slot_needs:
                    self.slot_needs.append(need)
                    counts_s.append(0)
                g = self.slot_needs.index(need)
                counts_s[g] += 1
                return LayerCache("slot", g, counts_s[g] - 1)
            raise TypeError(f"a layer declared an unknown cache need: {need!r}")

        # a layer that keeps several things declares a tuple of needs and is handed a tuple of views
        for cid in sorted(needs):
            need = needs[cid]
            self.layers[cid] = tuple(place(n) for n in need) if isinstance(need, tuple) else place(need)
        self.pages_per_group = [pages_per_group(n) if callable(pages_per_group) else int(pages_per_group)
                                for n in self.paged_needs]
        self.k: List[torch.Tensor] = []
        self.v: List[torch.Tensor] = []
        self.k_scales: List[Optional[torch.Tensor]] = []
        self.v_scales: List[Optional[torch.Tensor]] = []
        for need, n_layers, pages in zip(self.paged_needs, counts_p, self.pages_per_group):
            shape = (n_layers, pages, need.n_kv_heads, page_size, need.head_dim)
            vh, vd = need.value_shape()
            if cache_dtype is not None and need.eight_bit:
                blocks = shape[:3] + (max(1, page_size // EIGHT_BIT_BLOCK),)
                self.k.append(torch.zeros(shape, dtype=cache_dtype, device=device))
                self.v.append(torch.zeros(shape, dtype=cache_dtype, device=device))
                self.k_scales.append(torch.ones(blocks, device=device))
                self.v_scales.append(torch.ones(blocks, device=device))
                continue
            self.k_scales.append(None)
            self.v_scales.append(None)
            self.k.append(torch.zeros(shape, dtype=dtype, device=device))
            self.v.append(torch.zeros((n_layers, pages, vh, page_size, vd), dtype=dtype, device=device)
                          if need.values else None)
        for need in self.slot_needs:
            if need.dtype not in _SLOT_DTYPES:
                raise TypeError(f"a layer asks for state of dtype {need.dtype!r}; one of {sorted(_SLOT_DTYPES)}")
        self.state: List[torch.Tensor] = [
            torch.full((n_layers, max_requests) + tuple(need.shape), need.init, dtype=_SLOT_DTYPES[need.dtype],
                       device=device)
            for need, n_layers in zip(self.slot_needs, counts_s)]

    def reset_slot(self, slot: int) -> None:
        """Every layer's state of the slot back to its need's initial value (a request starts)."""
        for s, need in zip(self.state, self.slot_needs):
            s[:, slot].fill_(need.init)

    def pools(self, group: int) -> List[torch.Tensor]:
        """Everything a paged group keeps for its pages, each [layers, pages, ...]."""
        return [t for t in (self.k[group], self.v[group], self.k_scales[group], self.v_scales[group]) if t is not None]

    def copy_slot(self, src: int, dst: int) -> None:
        """Every layer's state of slot ``src`` to slot ``dst``."""
        for s in self.state:
            s[:, dst].copy_(s[:, src])

    def bytes_per_token(self) -> int:
        """Bytes a token takes over all paged layers (scales by the page, rounded down)."""
        return sum(k.shape[0] * page_bytes(n, self.page_size, self.dtype, self.cache_dtype) // self.page_size
                   for k, n in zip(self.k, self.paged_needs))

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.k + self.v + self.k_scales + self.v_scales + self.state if t is not None)
