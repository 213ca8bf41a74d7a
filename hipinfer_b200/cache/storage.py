"""Device memory behind the cache manager's page ids and state slots.

Per cache group and plane (keys, values, or what else the group's mixers keep per token) one
tensor [layer cache, page, head, page_size, width] in the compute element type: a (page, head)
pair is one contiguous run of page_size * width elements, which is what the attention kernels
stream. Keys and values may be kept in 8 bits instead: the same tensors hold codes, and planes "k_scale" and "v_scale"
[layer cache, page, head, blocks of 16 places] the float32 scales (ops.Cache8). Per declared state one tensor [state slot, *shape]. The pools start zeroed: a kernel
that loads a whole page and masks the tail must never meet a NaN pattern there.

The reference allocates `[layer][slot][kv head][max_seq][head_dim]` once (src/api.cu:1409-1411).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from ..kernels import ops
from .manager import CacheGroupSpec


@dataclass
class LayerCache:
    planes: Dict[str, torch.Tensor]      # plane name -> [page, head, page_size, width]
    group: int
    write: bool
    cache8: object = None                # the planes as an ops.Cache8, where they are in 8 bits

    @property
    def k(self) -> torch.Tensor:
        return self.planes["k"]

    @property
    def v(self) -> torch.Tensor:
        return self.planes["v"]


def _planes8(group: CacheGroupSpec, pages: int, page_size: int, dtype, device) -> Dict[str, torch.Tensor]:
    if [name for name, _, _ in group.planes] != ["k", "v"] or group.planes[0][1:] != group.planes[1][1:]:
        raise ValueError(f"cache group {group.name!r}: planes {group.planes} cannot be kept in 8 bits (keys and values of one shape can)")
    (_, heads, width), n = group.planes[0], group.n_layers
    codes = {name: torch.zeros(n, pages, heads, page_size, width, dtype=torch.uint8, device=device).view(dtype) for name in "kv"}
    return {**codes, **{f"{name}_scale": torch.zeros(n, pages, heads, ops.cache8_blocks(page_size), dtype=torch.float32, device=device) for name in "kv"}}


class CacheStorage:
    def __init__(self, groups: Sequence[CacheGroupSpec], num_pages: Sequence[int], page_size: int, dtype, device,
                 state_specs: Dict[Tuple[int, str], Tuple[Tuple[int, ...], torch.dtype]], num_state_slots: int,
                 cache_dtype: Optional[torch.dtype] = None, spare_pages: int = 0):
        """`spare_pages` of each group lie behind those that the cache manager hands out (a cache in 8 bits alone)."""
        self.groups, self.page_size, self.dtype, self.cache_dtype = list(groups), page_size, dtype, cache_dtype
        self.kv = [{name: torch.zeros(g.n_layers, n, heads, page_size, width, dtype=dtype, device=device)
                    for name, heads, width in g.planes} for g, n in zip(self.groups, num_pages)] if cache_dtype is None else \
                  [_planes8(g, n + spare_pages, page_size, cache_dtype, device) for g, n in zip(self.groups, num_pages)]
        self.state: Dict[Tuple[int, str], torch.Tensor] = {
            key: torch.zeros((num_state_slots,) + tuple(shape), dtype=dt, device=device)
            for key, (shape, dt) in state_specs.items()}
        self._layer_caches: Dict[Tuple[int, int, bool], LayerCache] = {}
        self._by_step: Dict[int, Dict[str, torch.Tensor]] = {}
        for (step, name), t in self.state.items():
            self._by_step.setdefault(step, {})[name] = t

    def layer_cache(self, plan) -> Optional[LayerCache]:
        if plan is None:
            return None
        key = (plan.group, plan.slot, plan.write)
        if key not in self._layer_caches:
            planes = {name: t[plan.slot] for name, t in self.kv[plan.group].items()}
            self._layer_caches[key] = LayerCache(planes, plan.group, plan.write,
                                                 None if self.cache_dtype is None else ops.Cache8(*(planes[n] for n in ("k", "v", "k_scale", "v_scale"))))
        return self._layer_caches[key]

    def layer_state(self, step: int) -> Dict[str, torch.Tensor]:
        return self._by_step.get(step, {})

    def zero_state_slot(self, slot: int) -> None:
        """A request admitted to `slot` starts from zero state."""
        for t in self.state.values():
            t[slot].zero_()

    def copy_pages(self, group: int, src: Sequence[int], dst: Sequence[int]) -> None:
        """Pages of a group copied to others, in all its layers and planes."""
        ops.copy_pages(list(self.kv[group].values()), src, dst)

    def bytes_per_token(self) -> int:
        if self.cache_dtype is not None:
            return -(-sum(t[:, 0].numel() * t.element_size() for g in self.kv for t in g.values()) // self.page_size)
        return sum(g.elements_per_token() for g in self.groups) * torch.empty((), dtype=self.dtype).element_size()

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for g in self.kv for t in g.values()) + \
            sum(t.numel() * t.element_size() for t in self.state.values())
