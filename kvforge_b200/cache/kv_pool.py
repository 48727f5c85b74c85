"""Device storage of the cache: per group one K and one V tensor
``[entries, num_blocks, kv_heads, block_size, head_dim]`` (an entry per layer call that keeps
a cache; V with the value size of a head where a mixer gives it one of its own), and per stateful mixer call a float tensor ``[num_slots, *state_shape]``.

umarhassan-cloud/kvforge keeps ``[num_blocks, block_size, kv_heads, head_dim]`` per layer
(src/tokenvault/cache/kv_cache.py:27-31).  Here the kv-head index comes before the
position inside a page, so the keys of one head in one page are one contiguous run of
``block_size * head_dim`` elements.
"""

from __future__ import annotations

import torch

from .. import ops
from ..parts.base import LayerCache


class KVPool:
    def __init__(self, model, num_blocks: int, block_size: int, num_slots: int, dtype: torch.dtype, device) -> None:
        self.num_blocks, self.block_size, self.dtype = num_blocks, block_size, dtype
        self.k: list[torch.Tensor] = []
        self.v: list[torch.Tensor] = []
        for g in model.groups:
            shape = (len(g.calls), num_blocks, g.need.kv_heads, block_size)
            self.k.append(torch.zeros((*shape, g.need.head_dim), dtype=dtype, device=device))
            # values that are the leading part of the keys (a latent shared by keys and values) have no tensor of their own
            self.v.append(self.k[-1] if g.need.v_in_k else torch.zeros((*shape, g.need.value_dim), dtype=dtype, device=device))
        self.states: list[torch.Tensor | None] = []
        for shape in model.state_shapes:
            self.states.append(None if shape is None else torch.zeros((num_slots, *shape), dtype=torch.float32, device=device))
        self._state_table: ops.StateTable | None = None
        self.caches: list[LayerCache | None] = []
        for idx, call in enumerate(model.spec.execution):
            owner = model.call_group[idx if call.kv_from is None else call.kv_from]
            if owner is None:
                cache = None if self.states[idx] is None else LayerCache(None, None, -1, True, self.states[idx])
            else:
                gi, entry = owner
                cache = LayerCache(self.k[gi][entry], self.v[gi][entry], gi, call.kv_from is None, self.states[idx])
            self.caches.append(cache)

    @property
    def memory_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.k + [v for k, v in zip(self.k, self.v) if v is not k])

    @property
    def bytes_per_block(self) -> int:
        return self.memory_bytes // max(1, self.num_blocks)

    def clear_state_slots(self, slots: list[int]) -> None:
        if not slots:
            return
        for st in self.states:
            if st is not None:
                st[slots] = 0

    def copy_pages(self, copies: list[tuple[int, int, int, int]]) -> None:
        """(group, source page, target page, positions) as ``BlockManager.fork`` returns them: one launch a group, every layer."""
        for gi, k in enumerate(self.k):
            rows = [c[1:] for c in copies if c[0] == gi]
            if rows:
                src, dst, tokens = torch.tensor(rows, dtype=torch.int32).t().contiguous().to(k.device)
                v = self.v[gi]
                ops.copy_pages(k, None if v is k else v, src, dst, tokens)

    def copy_states(self, copies: list[tuple[int, int]]) -> None:
        """(source slot, target slot): every mixer's state, one launch."""
        states = [t for t in self.states if t is not None]
        if not copies or not states:
            return
        if self._state_table is None:
            self._state_table = ops.StateTable(states)
        src, dst = torch.tensor(copies, dtype=torch.int32).t().contiguous().to(states[0].device)
        ops.copy_states(self._state_table, src, dst)


def bytes_per_block(model, block_size: int, dtype: torch.dtype) -> int:
    """Bytes that one page index costs over all groups and entries, keys and values
    (src/tokenvault/config.py:91-95 for a single group)."""
    elem = torch.tensor([], dtype=dtype).element_size()
    return sum(len(g.calls) * block_size * g.need.kv_heads * (g.need.head_dim + (0 if g.need.v_in_k else g.need.value_dim)) * elem for g in model.groups)
