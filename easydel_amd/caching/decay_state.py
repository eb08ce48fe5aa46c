"""State pool of linear attention with a decay per head: one float32 state per sequence and KV head, addressed by slot.

Where a paged cache grows with its sequence, a state stays ``k_headdim x v_headdim``: a running sequence owns one slot, and a
slot that it leaves behind (``state_out_indices``) is a snapshot other sequences can go on from, as shared prefix pages are.
The batch's ragged fields are those of the paged layers of the same step.
"""

from __future__ import annotations

from dataclasses import dataclass, field

import torch


@dataclass
class DecayStateCacheConfig:
    """Static description of the pool."""

    num_hidden_layers: int
    num_slots: int
    num_kv_heads: int
    k_headdim: int
    v_headdim: int

    @classmethod
    def create(cls, num_hidden_layers: int, num_kv_heads: int, k_headdim: int, v_headdim: int, *, num_slots: int | None = None,
               hbm_utilization: float = 0.1, free_hbm_bytes: int | None = None, device="cuda:0") -> "DecayStateCacheConfig":
        """``num_slots`` or as many slots as ``hbm_utilization`` of the free memory holds over all layers."""
        for name, value in (("num_hidden_layers", num_hidden_layers), ("num_kv_heads", num_kv_heads), ("k_headdim", k_headdim), ("v_headdim", v_headdim)):
            if value <= 0:
                raise ValueError(f"`{name}` must be positive")
        if num_slots is None:
            if free_hbm_bytes is None:
                free_hbm_bytes, _ = torch.cuda.mem_get_info(device)
            num_slots = int(free_hbm_bytes * hbm_utilization) // (num_hidden_layers * num_kv_heads * k_headdim * v_headdim * 4)
        if num_slots <= 0:
            raise ValueError("Computed `num_slots` is non-positive; increase `hbm_utilization` or reduce the state's size.")
        return cls(num_hidden_layers, int(num_slots), num_kv_heads, k_headdim, v_headdim)


@dataclass
class DecayStateMetadata:
    """Per-step metadata; every array is an int32 device tensor."""

    query_start_loc: torch.Tensor  # [max_num_reqs + 1]
    num_seqs: torch.Tensor  # [1]: live rows
    state_indices: torch.Tensor  # [max_num_reqs]: the slot a sequence goes on from
    context_lens: torch.Tensor | None = None  # [max_num_reqs], new tokens included: a sequence without earlier ones starts from zero
    state_out_indices: torch.Tensor | None = None  # [max_num_reqs]: the slot it leaves its state in, default the same

    @classmethod
    def from_ragged(cls, metadata, state_indices, state_out_indices=None) -> "DecayStateMetadata":
        """The fields a paged layer's ``RaggedPagesMetadata`` of the same step already holds, and the slots."""
        dist = getattr(metadata, "request_distribution", None)
        num_seqs = dist.reshape(-1)[2:3] if dist is not None else metadata.num_seqs.reshape(-1)[:1]
        return cls(query_start_loc=metadata.query_start_loc, num_seqs=num_seqs, state_indices=state_indices,
                   context_lens=metadata.context_lens, state_out_indices=state_out_indices)


@dataclass
class DecayStateCacheView:
    """One layer's states ``[num_slots, num_kv_heads, k_headdim, v_headdim]`` float32."""

    metadata: DecayStateCacheConfig
    state: torch.Tensor
    layer_index: int | None = None

    @classmethod
    def init(cls, config: DecayStateCacheConfig, layer_index: int | None = None, device="cuda:0") -> "DecayStateCacheView":
        shape = (config.num_slots, config.num_kv_heads, config.k_headdim, config.v_headdim)
        return cls(metadata=config, state=torch.zeros(shape, dtype=torch.float32, device=device), layer_index=layer_index)

    def concatenate_to_cache(self, key, value, cache_metadata) -> "DecayStateCacheView":
        """Nothing to do here: the operation advances the states."""
        return self


@dataclass
class DecayStateCache:
    """All layers' views."""

    views: list = field(default_factory=list)

    @classmethod
    def init_cache(cls, config: DecayStateCacheConfig, device="cuda:0") -> "DecayStateCache":
        return cls(views=[DecayStateCacheView.init(config, layer_index=i, device=device) for i in range(config.num_hidden_layers)])
