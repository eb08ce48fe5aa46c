"""The rotation a layer hands to the operations that write rotated keys: its table of cosines and sines and its pairing.

The reference keeps the same table (cosines, then sines, of every position's angles) and the same two pairings in its rotary
layers, which its attention block applies ahead of the cache write (easydel/layers/attention/_unified.py:1092-1133); here the
write applies it (``kernels.rope_page_scatter_ragged``).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass
class Rotary:
    """``cos_sin [positions, rope_dim]`` float32 on the GPU; ``is_neox_style``: pairs ``(d, d + rope_dim / 2)``, else ``(2 d, 2 d + 1)``.

    Any scaling of the angles (linear, by frequency bands, a factor on the cosines and sines) belongs into the table."""

    cos_sin: torch.Tensor
    is_neox_style: bool = True

    @classmethod
    def create(cls, rope_dim: int, max_positions: int, theta: float = 10000.0, is_neox_style: bool = True, device="cuda:0") -> "Rotary":
        """The plain table: angle ``p * theta ** (-2 d / rope_dim)``, in 64 bits (the angles of far positions need them)."""
        if rope_dim <= 0 or rope_dim % 2:
            raise ValueError(f"`rope_dim` must be positive and even, got {rope_dim}")
        if max_positions <= 0:
            raise ValueError(f"`max_positions` must be positive, got {max_positions}")
        inv = theta ** (-torch.arange(0, rope_dim, 2, dtype=torch.float64) / rope_dim)
        angle = torch.arange(max_positions, dtype=torch.float64)[:, None] * inv
        return cls(torch.cat((angle.cos(), angle.sin()), dim=1).to(torch.float32).to(device), is_neox_style)
