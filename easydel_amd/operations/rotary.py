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


def token_rows(t: torch.Tensor) -> torch.Tensor:
    """``t [T, ...]`` with token rows that a kernel reads in place: contiguous each, however far apart.  Rows of a projection are; parts of
    every head (and one row for all tokens) are copied."""
    shape, apart = t.shape, t.stride()
    if len(shape) == 3 and apart[2] == 1 and apart[1] == shape[2] and apart[0] >= shape[1] * shape[2]:  # the common case, in few steps
        return t
    if t.is_contiguous() or shape[0] == 0:
        return t
    return t if t[0].is_contiguous() and (shape[0] == 1 or apart[0] >= t[0].numel()) else t.contiguous()


def rotation_operands(result: torch.dtype, *operands: torch.Tensor) -> list[torch.Tensor]:
    """The operands as the rotating writes read them: of one type, token rows in place.  Where types differ, among them or from that of
    the ``result``, they meet in float32, which holds 16-bit values as they are: what is rounded is the result, once."""
    if any(t.dtype != result for t in operands):
        operands = [t.to(torch.float32) for t in operands]
    return [token_rows(t) for t in operands]
