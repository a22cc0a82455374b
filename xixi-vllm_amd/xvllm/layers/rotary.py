"""Rotary embedding module and its fp32 cos||sin table
(reference ``rotary.py:7-62``)."""
from __future__ import annotations

import torch
from torch import nn

from . import ops  # noqa: F401


def build_cos_sin_cache(head_dim: int, max_position_embeddings: int, rope_theta: float, first: int = 0) -> torch.Tensor:
    """[max_pos, head_dim] fp32 table: cos of the NeoX half-split angles in the
    first head_dim/2 columns, sin in the rest.  inv_freq_i = theta^(-2i/D),
    angle = pos * inv_freq_i, all in fp32 in that order (rotary.py:13-20).
    first: the rows of positions first .. max_pos - 1 alone."""
    exponent = torch.arange(0, head_dim, 2, dtype=torch.float) / head_dim
    inv_freq = 1.0 / (rope_theta ** exponent)
    pos = torch.arange(first, max_position_embeddings, dtype=torch.float)
    ang = pos[:, None] * inv_freq[None, :]
    return torch.cat((ang.cos(), ang.sin()), dim=-1)


class RotaryEmbedding(nn.Module):
    def __init__(self, head_dim: int, rotary_dim: int, max_position_embeddings: int, rope_theta: float) -> None:
        super().__init__()
        self.head_dim, self.rope_theta = head_dim, rope_theta
        self._outgrown: list[torch.Tensor] = []
        assert rotary_dim == head_dim, "rotary_dim must equal head_dim (full rotation)"
        self.register_buffer(
            "cos_sin_cache", build_cos_sin_cache(head_dim, max_position_embeddings, rope_theta), persistent=False
        )

    def reserve(self, positions: int) -> None:
        """Make the table hold positions 0 .. positions - 1.  The kernels index
        it by position and do not know its length: a step past it would read
        what lies behind the table, or fault.  Rows that are there stay as they
        are, and so does a table that a recorded graph may still read."""
        table = self.cos_sin_cache
        if positions <= table.shape[0]:
            return
        with torch.inference_mode(False), torch.device(table.device):
            more = build_cos_sin_cache(self.head_dim, positions, self.rope_theta, first=table.shape[0])
        self._outgrown.append(table)
        self.cos_sin_cache = torch.cat((table, more))

    def _apply(self, fn, recurse: bool = True):
        out = super()._apply(fn, recurse)
        if self.cos_sin_cache.dtype != torch.float32:  # the kernel reads an fp32 table
            self.cos_sin_cache = self.cos_sin_cache.to(torch.float32)
        return out

    def forward(self, positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor):
        return torch.ops.vllm.rotary_embedding(query, key, positions, self.cos_sin_cache, self.head_dim)
