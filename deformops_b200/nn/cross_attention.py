"""``RotaryCrossAttn``: dense attention to an encoder's states with rotary positions on both sides.

The layer a decoder holds beside :class:`MultiScaleDeformAttn2d`: the same queries and the same
flattened pyramid, but every state is looked at.
"""

from __future__ import annotations

from typing import Sequence

from torch import Tensor, nn

from ..core.linear import project, project_pair
from ..registry.cross_attention import cross_attention
from ..registry.msda import Backend
from ..registry.rotary import rotary

__all__ = ["RotaryCrossAttn"]


class RotaryCrossAttn(nn.Module):
    """Projections, rotary positions (where positions are given) and :func:`cross_attention`.

    ``num_kv_heads`` (default ``num_heads``) key heads are shared by equal numbers of query heads.
    ``sections``, ``base`` and ``interleaved`` are those of :func:`rotary`.
    """

    def __init__(self, dim: int, dim_memory: int | None = None, dim_output: int | None = None, *, num_heads: int,
                 num_kv_heads: int | None = None, sections: Sequence[int] | None = None, base: float = 10000.0,
                 interleaved: bool = False, backend: Backend | None = None):
        super().__init__()
        num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        for name, v in (("dim", dim), ("num_heads", num_heads), ("num_kv_heads", num_kv_heads)):
            if not isinstance(v, int) or v <= 0:
                raise ValueError(f"{name} must be a positive integer, got {v!r}")
        if dim % num_heads:
            raise ValueError(f"dim ({dim}) must be divisible by num_heads ({num_heads})")
        if num_heads % num_kv_heads:
            raise ValueError(f"num_heads ({num_heads}) must be divisible by num_kv_heads ({num_kv_heads})")
        self.dim, self.num_heads, self.num_kv_heads = dim, num_heads, num_kv_heads
        self.sections = None if sections is None else tuple(sections)
        self.base, self.interleaved, self.backend = base, interleaved, backend
        head = dim // num_heads
        self.proj_query = nn.Linear(dim, dim)
        self.proj_key = nn.Linear(dim_memory or dim, num_kv_heads * head)
        self.proj_value = nn.Linear(dim_memory or dim, num_kv_heads * head)
        self.proj_output = nn.Linear(dim, dim_output or dim)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        for proj in (self.proj_query, self.proj_key, self.proj_value, self.proj_output):
            nn.init.xavier_uniform_(proj.weight)
            nn.init.zeros_(proj.bias)

    def forward(self, q: Tensor, memory: Tensor, query_positions: Tensor | None = None,
                memory_positions: Tensor | None = None, key_padding_mask: Tensor | None = None,
                attention_mask: Tensor | None = None) -> Tensor:
        """``q (B,Q,dim)``, ``memory (B,S,dim_memory)``, positions ``(B,Q,A)`` and ``(B,S,A)`` (or without
        the batch) -> ``(B,Q,dim_output)``.  Masks as :func:`cross_attention` takes them."""
        B, Q, _ = q.shape
        S, head = memory.shape[1], self.dim // self.num_heads
        query = project(self.proj_query, q).view(B, Q, self.num_heads, head)
        key, value = project_pair(self.proj_key, self.proj_value, memory)
        key = key.view(B, S, self.num_kv_heads, head)
        value = value.view(B, S, self.num_kv_heads, head)
        options = {"sections": self.sections, "base": self.base, "interleaved": self.interleaved,
                   "backend": self.backend}
        if query_positions is not None:
            query = rotary(query, query_positions, **options)
        if memory_positions is not None:
            key = rotary(key, memory_positions, **options)
        out = cross_attention(query, key, value, key_padding_mask=key_padding_mask, attention_mask=attention_mask,
                              backend=self.backend)
        return project(self.proj_output, out)
