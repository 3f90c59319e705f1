"""The quantised key/value cache: e4m3 codes with one fp32 scale for each (token, head).

``kernels.kv_cache_write`` fills it behind the QKV projection, ``kernels.prefix_attention`` attends over it and
``kernels.kv_cache_read`` gives it back as bf16.  Per head and token it holds ``head_dim + 4`` bytes for keys and for values
where a bf16 cache holds ``2 * head_dim``.
"""

from __future__ import annotations

from typing import NamedTuple

import torch


class QuantizedKVCache(NamedTuple):
    """``k_codes`` / ``v_codes``: e4m3 (any one-byte type) [batch, kv_heads, capacity, head_dim]; ``k_scales`` / ``v_scales``:
    fp32 [batch, kv_heads, capacity].  All contiguous; a row stands for ``code * scale``.  Value scales that ``prefix_attention`` reads
    are below 2^32, as a write leaves them."""

    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor

    @classmethod
    def allocate(cls, batch: int, kv_heads: int, capacity: int, head_dim: int, device: torch.device | str) -> "QuantizedKVCache":
        """An empty cache: every row reads back as zero.  One that outlives a call is allocated outside graph capture, like every plan
        buffer; inside, it is the graph's own and empty again at every replay."""
        codes = lambda: torch.zeros((batch, kv_heads, capacity, head_dim), device=device, dtype=torch.uint8).view(torch.float8_e4m3fn)
        scales = lambda: torch.zeros((batch, kv_heads, capacity), device=device)
        return cls(codes(), scales(), codes(), scales())
