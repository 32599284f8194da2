"""An attention layer for a batch of requests that share a long prefix, in 4-bit projections.

Several requests (edit prompts, or the guided and the unguided branch of one) work on the same cached rows,
such as the video tokens of the stream: their keys and values are held once (``PrefixCache.k_prefix``), each
request has its own rows after them.  One step of L new tokens per request:

    x [B, L, hidden] -> QKV projection in 4 bits            fp4_linear
                     -> rotation, keys and values appended    rotary_embed_append
                     -> attention over prefix and own rows    shared_prefix_attention
                     -> output projection in 4 bits         fp4_linear

The layer has what these operators need and no more: no normalisation of q and k before the rotation, and one
position per token.

Nothing is read back to the host: lengths, positions and cache slots stay on the GPU, so a step can be
captured into a CUDA graph (capture it with ``cache.filled`` left to the caller).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

import joyomni_ops as jo


@dataclass
class Fp4Weight:
    """A Linear layer's weight [N, K] in 4 bits."""

    q: torch.Tensor                   # uint8 [N, K/2]
    block: torch.Tensor               # block scales in tiles
    row: Optional[torch.Tensor]       # fp32 [N, 1] (nvfp4)
    bias: Optional[torch.Tensor]      # [N]

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return jo.fp4_linear(x, self.q, self.block, self.row, self.bias)


def quantize_linear_fp4(w: torch.Tensor, bias: Optional[torch.Tensor] = None, format: str = "nvfp4") -> Fp4Weight:
    """A Linear weight [N, K] laid out once for fp4_linear."""
    return Fp4Weight(*jo.quant_fp4(w, format), bias)


@dataclass
class PrefixCache:
    """Keys and values of one layer: the shared prefix, already rotated, and each request's own rows."""

    k_prefix: torch.Tensor  # [P, HK, D]
    v_prefix: torch.Tensor
    k_own: torch.Tensor     # [B, S, HK, D], contiguous
    v_own: torch.Tensor
    lens: torch.Tensor      # int32 [B], rows of each request
    filled: int = 0         # what the host knows of lens: no request has more rows (step keeps it)

    @classmethod
    def allocate(cls, k_prefix: torch.Tensor, v_prefix: torch.Tensor, batch: int, rows: int) -> "PrefixCache":
        _, hk, d = k_prefix.shape
        own = [k_prefix.new_empty(batch, rows, hk, d) for _ in range(2)]
        return cls(k_prefix, v_prefix, *own, torch.zeros(batch, dtype=torch.int32, device=k_prefix.device))


@dataclass
class PrefixAttention:
    """Weights of the layer."""

    qkv: Fp4Weight          # [(H + 2 HK) D, hidden]
    out: Fp4Weight          # [hidden, H D]
    heads: int
    kv_heads: int
    head_dim: int
    interleaved: bool = False


def step(layer: PrefixAttention, x: torch.Tensor, cache: PrefixCache, cos: torch.Tensor, sin: torch.Tensor,
         counts: Optional[torch.Tensor] = None, most: Optional[int] = None) -> torch.Tensor:
    """L new tokens of each request through the layer: x [B, L, hidden] -> [B, L, hidden]; the cache grows.

    Token i of request b stands at position P + lens[b] + i of the tables (``rope.rotary_tables``).  counts
    (int32 [B], at most L): how many of the L tokens request b really has, the last counts[b] of its rows (the
    first of them is its token 0); the padding in front of them is not cached and its outputs mean nothing.  most: the largest of counts, which the host
    cannot see in them (L if not given); the cache's room is reckoned by it.
    """
    b, n, hidden = x.shape
    rows = cache.k_own.shape[1]
    most = n if most is None else most
    if not 0 <= most <= n:
        raise ValueError(f"of {n} tokens per request the largest count cannot be {most}")
    if cache.filled + most > rows:
        raise ValueError(f"the cache holds {rows} rows per request: up to {cache.filled} are used and {most} come in")
    h, hk, d = layer.heads, layer.kv_heads, layer.head_dim
    qkv = layer.qkv(x.reshape(b * n, hidden)).view(b * n, h + 2 * hk, d)
    q, k, v = qkv.split((h, hk, hk), 1)
    i = torch.arange(n, device=x.device, dtype=torch.int32)
    new = cache.lens.new_full((b,), n) if counts is None else counts
    row = cache.lens[:, None] + i - (n - new)[:, None]  # own row of token i; before the first: padding
    kept = (i >= (n - new)[:, None]) & (row < rows)  # a replay beyond the cache's end leaves the next request alone
    slot = torch.where(kept, row.long() + rows * torch.arange(b, device=x.device)[:, None], -1)
    position = (cache.k_prefix.shape[0] + row.clamp(min=0)).long()
    q = jo.rotary_embed_append(q, k, v, cos, sin, position.view(-1), slot.view(-1), cache.k_own.view(b * rows, hk, d),
                               cache.v_own.view(b * rows, hk, d), layer.interleaved)
    cache.lens += new
    cache.filled += most
    o, _ = jo.shared_prefix_attention(q.view(b, n, h, d), cache.k_prefix, cache.v_prefix, cache.k_own, cache.v_own,
                                      cache.lens)
    return layer.out(o.view(b * n, h * d)).view(b, n, -1)
