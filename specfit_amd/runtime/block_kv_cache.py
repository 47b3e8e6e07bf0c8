"""A key/value cache with its complete blocks in 8 bits (K9, K10).

``BlockKVCache`` takes the place of the bf16 ``DynamicCache`` that the
reference's target keeps (src/specfit/runtime/eagle3_tree.py:833-858 and
:1202-1240 are the calls on it): half the bytes per step at long contexts.
Tokens enter in bf16 and stay so until the block of 64 they belong to is
complete and committed; it is then folded, once, into 8 bits with a
power-of-two scale per head.  A draft tree's nodes are never folded before
they are accepted, so compaction moves bf16 rows and no value is rounded
twice.
"""
from __future__ import annotations

from typing import Sequence

import torch

from .. import ops

BLOCK = ops.KV_BLOCK


class BlockKVCache:
    """Keys and values of ``batch`` sequences of one length in ``layers``
    layers.

    capacity     tokens the cache holds
    tail_tokens  tokens that can be there beyond the last folded block: the
                 longest prompt chunk or draft tree of one forward
    held         "e4m3" (relative steps: keeps small values beside loud ones)
                 or "int8" (128 steps over a block's range)

    A forward appends each layer's new tokens and attends over all of them
    (``append`` and ``attend``, or ``update`` for attention implementations
    that take plain tensors); ``commit`` then folds complete blocks.  In
    between, ``compact`` keeps the accepted path of a draft tree and ``crop``
    drops tokens from the end.  Calls are enqueued on the current stream;
    a caller that uses several streams orders them.  A captured call replays
    with the lengths it was captured with."""

    is_compileable = False

    def __init__(self, layers: int, kv_heads: int, head_dim: int, capacity: int, *,
                 batch: int = 1, tail_tokens: int = 4096, held: str = "e4m3",
                 device: torch.device | str = "cuda") -> None:
        if capacity < 1 or tail_tokens < 1:
            raise ValueError("capacity and tail_tokens must be positive")
        blocks = -(-capacity // BLOCK)
        # A chunk may begin in the middle of a block.
        ring = min(blocks, -(-(tail_tokens + BLOCK - 1) // BLOCK))
        self.capacity = int(capacity)
        self.blocks = ops.KVBlocks(layers=layers, batch=batch, kv_heads=kv_heads,
                                   head_dim=head_dim, capacity_blocks=blocks, ring_blocks=ring,
                                   held=held, device=device)
        self._lengths = [0] * layers

    @classmethod
    def from_config(cls, config, capacity: int, **kwargs) -> "BlockKVCache":
        """A cache for a Hugging Face model config."""
        head_dim = getattr(config, "head_dim", None) or \
            config.hidden_size // config.num_attention_heads
        return cls(config.num_hidden_layers, config.num_key_value_heads, head_dim, capacity,
                   **kwargs)

    # -------------------------------------------------------------- lengths --
    def get_seq_length(self, layer_idx: int = 0) -> int:
        return self._lengths[layer_idx]

    def get_query_offset(self, layer_idx: int | None = 0) -> int:
        return self._lengths[layer_idx or 0]

    def get_mask_sizes(self, query_length: int, layer_idx: int | None = 0) -> tuple[int, int]:
        return self._lengths[layer_idx or 0] + int(query_length), 0

    @property
    def folded_tokens(self) -> int:
        """Tokens held in 8 bits."""
        return self.blocks.folded * BLOCK

    # ---------------------------------------------------------------- calls --
    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """Adds key and value [batch, kv_heads, T, head_dim] (bf16) to
        ``layer``."""
        blocks = self.blocks
        start = self._lengths[layer]
        end = start + key.shape[-2]
        if end > self.capacity:
            raise ValueError(f"the block cache holds {self.capacity} tokens; {end} do not fit")
        if -(-end // BLOCK) - blocks.folded > blocks.ring_blocks:
            raise ValueError(
                f"{end - self.folded_tokens} tokens behind the folded blocks do not fit the tail; "
                "commit what is final, or make the cache with more tail_tokens")
        ops.kv_append(blocks, layer, key, value, start)
        self._lengths[layer] = end

    def attend(self, layer: int, query: torch.Tensor, mask: torch.Tensor | None = None,
               scale: float | None = None) -> torch.Tensor:
        """Attention of query [batch, Hq, Q, head_dim] over the layer's tokens:
        [batch, Q, Hq, head_dim].  mask: bool [batch or 1, 1, Q, M] over the
        last M tokens (those before are admitted), or None for causal."""
        if scale is None:
            scale = self.blocks.head_dim ** -0.5
        return ops.block_attention(self.blocks, layer, query, self._lengths[layer], mask, scale)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int,
               *args, **kwargs) -> tuple[torch.Tensor, torch.Tensor]:
        """DynamicCache.update: appends, and returns the layer's keys and
        values as bf16 tensors (read back whole; ``attend`` is the path
        without that copy)."""
        self.append(layer_idx, key_states, value_states)
        return self.read(layer_idx)

    def read(self, layer: int, start: int = 0, stop: int | None = None
             ) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values of tokens start .. stop - 1 (default: all) as the
        attention sees them, bf16 [batch, kv_heads, tokens, head_dim]."""
        stop = self._lengths[layer] if stop is None else stop
        if not 0 <= start <= stop <= self._lengths[layer]:
            raise ValueError(f"tokens {start} .. {stop} of {self._lengths[layer]}")
        return ops.kv_read(self.blocks, layer, start, stop)

    def scales(self, layer: int) -> torch.Tensor:
        """fp32 [2, batch, kv_heads, folded blocks]: the scales of keys (0)
        and values (1)."""
        b = self.blocks
        if not 0 <= layer < b.layers:
            raise IndexError(f"layer {layer} of a block cache of {b.layers} layers")
        kind, per_layer, head, _ = b.scales.stride()
        return b.scales.as_strided((2, b.batch, b.kv_heads, b.folded),
                                   (kind, head * b.kv_heads, head, 1), layer * per_layer)

    def _length(self) -> int:
        if len(set(self._lengths)) != 1:
            raise RuntimeError("the layers of the block cache differ in length")
        return self._lengths[0]

    def commit(self) -> None:
        """Folds every complete block."""
        count = min(self._lengths) // BLOCK - self.blocks.folded
        if count > 0:
            ops.kv_fold(self.blocks, count)

    def compact(self, base_kv_length: int, positions: Sequence[int]) -> None:
        """Keeps the first ``base_kv_length`` tokens and, of those behind them,
        the ones at ``positions`` (strictly ascending), in every layer."""
        end = self._length()
        if not 0 <= base_kv_length <= end:
            raise ValueError("base_kv_length is not a length of the cache")
        if base_kv_length < self.folded_tokens and tuple(positions) != tuple(range(len(positions))):
            raise ValueError("tokens of folded blocks cannot be moved")
        kept = base_kv_length + len(positions)
        if kept < self.folded_tokens:
            raise ValueError("tokens of folded blocks cannot be dropped")
        ops.kv_compact(self.blocks, base_kv_length, positions, end)
        self._lengths = [kept] * len(self._lengths)

    def crop(self, max_length: int, layer: int | None = None) -> None:
        """Drops the tokens from ``max_length`` on (negative: that many from
        the end), in every layer or in one."""
        if layer is not None and not 0 <= layer < len(self._lengths):
            raise IndexError(f"layer {layer} of a block cache of {len(self._lengths)} layers")
        layers = range(len(self._lengths)) if layer is None else (layer,)
        longest = max(self._lengths[l] for l in layers)
        if max_length < 0:
            max_length = max(0, longest + max_length)
        if max_length < min(longest, self.folded_tokens):
            raise ValueError("tokens of folded blocks cannot be dropped")
        for l in layers:
            self._lengths[l] = min(self._lengths[l], max_length)

    def reset(self) -> None:
        """Empties the cache."""
        self.blocks.folded = 0
        self._lengths = [0] * len(self._lengths)
