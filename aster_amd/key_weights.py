"""Softmax weights gathered per key of a paged cache, by which tokens are evicted from it.

A :class:`KeyWeights` holds, for each of ``rows`` sequences, the weight that every key of
every layer and KV head has gathered so far; ``PagedKVCache.paged_attention_weights`` adds a
step's weights to it and ``PagedKVCache.evict`` keeps the heaviest keys. Rows belong to
sequences, not to pages: sequences that share prefix pages gather apart. The reference keeps
every token (no counterpart in src/aster/inference/state.py).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _native

_ALIGN = 16  # a row's capacity is a multiple of the block size


@dataclass(frozen=True)
class EvictedTokens:
    """What an eviction left: ``kept`` int32 ``[S, L, Hkv, keep]``, the positions (before it)
    of the tokens that stay, ascending, -1 behind the last; ``lengths`` int32 ``[S]``."""

    kept: torch.Tensor
    lengths: torch.Tensor


class KeyWeightRows:
    """The rows of a batch's sequences, in batch order (``KeyWeights.select``)."""

    def __init__(self, weights, rows):
        rows = [int(r) if isinstance(r, int) and not isinstance(r, bool) else None for r in rows]
        if any(r is None or not 0 <= r < weights.rows for r in rows):
            raise ValueError(f"Key weight rows are ints in [0, {weights.rows})")
        if len(set(rows)) != len(rows):
            raise ValueError("Key weight rows of one batch must be distinct")
        self.weights, self.rows = weights, tuple(rows)
        self.table = torch.tensor(rows, dtype=torch.int32).to(weights.values.device)
        v = weights.values
        self._descs = [_native.KeyWeightsDesc(
            values=v[0, layer].data_ptr(), row_stride=v.stride(0), head_stride=v.stride(2),
            rows=self.table.data_ptr(), num_rows=weights.rows, capacity=weights.capacity)
            for layer in range(v.shape[1])]

    def __len__(self):
        return len(self.rows)

    def desc(self, layer):
        return self._descs[layer]


class KeyWeights:
    """Gathered weights ``values`` fp32 ``[rows, num_layers, num_kv_heads, capacity]`` of a
    :class:`PagedKVCache`'s keys, all zero at first. ``capacity``: the most tokens a sequence
    may have (rounded up to whole pages). A row may go to another sequence without being
    cleared: a call sets the weights of its own new tokens and adds to those before them. So a
    fork's row begins as a copy of its parent's values, and rows do not travel with archived
    sequences."""

    def __init__(self, cache, *, rows, capacity):
        if any(type(v) is not int or v < 1 for v in (rows, capacity)):
            raise ValueError("Key weight rows and capacity must be positive integers")
        self.rows, self.capacity = rows, -(-capacity // _ALIGN) * _ALIGN
        self.layout = (cache.num_layers, cache.num_kv_heads, cache.device)
        self.values = torch.zeros((rows, cache.num_layers, cache.num_kv_heads, self.capacity),
                                  dtype=torch.float32, device=cache.device)

    def select(self, rows):
        """The rows of a batch's sequences, each at most once."""
        return KeyWeightRows(self, rows)

    def check(self, cache, selected, num_seqs, what="key_weights"):
        """``selected`` as rows of a :class:`KeyWeights` that fits ``cache`` and the batch."""
        if not isinstance(selected, KeyWeightRows) or selected.weights is not self:
            raise ValueError(f"{what} must be rows selected from a KeyWeights")
        if self.layout != (cache.num_layers, cache.num_kv_heads, cache.device):
            raise ValueError(f"{what} were made for another cache layout")
        if len(selected) != num_seqs:
            raise ValueError(f"{what} must have one row per sequence")


def check_budget(keep, recent, sinks):
    """The tokens an eviction keeps, and those of them that stay for their place."""
    if any(type(v) is not int or v < 0 for v in (keep, recent, sinks)) or keep < 1 \
            or sinks + recent > keep:
        raise ValueError("keep must be a positive int that holds the sinks and recent tokens")


def require_rows(cache, selected, num_seqs, what="key_weights"):
    if not isinstance(selected, KeyWeightRows):
        raise ValueError(f"{what} must be rows selected from a KeyWeights")
    selected.weights.check(cache, selected, num_seqs, what)
    return selected.weights
