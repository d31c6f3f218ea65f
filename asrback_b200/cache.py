"""Cache rows moved in place over the C ABI: the commit of a draft tree's
accepted nodes and the eviction of keys by accumulated attention weight.

Both have no counterpart in the reference, whose caches only grow. They take
its cache tensors, Qwen3's position-major ``(B, L, kv_heads, D)`` or Whisper's
head-major ``(B, H, L, D)``, one layer's or all layers' with a leading
dimension, and move rows without a second copy of the cache.
"""

from __future__ import annotations

import torch
from torch import Tensor

from . import _native, attention, step

__all__ = ["qwen3_commit_tree", "whisper_commit_tree", "qwen3_evict", "whisper_evict"]


def _caches(keys: Tensor, values: Tensor, heads_first: bool) -> tuple[tuple, tuple, int]:
    """The caches' sizes (layers, batch, heads, head_dim, length) and strides
    (layer, row, position, head; a dimension of one has none), and their dtype."""
    dtype = attention._dtype_code(keys, values)
    size, stride = keys.shape, keys.stride()
    if len(size) not in (4, 5) or values.shape != size or values.stride() != stride:
        raise ValueError("asrback_b200: keys and values must be caches of one shape and layout, "
                         "one layer's (4-D) or all layers' (5-D)")
    if stride[-1] != 1 or values.device != keys.device:
        raise ValueError("asrback_b200: the caches must be on one device, head_dim with unit stride")
    if len(size) == 4:
        size, stride = (1, *size), (0, *stride)
    layers, batch, length, heads, head_dim = size
    layer, row, position, head, _ = stride
    if heads_first:
        length, heads, position, head = heads, length, head, position
    return ((layers, batch, heads, head_dim, length),
            (layer if layers > 1 else 0, row if batch > 1 else 0,
             position if length > 1 else head_dim, head if heads > 1 else head_dim), dtype)


def _weights(weights: Tensor, keys: Tensor, sizes: tuple) -> tuple:
    """Pointer and strides (layer, row, head) of the accumulated weights."""
    layers, batch, heads, _, length = sizes
    shape = (batch, heads, length) if keys.dim() == 4 else (layers, batch, heads, length)
    if keys.dim() == 4 and weights.dim() == 4:
        shape = (1, *shape)
    if weights.dtype is not torch.float32 or weights.shape != shape \
            or weights.device != keys.device or (length > 1 and weights.stride(-1) != 1):
        raise ValueError("asrback_b200: weights must be ([layers,] batch, heads, length) float32 "
                         "with unit last stride, on the caches' device")
    stride = weights.stride()[:-1]
    return (weights.data_ptr(), *(stride if len(stride) == 3 else (0, *stride)))


def _commit(keys: Tensor, values: Tensor, accepted: step.AcceptedPath, weights: Tensor | None,
            heads_first: bool) -> None:
    sizes, strides, dtype = _caches(keys, values, heads_first)
    layers, batch, heads, head_dim, length = sizes
    device, nodes = keys.device, accepted.path.shape[1]
    path = attention._int_rows(accepted.path, "path", torch.int32, (batch, nodes), device)
    counts = attention._int_rows(accepted.counts, "counts", torch.int32, (batch,), device)
    start = attention._int_rows(accepted.start, "start", torch.int64, (batch,), device)
    w = (0, 0, 0, 0) if weights is None else _weights(weights, keys, sizes)
    with attention._on(device):
        _native.call_packed(
            "asrback_commit_tree", dtype, layers, batch, nodes, heads, head_dim, length,
            keys.data_ptr(), values.data_ptr(), *strides, *w, path.data_ptr(), counts.data_ptr(),
            start.data_ptr(), attention._state(device).status.data_ptr(),
            attention._stream(device))


def _evict(keys: Tensor, values: Tensor, weights: Tensor, lengths: Tensor, budget: int, sink: int,
           recent: int, heads_first: bool) -> tuple[Tensor, Tensor]:
    sizes, strides, dtype = _caches(keys, values, heads_first)
    layers, batch, heads, head_dim, length = sizes
    device = keys.device
    w = _weights(weights, keys, sizes)
    lengths = attention._int_rows(lengths, "lengths", torch.int64, (batch,), device)
    if not 1 <= budget <= length or sink < 0 or recent < 0 or sink + recent > budget:
        raise ValueError(f"asrback_b200: budget must be in [1, {length}] and hold sink + recent, "
                         f"got {budget}, {sink}, {recent}")
    with attention._on(device):
        new_lengths = torch.empty(batch, dtype=torch.int64, device=device)
        shape = (batch, heads, budget) if keys.dim() == 4 else (layers, batch, heads, budget)
        kept = torch.empty(shape, dtype=torch.int32, device=device)
        _native.call_packed(
            "asrback_evict", dtype, layers, batch, heads, head_dim, length, keys.data_ptr(),
            values.data_ptr(), *strides, *w, lengths.data_ptr(), budget, sink, recent,
            new_lengths.data_ptr(), kept.data_ptr(), attention._state(device).status.data_ptr(),
            attention._stream(device))
    return new_lengths, kept


def qwen3_commit_tree(keys: Tensor, values: Tensor, accepted: step.AcceptedPath,
                      weights: Tensor | None = None) -> None:
    """Brings the accepted nodes' rows of Qwen3 caches ``([layers,] B, L,
    kv_heads, D)`` in order, in place: row ``start + path[k]`` moves to ``start
    + k`` (``accepted`` from :func:`asrback_b200.step.accept_tree`). ``weights``
    ``([layers,] B, kv_heads, L)`` float32 move along, with all that a call over
    the tree put in them: rejected nodes' shares too."""
    _commit(keys, values, accepted, weights, False)


def whisper_commit_tree(keys: Tensor, values: Tensor, accepted: step.AcceptedPath,
                        weights: Tensor | None = None) -> None:
    """As :func:`qwen3_commit_tree`, for Whisper caches ``([layers,] B, H, L,
    D)``."""
    _commit(keys, values, accepted, weights, True)


def qwen3_evict(keys: Tensor, values: Tensor, weights: Tensor, lengths: Tensor, budget: int,
                sink: int = 0, recent: int = 0) -> tuple[Tensor, Tensor]:
    """Evicts keys by accumulated attention weight from Qwen3 caches
    ``([layers,] B, L, kv_heads, D)``, in place. Per layer, row and head, a row
    with more than ``budget`` keys (``lengths`` ``(B,)`` int64) keeps its first
    ``sink`` slots, its last ``recent`` slots and, of the others, those with the
    largest ``weights`` ``([layers,] B, kv_heads, L)`` float32 (the lower slot on
    ties; NaN counts as -inf). Kept keys, values and weights move to the front in
    their old order. Returns the new lengths ``min(lengths, budget)`` and the
    kept keys' old slots ``([layers,] B, kv_heads, budget)`` int32, -1 behind a
    shorter row's.

    The weights come from :func:`asrback_b200.attention.qwen3_attention_tree`,
    which then takes the new lengths beside the unchanged positions. (From calls
    over accepted nodes: single tokens, prompts, accepted paths.)"""
    return _evict(keys, values, weights, lengths, budget, sink, recent, False)


def whisper_evict(keys: Tensor, values: Tensor, weights: Tensor, lengths: Tensor, budget: int,
                  sink: int = 0, recent: int = 0) -> tuple[Tensor, Tensor]:
    """As :func:`qwen3_evict`, for Whisper caches ``([layers,] B, H, L, D)``."""
    return _evict(keys, values, weights, lengths, budget, sink, recent, True)
