"""Greedy step epilogue over the C ABI: the logits, ``_choose`` and the
decode-state update of one step in one kernel launch.

Reference (asrback project paths), on the greedy path (``temperatures`` None):

- ``Transcriber._step`` after the decoder, ``src/asrback/models/whisper.py:949-960``:
  ``logits`` (``:337-342``, the tied ``embed_tokens`` weight), ``_choose``
  (``:962-975``, with the suppress mask) and the state update;
- ``Qwen3ASRTranscriber._step``, ``src/asrback/models/qwen3_asr.py:1189-1201``:
  ``_lm_head``, ``_choose`` (``:1203-1213``) and the state update with several
  EOS ids (``torch.isin``).

bf16 runs the logits on the tensor cores (fp32 sums rounded to bf16, as the
reference's bf16 matmul returns them); float32 runs a SIMT kernel. Sampling
(a positive temperature) is not fused: the reference's graphs cover greedy
steps only, and the patched ``_step`` hands sampled steps to the original.

For a step that ran a tree of drafted tokens per row (speculative decoding, no
counterpart in the reference), :func:`accept_tree` walks each tree along the
tokens the model chose and updates the decode state by as many greedy steps as
the drafts were right, and :func:`greedy_tree_step` does the nodes' logits too.
"""

from __future__ import annotations

import ctypes
import functools
import threading
from collections.abc import Sequence
from typing import NamedTuple

import torch
from torch import Tensor

from . import _native, attention

__all__ = ["greedy_choose", "greedy_step", "AcceptedPath", "accept_tree", "greedy_tree_step",
           "MAX_BATCH"]

MAX_BATCH = 128  # bf16; float32 takes up to 64 rows

_workspaces: dict[int, Tensor] = {}
_lock = threading.Lock()


def _workspace(device: torch.device) -> Tensor:
    index = device.index if device.index is not None else torch.cuda.current_device()
    workspace = _workspaces.get(index)
    if workspace is None:
        with _lock:
            workspace = _workspaces.get(index)
            if workspace is None:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError(
                        "asrback_b200: the step workspace is allocated on a device's first "
                        "greedy step; run one step before capturing it")
                nbytes = _native.load().asrback_greedy_step_workspace_bytes(MAX_BATCH)
                workspace = torch.zeros(nbytes, dtype=torch.uint8,
                                        device=torch.device("cuda", index))
                _workspaces[index] = workspace
    return workspace


def _rows(t: Tensor, name: str) -> Tensor:
    if t.dim() != 2 or t.stride(-1) != 1:
        raise ValueError(f"asrback_b200: {name} must be 2-D with contiguous rows, got "
                         f"{tuple(t.shape)} strides {t.stride()}")
    return t


def _vector(t: Tensor, name: str, dtype: torch.dtype, batch: int) -> Tensor:
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != batch or t.stride(0) != 1:
        raise ValueError(f"asrback_b200: {name} must be a contiguous ({batch},) {dtype} tensor")
    return t


def _launch(hidden: Tensor, weight: Tensor, suppress: Tensor | None, out_token, out_logprob,
            state: dict | None, eos_ids: Sequence[int], workspace: Tensor | None = None) -> None:
    """``workspace``: a zero-filled one of the call's own; by default the device's."""
    hidden = _rows(hidden, "hidden")
    weight = _rows(weight, "weight")
    dtype = attention._dtype_code(hidden, weight)
    batch, width = hidden.shape
    vocab = weight.shape[0]
    if weight.shape[1] != width:
        raise ValueError(f"asrback_b200: weight {tuple(weight.shape)} does not match hidden "
                         f"width {width}")
    if weight.device != hidden.device:
        raise ValueError("asrback_b200: weight must be on the hidden states' device")
    if suppress is not None:
        if suppress.shape != (vocab,) or suppress.dtype not in (torch.bool, torch.uint8) \
                or suppress.stride(0) != 1 or suppress.device != hidden.device:
            raise ValueError(f"asrback_b200: suppress must be a contiguous ({vocab},) bool tensor "
                             "on the hidden states' device")
    eos = [int(e) for e in eos_ids]
    eos_host = (ctypes.c_int64 * max(len(eos), 1))(*eos)
    device = hidden.device
    if workspace is None:
        workspace = _workspace(device)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    if state is None:
        tokens = position = end = finished = sums = generated = None
        tokens_stride = generated_stride = generated_cols = 0
    else:
        tokens = state["tokens"]
        if tokens.dtype != torch.int64 or tokens.shape[0] != batch or tokens.numel() != batch:
            raise ValueError(f"asrback_b200: tokens must be ({batch},) or ({batch}, 1) int64")
        tokens_stride = tokens.stride(0)
        position = _vector(state["position"], "position", torch.int64, batch)
        end = _vector(state["end"], "end", torch.int64, batch)
        finished = _vector(state["finished"], "finished", torch.bool, batch)
        sums = _vector(state["sum_logprobs"], "sum_logprobs", torch.float32, batch)
        generated = state["generated"]
        if generated.dtype != torch.int64 or generated.dim() != 2 or generated.shape[0] != batch \
                or generated.stride(1) != 1:
            raise ValueError(f"asrback_b200: generated must be ({batch}, length) int64 with "
                             "contiguous rows")
        generated_stride, generated_cols = generated.stride(0), generated.shape[1]
        for t in (tokens, position, end, finished, sums, generated):
            if t.device != device:
                raise ValueError("asrback_b200: the decode state must be on the hidden states' "
                                 "device")
    with torch.cuda.device(device):
        _native.call(
            "asrback_greedy_step", dtype, batch, vocab, width,
            hidden.data_ptr(), hidden.stride(0), weight.data_ptr(), weight.stride(0),
            ptr(suppress), ptr(out_token), ptr(out_logprob),
            ptr(tokens), tokens_stride, ptr(position), ptr(end), ptr(finished), ptr(sums),
            ptr(generated), generated_stride, generated_cols,
            eos_host, len(eos),
            workspace.data_ptr(), workspace.numel(), attention._state(device).status.data_ptr(),
            attention._stream(device))


def greedy_choose(hidden: Tensor, weight: Tensor,
                  suppress: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """Greedy ``_choose`` of ``hidden (batch, d) @ weight (vocab, d).T``:
    ``(token int64, logprob float32)``, each ``(batch,)``. Like
    :func:`greedy_step`, it uses the device's one workspace: not for calls, or
    replays of captured ones, that may run at the same time on several streams."""
    batch = hidden.shape[0]
    token = torch.empty(batch, dtype=torch.int64, device=hidden.device)
    logprob = torch.empty(batch, dtype=torch.float32, device=hidden.device)
    _launch(hidden, weight, suppress, token, logprob, None, ())
    return token, logprob


def greedy_step(hidden: Tensor, weight: Tensor, tokens: Tensor, position: Tensor, end: Tensor,
                finished: Tensor, sum_logprobs: Tensor, generated: Tensor,
                eos_ids: Sequence[int], suppress: Tensor | None = None) -> None:
    """One greedy ``_step`` after the decoder, updating the decode state in
    place: ``tokens`` ``(batch,)`` or ``(batch, 1)``, ``position``, ``end``
    (int64), ``finished`` (bool), ``sum_logprobs`` (float32), ``generated``
    ``(batch, length)`` (int64); ``eos_ids`` are host ints (at most 8). All calls
    on a device share one workspace, so that steps (and captured ones' replays)
    have to follow one another on it; :func:`greedy_tree_step` has its own."""
    state = dict(tokens=tokens, position=position, end=end, finished=finished,
                 sum_logprobs=sum_logprobs, generated=generated)
    _launch(hidden, weight, suppress, None, None, state, eos_ids)


class AcceptedPath(NamedTuple):
    """What :func:`accept_tree` accepted: ``path`` ``(B, N)`` int32, the row's
    accepted nodes from node 0 on, then -1; ``counts`` ``(B,)`` int32, their
    number, which is the number of tokens emitted; ``start`` ``(B,)`` int64, the
    cache slot of node 0."""

    path: Tensor
    counts: Tensor
    start: Tensor


@functools.lru_cache(maxsize=64)
def _eos_array(eos_ids: tuple[int, ...]) -> ctypes.Array:
    return (ctypes.c_int64 * len(eos_ids))(*eos_ids)


def _node_rows(t: Tensor, name: str, dtype: torch.dtype, shape: tuple, device) -> tuple:
    """The tensor (which keeps its memory alive) and its row stride."""
    if t.dtype is not dtype or t.shape != shape or t.device != device:
        raise ValueError(f"asrback_b200: {name} must be {shape} {dtype} on {device}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    row, node = t.stride()
    return (t, row) if node == 1 and row >= shape[1] else (t.contiguous(), shape[1])


def accept_tree(tree: attention.DraftTree, drafts: Tensor, chosen: Tensor, logprob: Tensor,
                tokens: Tensor, position: Tensor, end: Tensor, finished: Tensor,
                sum_logprobs: Tensor, generated: Tensor, eos_ids: Sequence[int],
                lengths: Tensor | None = None) -> AcceptedPath:
    """Walks each row's tree from node 0: the token ``chosen`` at a node is
    emitted, and the walk goes on to the lowest child whose draft it is. It ends
    when no child holds it or the row is finished (EOS, or its position at
    ``end``). Every emitted token updates the decode state as
    :func:`greedy_step` does; finished rows, and rows without nodes, stay as they
    are. (A row that the attention skipped has to be one of these: its nodes chose
    from zeros.)

    ``drafts`` ``(B, N)`` int64: the nodes' tokens; ``chosen`` int64 and
    ``logprob`` float32 ``(B, N)``: what :func:`greedy_choose` says of each
    node's hidden state. ``lengths`` ``(B,)`` int64: the cache lengths, advanced
    with ``position``, for a cache whose slots are not its positions. The
    caches' rows are brought in order by :func:`asrback_b200.cache.qwen3_commit_tree`
    or :func:`~asrback_b200.cache.whisper_commit_tree` with the returned path."""
    parents = tree.parents
    batch, nodes = parents.shape
    device = parents.device
    if not parents.is_cuda or parents.dtype is not torch.int32:
        raise ValueError("asrback_b200: tree must be a draft_tree() plan on a CUDA device")
    parents_stride, unit = parents.stride()
    if unit != 1 or 0 < parents_stride < nodes:
        parents, parents_stride = parents.contiguous(), nodes
    counts = _vector(tree.counts, "tree.counts", torch.int32, batch)
    drafts, drafts_stride = _node_rows(drafts, "drafts", torch.int64, (batch, nodes), device)
    chosen, chosen_stride = _node_rows(chosen, "chosen", torch.int64, (batch, nodes), device)
    logprob, logprob_stride = _node_rows(logprob, "logprob", torch.float32, (batch, nodes), device)
    if tokens.dtype is not torch.int64 or tokens.shape[0] != batch or tokens.numel() != batch:
        raise ValueError(f"asrback_b200: tokens must be ({batch},) or ({batch}, 1) int64")
    position = _vector(position, "position", torch.int64, batch)
    end = _vector(end, "end", torch.int64, batch)
    finished = _vector(finished, "finished", torch.bool, batch)
    sums = _vector(sum_logprobs, "sum_logprobs", torch.float32, batch)
    if generated.dtype is not torch.int64 or generated.dim() != 2 or generated.shape[0] != batch \
            or generated.stride(1) != 1:
        raise ValueError(f"asrback_b200: generated must be ({batch}, length) int64 with "
                         "contiguous rows")
    if lengths is not None:
        lengths = _vector(lengths, "lengths", torch.int64, batch)
    for t in (counts, tokens, position, end, finished, sums, generated, lengths):
        if t is not None and t.device != device:
            raise ValueError("asrback_b200: the decode state must be on the tree's device")
    eos_host = _eos_array(tuple(map(int, eos_ids)))
    with attention._on(device):
        path = parents.new_empty((batch, nodes))
        accepted, start = torch.empty_like(counts), torch.empty_like(position)
        columns = generated.shape[1]
        _native.call_packed(
            "asrback_accept_tree", batch, nodes, parents.data_ptr(), parents_stride,
            counts.data_ptr(), drafts.data_ptr(), drafts_stride, chosen.data_ptr(), chosen_stride,
            logprob.data_ptr(), logprob_stride,
            tokens.data_ptr(), tokens.stride(0) if batch > 1 else 1, position.data_ptr(),
            end.data_ptr(), finished.data_ptr(), sums.data_ptr(), generated.data_ptr(),
            generated.stride(0) if batch > 1 else columns, columns,
            0 if lengths is None else lengths.data_ptr(), ctypes.addressof(eos_host),
            len(eos_host), path.data_ptr(), accepted.data_ptr(), start.data_ptr(),
            attention._state(device).status.data_ptr(), attention._stream(device))
    return AcceptedPath(path, accepted, start)


def greedy_tree_step(hidden: Tensor, weight: Tensor, tree: attention.DraftTree, drafts: Tensor,
                     tokens: Tensor, position: Tensor, end: Tensor, finished: Tensor,
                     sum_logprobs: Tensor, generated: Tensor, eos_ids: Sequence[int],
                     suppress: Tensor | None = None, lengths: Tensor | None = None) -> AcceptedPath:
    """A greedy step after the decoder has run a tree of drafted tokens per
    row: every node's logits and choice from ``hidden`` ``(B, N, d)`` (as
    :func:`greedy_choose`, ``MAX_BATCH`` rows per launch), then
    :func:`accept_tree`. The call has a workspace of its own: calls on several
    streams and captured ones replayed side by side do not meet in it."""
    if hidden.dim() != 3 or hidden.shape[:2] != tree.parents.shape:
        raise ValueError(f"asrback_b200: hidden must be (batch, nodes, width) for trees of "
                         f"{tuple(tree.parents.shape)}, got {tuple(hidden.shape)}")
    attention._dtype_code(hidden, weight)
    batch, nodes, width = hidden.shape
    rows = hidden.flatten(0, 1)
    # float32 takes 64 rows, and as many as 200 KB of shared memory hold.
    limit = MAX_BATCH if hidden.dtype == torch.bfloat16 else max(1, min(64, 51200 // width))
    token = torch.empty(batch * nodes, dtype=torch.int64, device=hidden.device)
    logprob = torch.empty(batch * nodes, dtype=torch.float32, device=hidden.device)
    with attention._on(hidden.device):
        nbytes = _native.load().asrback_greedy_step_workspace_bytes(min(limit, batch * nodes))
    # The kernel's tickets begin at zero; the launches of a call follow one another.
    workspace = torch.zeros(nbytes, dtype=torch.uint8, device=hidden.device)
    for first in range(0, batch * nodes, limit):
        part = slice(first, first + limit)
        _launch(rows[part], weight, suppress, token[part], logprob[part], None, (), workspace)
    return accept_tree(tree, drafts, token.view(batch, nodes), logprob.view(batch, nodes), tokens,
                       position, end, finished, sum_logprobs, generated, eos_ids, lengths)
