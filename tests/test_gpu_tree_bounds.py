"""The draft-tree attention within the bounds of ``tests/tree_bounds.py``: a part of
a row left out, a key's weight not gathered or a wrong merge exceeds them
(``tests/test_tree_bounds.py``)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from asrback_b200 import attention, cache, step
from tests import tree_bounds as bounds
from tests.test_gpu_tree import DTYPES, _call, _gpu, _inputs, _tree
from tests.test_tree_bounds import CASES

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status():
    attention.read_status()
    yield
    assert attention.read_status() == 0


def _run(seed, family, tag, nodes, heads, kv_heads, dim, length, lengths, counts, weights, ahead=0,
         code=True):
    x = _inputs(seed, family, tag, len(lengths), nodes, length, heads, kv_heads, dim, lengths, counts,
                ahead=ahead, weights=weights)
    x = bounds.coded(x) if code else x
    bounds.check(x, _call(x))


@pytest.mark.parametrize("case", CASES, ids=lambda case: "-".join(map(str, case[:7])))
def test_cases_whose_faults_would_show(case):
    _run(case[2], *case)


@pytest.mark.parametrize("family,tag,nodes,heads,kv_heads,dim,length,weights", [
    ("qwen3", "f32", 4, 4, 2, 64, 5000, True), ("qwen3", "f32", 20, 2, 1, 128, 3000, False),
    ("qwen3", "bf16", 16, 2, 2, 64, 20000, True), ("qwen3", "bf16", 24, 1, 1, 64, 20000, False),
    ("qwen3", "bf16", 64, 4, 1, 128, 9000, False), ("qwen3", "bf16", 50, 2, 1, 64, 9000, False),
    ("whisper", "bf16", 12, 2, 2, 64, 12000, True), ("whisper", "bf16", 64, 2, 2, 64, 12000, False)])
def test_long_rows(family, tag, nodes, heads, kv_heads, dim, length, weights):
    _run(nodes, family, tag, nodes, heads, kv_heads, dim, length, [length - nodes, length // 3], None,
         weights)


@pytest.mark.parametrize("family,tag,heads,kv_heads,dim,nodes,weights", [
    ("qwen3", "bf16", 16, 8, 128, 1, True), ("qwen3", "bf16", 16, 8, 128, 8, True),
    ("qwen3", "bf16", 16, 8, 128, 16, False), ("qwen3", "bf16", 16, 4, 64, 4, True),
    ("qwen3", "bf16", 16, 4, 64, 5, False), ("qwen3", "bf16", 4, 2, 128, 60, False),
    ("whisper", "bf16", 20, 20, 64, 7, False), ("whisper", "bf16", 20, 20, 64, 16, True),
    ("whisper", "bf16", 4, 4, 64, 25, False), ("whisper", "bf16", 4, 4, 64, 40, False),
    ("qwen3", "f32", 16, 8, 128, 2, True)])
@pytest.mark.parametrize("code", [True, False])
def test_many_items_per_sm(family, tag, heads, kv_heads, dim, nodes, weights, code):
    """Rows of one to many tiles, so that a CTA runs through items and pieces."""
    rows = [700, 447 - nodes, 5, 64, 0, 128, 1, 63, 300, 190, 65, 2]
    lengths = np.minimum(np.array(rows * 4), 704 if family == "qwen3" else 447 - nodes)
    counts = np.random.default_rng(nodes).integers(0, nodes + 1, len(lengths))
    counts[::3] = nodes
    _run(nodes, family, tag, nodes, heads, kv_heads, dim, 768, lengths, counts, weights,
         ahead=13 if family == "qwen3" else 0, code=code)


@pytest.mark.parametrize("tag,nodes,heads", [
    ("bf16", 1, 2), ("bf16", 9, 3), ("bf16", 16, 2), ("bf16", 17, 3), ("bf16", 40, 2), ("bf16", 64, 1),
    ("f32", 1, 2), ("f32", 17, 3)])
def test_heads_of_128_as_they_come(tag, nodes, heads):
    """The form without norm and rotation, with heads of 128."""
    _run(nodes, "whisper", tag, nodes, heads, heads, 128, 500, [400, 0, 129, 500 - nodes],
         [nodes, nodes, (nodes + 1) // 2, nodes], nodes <= 16)


def _inside(t, before, after):
    """A view equal to ``t`` in a larger tensor, ``before``/``after`` longer per
    dimension, and a function that says whether what surrounds it is as it was."""
    big = torch.full([n + a + b for n, a, b in zip(t.shape, before, after)], 3.0, dtype=t.dtype,
                     device=t.device)
    view = big[tuple(slice(a, a + n) for a, n in zip(before, t.shape))]
    view.copy_(t)

    def untouched():
        rest = big.clone()
        rest[tuple(slice(a, a + n) for a, n in zip(before, t.shape))] = 3.0
        return bool((rest == 3.0).all())

    return view, untouched


@pytest.mark.parametrize("family,tag,heads,kv_heads,dim,nodes,weights", [
    ("qwen3", "bf16", 4, 2, 128, 5, True), ("qwen3", "bf16", 4, 2, 64, 16, False),
    ("qwen3", "bf16", 4, 2, 128, 33, False), ("qwen3", "f32", 4, 2, 64, 5, True),
    ("whisper", "bf16", 3, 3, 64, 9, True), ("whisper", "bf16", 3, 3, 64, 64, False),
    ("whisper", "f32", 3, 3, 128, 7, True)])
def test_views_of_larger_caches(family, tag, heads, kv_heads, dim, nodes, weights):
    """Caches and weights narrowed to a bucket, a share of the heads and of the
    rows; projections within wider rows. Nothing around them is written."""
    x = bounds.coded(_inputs(nodes, family, tag, 3, nodes, 300, heads, kv_heads, dim,
                             [300 - nodes, 0, 131], [nodes, nodes, (nodes + 1) // 2],
                             weights=weights))
    around = []
    held = dict(x)
    for n in ("keys", "values"):
        held[n], check = _inside(x[n], (1, 2, 3, 0), (0, 1, 2, 0))
        around.append(check)
    if weights:
        held["weights"], check = _inside(x["weights"], (1, 1, 7), (1, 0, 2))
        around.append(check)
    if family == "qwen3":
        held["qkv"], _ = _inside(x["qkv"], (0, 1, 64), (1, 0, 64))
    at = {n: _gpu(x[n], torch.int64) for n in ("lengths", "positions")}
    tree = _tree(x["parents"], x["counts"])
    if family == "qwen3":
        out = attention.qwen3_attention_tree(
            held["qkv"], x["wq"], x["wk"], 1e-6, x["cos"], x["sin"], at["positions"], tree,
            held["keys"], held["values"], heads, kv_heads, lengths=at["lengths"],
            weights=held["weights"])
    else:
        out = attention.whisper_self_attention_tree(
            x["q"], x["k"], x["v"], held["keys"], held["values"], at["lengths"], tree,
            weights=held["weights"])
    bounds.check(x, (out, *(bounds.position_major(x, held[n]) for n in ("keys", "values")),
                     held["weights"]))
    assert all(check() for check in around)


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("heads_first,length,budget,dim", [
    (False, 300, 100, 128), (True, 300, 100, 64), (False, 5000, 1200, 64), (True, 2100, 2000, 128)])
def test_moves_in_views_of_larger_caches(tag, heads_first, length, budget, dim):
    """A commit and an eviction of all layers, whose caches lie row by row (the
    layers inside), narrowed: as in tensors of their own."""
    rng = np.random.default_rng(length)
    layers, batch, heads, nodes = 3, 4, 2, 9
    shape = (batch, layers, heads, length, dim) if heads_first else (batch, layers, length, heads, dim)
    own = [_gpu(rng.standard_normal(shape), DTYPES[tag]) for _ in range(2)]
    own.append(_gpu(rng.random((batch, layers, heads, length)), torch.float32))
    views, around = zip(*(_inside(t, (1, 1, 2, 1) + (0,) * (t.dim() - 4), (0, 1, 0, 3) + (0,) * (t.dim() - 4))
                          for t in own))
    counts = np.array([4, 0, 9, 1])
    path = np.full((batch, nodes), -1)
    for b, n in enumerate(counts):
        path[b, :n] = np.sort(rng.permutation(nodes)[:n])
    accepted = step.AcceptedPath(_gpu(path, torch.int32), _gpu(counts, torch.int32),
                                 _gpu(np.array([length - nodes, 5, 17, 0]), torch.int64))
    lengths = _gpu(np.array([length, budget, budget + 1, length - 1]), torch.int64)
    commit, evict = ((cache.whisper_commit_tree, cache.whisper_evict) if heads_first else
                     (cache.qwen3_commit_tree, cache.qwen3_evict))
    results = []
    for tensors in (own, views):
        keys, values, weights = (t.transpose(0, 1) for t in tensors)
        keys, values, weights = ((keys, values, weights) if tensors is views else
                                 (t.contiguous() for t in (keys, values, weights)))
        commit(keys, values, accepted, weights=weights)
        results.append((keys, values, weights, *evict(keys, values, weights, lengths, budget, 2, 5)))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert all(check() for check in around)
