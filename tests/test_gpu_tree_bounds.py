"""The draft-tree attention within the bounds of ``tests/tree_bounds.py``: a part of
a row left out, a key's weight not gathered or a wrong merge exceeds them
(``tests/test_tree_bounds.py``)."""

from __future__ import annotations

import numpy as np
import pytest

from asrback_b200 import attention
from tests import tree_bounds as bounds
from tests.test_gpu_tree import _call, _inputs
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
