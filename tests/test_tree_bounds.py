"""The bounds of ``tests/tree_bounds.py`` take what the definition gives, rounded
once, and refuse results with something missing (made on the CPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import test_gpu_tree as gpu
from tests import tree_bounds as bounds

# Of the GPU's tests: family, type, nodes, heads, kv_heads, dim, length, lengths, counts, weights.
LONG = ("qwen3", "bf16", 3, 2, 1, 128, 40000, [39990], [3], True)
ROWS = [0, 200, 64, 301, 77]
WEIGHTS = [
    ("qwen3", "bf16", 1, 16, 8, 128, 333, ROWS, [1, 1, 1, 1, 0], True),
    ("qwen3", "bf16", 8, 16, 8, 128, 333, ROWS, [8, 1, 8, 8, 0], True),
    ("qwen3", "bf16", 5, 6, 2, 64, 333, ROWS, [5, 1, 5, 5, 0], True),
    ("qwen3", "f32", 3, 16, 8, 128, 333, ROWS, [3, 1, 3, 3, 0], True),
    ("whisper", "bf16", 16, 6, 6, 64, 333, ROWS, [16, 1, 16, 16, 0], True),
    ("whisper", "f32", 4, 6, 6, 64, 333, ROWS, [4, 1, 4, 4, 0], True)]
CASES = [LONG, ("qwen3", "bf16", 40, 4, 2, 128, 8192, [8000], [40], False), *WEIGHTS]


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(gpu, "DEV", "cpu")


def make(case):
    family, tag, nodes, heads, kv_heads, dim, length, lengths, counts, weights = case
    x = gpu._inputs(nodes, family, tag, len(lengths), nodes, length, heads, kv_heads, dim, lengths,
                    counts, weights=weights)
    return bounds.coded(x)


def result(x, want):
    """The definition's results as a call gives them."""
    dtype = x["keys"].dtype
    new = [torch.from_numpy(want[n]).to(dtype) for n in ("out", "keys", "values")]
    return [*new, None if x["weights"] is None else torch.from_numpy(want["weights"]).float()]


def without_tile(x, tile):
    """``x`` with the keys of cached tile ``tile`` of row 0 taken out."""
    x = dict(x, lengths=x["lengths"].copy())
    x["lengths"][0] -= bounds.TILE
    for n in ("keys", "values"):
        t = bounds.position_major(x, x[n]).clone()
        t[0, tile * bounds.TILE:-bounds.TILE] = t[0, (tile + 1) * bounds.TILE:].clone()
        x[n] = t.transpose(1, 2) if x["family"] == "whisper" else t
    return x


@pytest.mark.parametrize("case", CASES, ids=lambda case: "-".join(map(str, case[:7])))
def test_results_that_lack_something_are_refused(case):
    x = make(case)
    got = result(x, bounds.definition(x)[0])
    bounds.check(x, got)

    def refused(name, changed):
        again = list(got)
        again[("out", "keys", "values", "weights").index(name)] = changed
        with pytest.raises(AssertionError):
            bounds.check(x, again)

    refused("out", torch.zeros_like(got[0]))
    refused("out", got[0] * 1.05)
    half = dict(x, values=x["values"].clone())
    row = int(np.argmax(x["lengths"] * (x["counts"] > 0)))
    bounds.position_major(x, half["values"])[row, :x["lengths"][row] // 2] = 0
    refused("out", result(x, bounds.definition(half)[0])[0])
    moved = got[1].clone()
    moved[row, x["lengths"][row]] *= 1.05  # a new key
    refused("keys", moved)
    if x["weights"] is None:
        return
    w, before = got[3], x["weights"]
    for b in np.flatnonzero(x["counts"] * x["lengths"]):
        m = x["lengths"][b]
        for first, last in ((0, m), (0, 1), (m - 1, m), (m // 2, m // 2 + 1)):
            kept = w.clone()  # nothing added
            kept[b, 0, first:last] = before[b, 0, first:last]
            refused("weights", kept)
        for factor in (0.98, 1.02):
            refused("weights", torch.where(torch.arange(w.shape[2]) < m, before + factor * (w - before),
                                           w))
        kept = w.clone()
        kept[b, -1, m] += before[b, -1, m]  # added where it is assigned
        refused("weights", kept)


@pytest.mark.parametrize("case,tiles", [(LONG, [0, 1, 100, 311, 500, 623]),
                                        (CASES[1], [0, 60, 124])])
def test_an_output_without_one_tile_is_refused(case, tiles):
    x = make(case)
    got = result(x, bounds.definition(x)[0])
    for tile in tiles:
        lacking = list(got)
        lacking[0] = result(x, bounds.definition(without_tile(x, tile))[0])[0]
        with pytest.raises(AssertionError, match="outputs"):
            bounds.check(x, lacking)


def test_the_older_bound_takes_an_output_of_zeros():
    """Why these bounds: over a long cache the rotated keys' rounding, allowed for on
    every key, is more than the outputs are."""
    x = make(LONG)
    x = dict(x, values=gpu._inputs(3, *LONG[:2], 1, 3, 40000, 2, 1, 128, [39990])["values"])
    want = bounds.definition(x)[0]
    d = 2 * 2.0 ** -7 * want["reach"][..., 1]
    assert (np.abs(want["out"]) < want["mass"] * np.expm1(2 * d)[..., None]).mean() > 0.99
