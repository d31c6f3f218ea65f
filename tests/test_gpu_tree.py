"""Draft-tree attention, acceptance, commit and eviction on the GPU against the
float64 oracle (``oracle/tree.py``).

Tolerances. A bf16 output is rounded once (2^-8 of it at most, half a step) and
its probabilities once before the second product (2^-8 of the sum of |p v|, the
``mass``). A rotated q is taken in two bf16 parts (2^-17). A rotated k that
falls on the other side of a rounding border in float32 than in float64 moves
one element by a step (2^-7): two such elements per key are allowed for, each
worth 2^-7 * max |q k| in its score. Float32 sums of n terms add n * 2^-24 of the terms' sum. A score
off by d moves a probability by the factor e^(2 d) at most (once itself, once
in the sum).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from asrback_b200 import _native, attention, cache, step
from asrback_b200.transcription import CapturedGraph
from oracle import attention as oracle_attention
from oracle import tree as oracle

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def clean_status():
    attention.read_status()
    yield


def _parents(rng, batch, nodes, shape):
    parents = np.full((batch, nodes), -1)
    for i in range(1, nodes):
        parents[:, i] = (i - 1 if shape == "chain" else 0 if shape == "star" else
                         rng.integers(-1, i, batch) if shape == "forest" else
                         rng.integers(max(0, i - 5), i, batch))
    return parents


def _gpu(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV).to(dtype)


def _np(t):
    return t.detach().double().cpu().numpy()


def _tree(parents, counts):
    return attention.draft_tree(_gpu(parents, torch.int32), _gpu(counts, torch.int32))


def _inputs(seed, family, tag, batch, nodes, length, heads, kv_heads, dim, lengths, counts=None,
            shape="tree", ahead=0, weights=False):
    rng = np.random.default_rng(seed)
    dtype = DTYPES[tag]
    draw = lambda *s: _gpu(rng.standard_normal(s), dtype)  # noqa: E731
    counts = np.full(batch, nodes) if counts is None else np.asarray(counts)
    x = dict(family=family, tag=tag, heads=heads, kv_heads=kv_heads, dim=dim,
             parents=_parents(rng, batch, nodes, shape), counts=counts,
             lengths=np.asarray(lengths), positions=np.asarray(lengths) + ahead)
    x["keys"], x["values"] = draw(batch, length, kv_heads, dim), draw(batch, length, kv_heads, dim)
    if family == "whisper":
        x["keys"], x["values"] = (t.transpose(1, 2).contiguous() for t in (x["keys"], x["values"]))
        # _split_heads views of one fused projection, whose rows are wider.
        fused = draw(batch, nodes, 3, heads, dim)
        x["q"], x["k"], x["v"] = (fused[:, :, i].transpose(1, 2) for i in range(3))
    else:
        x["qkv"] = draw(batch, nodes, (heads + 2 * kv_heads) * dim) * 2
        x["wq"], x["wk"] = draw(dim) * 0.1 + 1, draw(dim) * 0.1 + 1
        cos, sin = oracle_attention.rope_tables(1e6, dim, length + ahead + nodes)
        x["cos"], x["sin"] = _gpu(cos, dtype), _gpu(sin, dtype)
    x["weights"] = _gpu(rng.random((batch, kv_heads, length)), torch.float32) if weights else None
    return x


def _call(x, tree=None):
    """The op on clones of the caches: out, keys, values (B, L, KVH, D), weights."""
    tree = _tree(x["parents"], x["counts"]) if tree is None else tree
    keys, values = x["keys"].clone(), x["values"].clone()
    weights = None if x["weights"] is None else x["weights"].clone()
    lengths, positions = _gpu(x["lengths"], torch.int64), _gpu(x["positions"], torch.int64)
    if x["family"] == "whisper":
        out = attention.whisper_self_attention_tree(x["q"], x["k"], x["v"], keys, values, lengths,
                                                    tree, weights=weights)
        keys, values = keys.transpose(1, 2), values.transpose(1, 2)
    else:
        out = attention.qwen3_attention_tree(
            x["qkv"], x["wq"], x["wk"], 1e-6, x["cos"], x["sin"], positions, tree, keys, values,
            x["heads"], x["kv_heads"], lengths=lengths, weights=weights)
    return out, keys, values, weights


def _want(x):
    above, depths = oracle.plan(x["parents"], x["counts"])
    heads, kv_heads, dim = x["heads"], x["kv_heads"], x["dim"]
    rotary = None
    if x["family"] == "whisper":
        q, k, v = (_np(x[n]).transpose(0, 2, 1, 3) for n in "qkv")
        keys, values = _np(x["keys"]).transpose(0, 2, 1, 3), _np(x["values"]).transpose(0, 2, 1, 3)
    else:
        qkv = _np(x["qkv"]).reshape(*x["qkv"].shape[:2], -1, dim)
        q, k, v = np.split(qkv, (heads, heads + kv_heads), 2)
        keys, values = _np(x["keys"]), _np(x["values"])
        rotary = (_np(x["wq"]), _np(x["wk"]), 1e-6, _np(x["cos"]), _np(x["sin"]), x["positions"],
                  depths)
    weights = None if x["weights"] is None else _np(x["weights"])
    return oracle.tree_attention(q, k, v, keys, values, x["lengths"], above, x["counts"],
                                 dim ** -0.5, weights, rotary, x["tag"] == "bf16")


def _check(x, got, want):
    out, keys, values, weights = got
    bf16, dim = x["tag"] == "bf16", x["dim"]
    full, top = want["reach"][..., 0], want["reach"][..., 1]
    n_keys = int(x["lengths"].max()) + 64
    d = dim * 2.0 ** -24 * full + 2.0 ** -22 * (1 + full)
    if bf16 and x["family"] == "qwen3":
        d = d + 2 * 2.0 ** -7 * top + 2.0 ** -17 * full
    shift = np.expm1(2 * d)
    rounding = 2.0 ** -8 if bf16 else 2.0 ** -24
    tol = rounding * np.abs(want["out"]) + want["mass"] * (
        (2.0 ** -8 if bf16 else 0.0) + shift[..., None] + n_keys * 2.0 ** -24)
    np.testing.assert_array_less(np.abs(_np(out).reshape(want["out"].shape) - want["out"]),
                                 tol + 1e-30)
    # New rows: one rounding of a float32 norm and rotation. Others: untouched.
    k_tol = (2.0 ** -7 if bf16 else 2.0 ** -20) * np.abs(want["keys"]) + 1e-6
    assert (np.abs(_np(keys) - want["keys"]) <= k_tol).all()
    np.testing.assert_array_equal(_np(values), want["values"])
    before = x["keys"].transpose(1, 2) if x["family"] == "whisper" else x["keys"]
    for b, (n, m) in enumerate(zip(x["counts"], x["lengths"])):
        assert torch.equal(keys[b, :m], before[b, :m])
        assert torch.equal(keys[b, m + n:], before[b, m + n:])
    if weights is not None:
        gained = want["weights"] - _np(x["weights"])
        rows = x["counts"].max() * x["heads"] // x["kv_heads"]
        slack = shift.max() * np.maximum(np.abs(gained), 0) + rows * 2.0 ** -23 \
            * (np.abs(gained) + np.abs(want["weights"]))
        slack = np.where(np.arange(gained.shape[2]) >= x["lengths"].min(),
                         slack + shift.max() * rows, slack)
        np.testing.assert_array_less(np.abs(_np(weights) - want["weights"]), slack + 1e-30)
    assert attention.read_status() == 0


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("nodes,shape", [(1, "chain"), (5, "forest"), (16, "tree"), (17, "star"),
                                         (64, "chain"), (33, "tree")])
def test_qwen3_trees(tag, nodes, shape):
    """Lengths around the 64-key tile, an empty cache, a full one; rows with
    fewer nodes and one with none."""
    length = 64 + 3 * 64
    lengths = [0, 63, 64, 65, length - nodes, 130, 1]
    counts = [nodes, nodes, (nodes + 1) // 2, nodes, nodes, 0, 1]
    x = _inputs(nodes, "qwen3", tag, 7, nodes, length, 16, 8, 128, lengths, counts, shape)
    _check(x, _call(x), _want(x))


@pytest.mark.parametrize("heads,kv_heads,dim,nodes", [
    (8, 8, 128, 7), (4, 1, 64, 3), (12, 2, 64, 11), (32, 4, 128, 2), (16, 1, 128, 64), (1, 1, 64, 1)])
def test_qwen3_head_layouts(heads, kv_heads, dim, nodes):
    x = _inputs(heads, "qwen3", "bf16", 2, nodes, 200, heads, kv_heads, dim, [100, 136], ahead=23)
    _check(x, _call(x), _want(x))


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("batch,nodes,heads", [(1, 1, 20), (3, 8, 6), (2, 20, 20), (1, 64, 6)])
def test_whisper_trees(tag, batch, nodes, heads):
    lengths = [448 - nodes, 0, 129][:batch]
    x = _inputs(batch, "whisper", tag, batch, nodes, 448, heads, heads, 64, lengths)
    _check(x, _call(x), _want(x))


@pytest.mark.parametrize("family,tag,nodes,heads,kv_heads,dim", [
    ("qwen3", "bf16", 1, 16, 8, 128), ("qwen3", "bf16", 8, 16, 8, 128),
    ("qwen3", "bf16", 5, 6, 2, 64), ("qwen3", "f32", 3, 16, 8, 128),
    ("whisper", "bf16", 16, 6, 6, 64), ("whisper", "f32", 4, 6, 6, 64)])
def test_weights(family, tag, nodes, heads, kv_heads, dim):
    lengths, counts = [0, 200, 64, 301, 77], [nodes, 1, nodes, nodes, 0]
    x = _inputs(nodes, family, tag, 5, nodes, 333, heads, kv_heads, dim, lengths, counts,
                ahead=11 if family == "qwen3" else 0, weights=True)
    _check(x, _call(x), _want(x))


@pytest.mark.parametrize("family,tag,heads,kv_heads,dim,nodes,weights", [
    ("qwen3", "bf16", 16, 8, 128, 1, True), ("qwen3", "bf16", 16, 8, 128, 16, False),
    ("qwen3", "bf16", 16, 4, 64, 5, False), ("qwen3", "bf16", 16, 8, 128, 60, False),
    ("whisper", "bf16", 20, 20, 64, 7, False), ("whisper", "bf16", 20, 20, 64, 16, True),
    ("whisper", "bf16", 20, 20, 64, 25, False), ("whisper", "bf16", 20, 20, 64, 40, False),
    ("qwen3", "f32", 16, 8, 128, 2, True)])
def test_many_items_per_sm(family, tag, heads, kv_heads, dim, nodes, weights):
    """Rows of one to many tiles, some empty, so that a CTA runs through many
    items and pieces of items; twice, back to back, with the same results."""
    rows = [700, 447 - nodes, 5, 64, 0, 128, 1, 63, 300, 190, 65, 2]
    lengths = np.minimum(np.array(rows * 6), 704 if family == "qwen3" else 447 - nodes)
    rng = np.random.default_rng(nodes)
    counts = rng.integers(0, nodes + 1, len(lengths))
    counts[::3] = nodes
    x = _inputs(nodes, family, tag, len(lengths), nodes, 768, heads, kv_heads, dim, lengths, counts,
                weights=weights)
    got = [_call(x) for _ in range(4)]
    _check(x, got[0], _want(x))
    for again in got[1:]:
        assert all(a is None or torch.equal(a, b) for a, b in zip(again, got[0]))


def test_long_cache_splits_over_the_gpu():
    """One row, one head: every CTA takes a piece of one item."""
    x = _inputs(0, "qwen3", "bf16", 1, 3, 40000, 2, 1, 128, [39990], weights=True)
    _check(x, _call(x), _want(x))


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements, the row at its end."""
    length = 33000
    shape = (64, length, 8, 128)
    if torch.cuda.mem_get_info()[0] < 3 * 4 * np.prod(shape, dtype=np.int64):
        pytest.skip("needs 26 GB")
    gen = torch.Generator(device=DEV).manual_seed(0)
    keys = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
    values = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
    keys[-1] = torch.randn(shape[1:], generator=gen, device=DEV)
    values[-1] = torch.randn(shape[1:], generator=gen, device=DEV)
    lengths = np.full(64, 5)
    lengths[-1] = length - 2
    small = _inputs(1, "qwen3", "bf16", 64, 2, 64, 16, 8, 128, np.full(64, 5))
    x = dict(small, lengths=lengths, positions=lengths)
    cos, sin = oracle_attention.rope_tables(1e6, 128, length)
    x["cos"], x["sin"] = _gpu(cos, torch.bfloat16), _gpu(sin, torch.bfloat16)
    tree = _tree(x["parents"], x["counts"])
    at = _gpu(lengths, torch.int64)
    out = attention.qwen3_attention_tree(x["qkv"], x["wq"], x["wk"], 1e-6, x["cos"], x["sin"], at,
                                         tree, keys, values, 16, 8)
    one = dict(x, lengths=lengths[-1:], positions=lengths[-1:], counts=x["counts"][-1:],
               parents=x["parents"][-1:], qkv=x["qkv"][-1:], keys=keys[-1:], values=values[-1:])
    want = _want(one)
    _check(dict(one, keys=keys[-1:].clone(), values=values[-1:].clone()),
           (out[-1:], keys[-1:], values[-1:], None), want)
    # Eviction and commit reach the same far rows.
    weights = torch.rand((64, 8, length), generator=gen, device=DEV)
    row, slots = keys[-1].clone(), None
    new, kept = cache.qwen3_evict(keys, values, weights, at, 1000, recent=10)
    assert new.tolist() == [5] * 63 + [1000]
    for h in range(8):
        slots = kept[-1, h].long()
        assert torch.equal(keys[-1, :1000, h], row[slots, h])


def test_results_repeat():
    x = _inputs(3, "qwen3", "bf16", 5, 9, 1000, 16, 8, 128, [900, 100, 3, 517, 640], weights=False)
    first = _call(x)
    for _ in range(5):
        again = _call(x)
        assert all(torch.equal(a, b) for a, b in zip(first[:3], again[:3]))


@pytest.mark.parametrize("tag", ["bf16", "f32"])
def test_masked_places_do_not_matter(tag):
    """NaN and infinities behind the row, in padding nodes and in nodes that a
    node does not see."""
    x = _inputs(5, "qwen3", tag, 3, 20, 300, 16, 8, 128, [200, 0, 65], [20, 13, 0])
    clean = _call(x)
    dirty = dict(x, keys=x["keys"].clone(), values=x["values"].clone(), qkv=x["qkv"].clone())
    for b, (n, m) in enumerate(zip(x["counts"], x["lengths"])):
        dirty["keys"][b, m:], dirty["values"][b, m:] = float("nan"), float("inf")
        dirty["qkv"][b, n:] = float("nan")
    got = _call(dirty)
    assert torch.equal(got[0], clean[0])
    # The last node of row 0 is no one's ancestor: its value reaches only itself.
    width = x["dim"] * x["kv_heads"]
    dirty["qkv"][0, 19, -width:] = float("inf")
    dirty["qkv"][0, 18, -width:] = float("nan")
    above, _ = oracle.plan(x["parents"], x["counts"])
    got = _call(dirty)[0]
    sees = above[0][:, 18] | above[0][:, 19]
    assert not torch.isfinite(got[0, 19]).any() and torch.isnan(got[0, 18]).all()
    d = (got[0].float() - clean[0][0].float())[torch.from_numpy(~sees)]
    # The products are summed in another order, with the same roundings.
    mass = _want(x)["mass"][0][~sees].reshape(d.shape)
    assert (d.abs().cpu().numpy() <= mass * 2.0 ** (-8 if tag == "bf16" else -20)).all()


@pytest.mark.parametrize("heads,kv_heads,dim,nodes", [
    (4, 2, 64, 16), (16, 8, 128, 8), (2, 2, 64, 7), (8, 1, 128, 16), (6, 2, 64, 21)])
def test_an_unseen_value_does_not_matter(heads, kv_heads, dim, nodes):
    """The last two nodes' values are infinite and NaN: whoever does not see them
    is as without."""
    x = _inputs(dim + nodes, "qwen3", "bf16", 2, nodes, 300, heads, kv_heads, dim, [190, 0])
    clean, mass = _call(x)[0], _want(x)["mass"]
    dirty = dict(x, qkv=x["qkv"].clone())
    dirty["qkv"][:, nodes - 1, -dim * kv_heads:] = float("inf")
    dirty["qkv"][:, nodes - 2, -dim * kv_heads:] = float("nan")
    got = _call(dirty)[0]
    above, _ = oracle.plan(x["parents"], x["counts"])
    sees = above[:, :, nodes - 1] | above[:, :, nodes - 2]
    assert not torch.isfinite(got[torch.from_numpy(sees)]).any()
    d = (got.float() - clean.float())[torch.from_numpy(~sees)].abs().cpu().numpy()
    # The products are summed in another order, with the same roundings.
    assert (d <= mass[~sees].reshape(d.shape) * 2.0 ** -8).all()


@pytest.mark.parametrize("family,heads,kv_heads,dim", [
    ("whisper", 3, 3, 64), ("qwen3", 4, 2, 64), ("qwen3", 2, 2, 128)])
@pytest.mark.parametrize("nodes", [9, 15, 16, 17, 31, 32, 33, 49])
def test_blocks_of_every_size(family, heads, kv_heads, dim, nodes):
    x = _inputs(nodes, family, "bf16", 3, nodes, 200, heads, kv_heads, dim, [128, 200 - nodes, 3],
                [nodes, nodes, nodes - 2])
    _check(x, _call(x), _want(x))


def test_rows_that_do_not_fit_are_skipped():
    x = _inputs(6, "qwen3", "bf16", 6, 4, 100, 16, 8, 128, [50, 97, -1, 96, 1 << 40, 10])
    x["positions"] = np.array([50, 97, 3, 96, 5, 1 << 33])
    got = _call(x)
    assert attention.read_status() == _native.STATUS_POSITION
    good = [0, 3]
    for b in set(range(6)) - set(good):
        assert not got[0][b].any()
        assert torch.equal(got[1][b], x["keys"][b]) and torch.equal(got[2][b], x["values"][b])
    part = {n: x[n][good] for n in ("qkv", "keys", "values", "parents", "counts", "lengths",
                                    "positions")}
    _check(dict(x, **part), tuple(t[good] for t in got[:3]) + (None,), _want(dict(x, **part)))


def test_invalid_trees_are_flagged():
    parents = np.array([[-1, 0, 1], [-1, 1, 0], [-2, 0, 0], [-1, 0, 5], [-1, 0, 0], [0, 0, 0]])
    counts = np.array([3, 3, 3, 2, 4, 0])
    tree = _tree(parents, counts)
    assert attention.read_status() == _native.STATUS_TREE
    assert tree.counts.tolist() == [3, 0, 0, 2, 0, 0]
    assert tree.ancestors.tolist() == [[1, 3, 7], [0, 0, 0], [0, 0, 0], [1, 3, 0], [0] * 3, [0] * 3]
    assert tree.depths.tolist() == [[0, 1, 2], [0] * 3, [0] * 3, [0, 1, 0], [0] * 3, [0] * 3]


@pytest.mark.parametrize("nodes,shape", [(1, "chain"), (64, "chain"), (64, "star"), (64, "tree"),
                                         (40, "forest")])
def test_plan(nodes, shape):
    rng = np.random.default_rng(nodes)
    parents = _parents(rng, 9, nodes, shape)
    counts = rng.integers(0, nodes + 1, 9)
    above, depths = oracle.plan(parents, counts)
    bits = (above.astype(object) << np.arange(nodes).astype(object)).sum(-1)
    tree = _tree(parents, counts)
    assert [[v & (1 << 64) - 1 for v in row] for row in tree.ancestors.tolist()] == bits.tolist()
    assert tree.depths.tolist() == depths.tolist() and tree.counts.tolist() == counts.tolist()
    one = attention.draft_tree(_gpu(parents[:1], torch.int32).expand(5, nodes))
    assert torch.equal(one.ancestors, one.ancestors[:1].expand(5, nodes))


def _accept_case(seed, batch, nodes, length=512, vocab=6):
    """Few tokens, so that drafts agree often, siblings share tokens and ends
    of sequence fall anywhere."""
    rng = np.random.default_rng(seed)
    parents = _parents(rng, batch, nodes, "tree")
    counts = rng.integers(0, nodes + 1, batch) if seed % 2 else np.full(batch, nodes)
    chosen, drafts = rng.integers(0, vocab, (2, batch, nodes))
    follow = np.take_along_axis(chosen, np.maximum(parents, 0), 1)
    drafts = np.where(rng.random((batch, nodes)) < 0.6, follow, drafts)
    position = rng.integers(0, length - nodes - 1, batch)
    state = dict(tokens=drafts[:, 0], position=position, end=position + rng.integers(0, 40, batch),
                 finished=rng.random(batch) < 0.2, sum_logprobs=rng.random(batch).astype(np.float32),
                 generated=rng.integers(0, vocab, (batch, length)))
    return parents, counts, drafts, chosen, -rng.random((batch, nodes)).astype(np.float32), state


def _device_state(state):
    return {name: torch.from_numpy(np.array(v, copy=True)).to(DEV) for name, v in state.items()}


@pytest.mark.parametrize("seed,batch,nodes", [(0, 1, 1), (1, 7, 5), (2, 64, 16), (3, 130, 64),
                                              (4, 3, 33)])
@pytest.mark.parametrize("own_lengths", [False, True])
def test_accept(seed, batch, nodes, own_lengths):
    parents, counts, drafts, chosen, logprob, state = _accept_case(seed, batch, nodes)
    lengths = state["position"] // 2 if own_lengths else None
    want = oracle.accept(parents, counts, drafts, chosen, logprob, state, (5,), lengths)
    dev = _device_state(state)
    dev_lengths = None if lengths is None else _gpu(lengths, torch.int64)
    got = step.accept_tree(_tree(parents, counts), _gpu(drafts, torch.int64),
                           _gpu(chosen, torch.int64), _gpu(logprob, torch.float32),
                           dev["tokens"][:, None], dev["position"], dev["end"], dev["finished"],
                           dev["sum_logprobs"], dev["generated"], [5], lengths=dev_lengths)
    np.testing.assert_array_equal(got.path.cpu(), want[0])
    np.testing.assert_array_equal(got.counts.cpu(), want[1])
    np.testing.assert_array_equal(got.start.cpu(), want[2])
    for name in state:  # the sums too: the same float32 additions in the same order
        np.testing.assert_array_equal(dev[name].cpu(), want[3][name], err_msg=name)
    if own_lengths:
        np.testing.assert_array_equal(dev_lengths.cpu(), want[4])
    assert attention.read_status() == 0


def test_accept_past_the_generated_tokens_is_flagged():
    parents, counts, drafts, chosen, logprob, state = _accept_case(2, 4, 8)
    state.update(position=np.array([510, 3, 511, -9]), finished=np.zeros(4, bool),
                 end=np.full(4, 9999))
    dev = _device_state(state)
    before = dev["generated"].clone()
    step.accept_tree(_tree(parents, counts), _gpu(drafts, torch.int64), _gpu(chosen, torch.int64),
                     _gpu(logprob, torch.float32), dev["tokens"], dev["position"], dev["end"],
                     dev["finished"], dev["sum_logprobs"], dev["generated"], [])
    assert attention.read_status() == _native.STATUS_POSITION
    assert torch.equal(dev["generated"][2], before[2]) and torch.equal(dev["generated"][3], before[3])


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("heads_first,layers,batch,nodes,heads,dim", [
    (False, 3, 5, 64, 8, 128), (True, 2, 3, 9, 20, 64), (False, 1, 1, 1, 1, 64), (True, 1, 4, 20, 3, 128)])
def test_commit(tag, heads_first, layers, batch, nodes, heads, dim):
    rng = np.random.default_rng(nodes)
    length = 150
    base = _gpu(rng.standard_normal((2, layers, batch, length, heads, dim)), DTYPES[tag])
    weights = _gpu(rng.random((layers, batch, heads, length)), torch.float32)
    counts = rng.integers(0, nodes + 1, batch)
    path = np.full((batch, nodes), -1)
    for b in range(batch):
        path[b, :counts[b]] = np.sort(rng.permutation(nodes)[:counts[b]])
    start = rng.integers(0, length - nodes + 1, batch)
    accepted = step.AcceptedPath(_gpu(path, torch.int32), _gpu(counts, torch.int32),
                                 _gpu(start, torch.int64))
    caches = [(c.transpose(2, 3) if heads_first else c).contiguous() for c in base]
    want = [oracle.commit(_np(c), path, counts, start) for c in base]
    want_weights = oracle.commit(_np(weights.transpose(2, 3)), path, counts, start)
    commit = cache.whisper_commit_tree if heads_first else cache.qwen3_commit_tree
    if layers == 1:
        commit(caches[0][0], caches[1][0], accepted, weights=weights[0])
    else:
        commit(caches[0], caches[1], accepted, weights=weights)
    for c, w in zip(caches, want):
        np.testing.assert_array_equal(_np(c.transpose(2, 3) if heads_first else c), w)
    np.testing.assert_array_equal(_np(weights.transpose(2, 3)), want_weights)
    assert attention.read_status() == 0


def test_commit_skips_invalid_paths():
    keys = torch.randn((1, 5, 40, 2, 64), device=DEV)
    values = torch.randn_like(keys)
    before = keys.clone()
    path = torch.tensor([[1, 0, -1], [0, 3, -1], [0, 2, -1], [1, -1, -1], [0, 1, 2]])
    accepted = step.AcceptedPath(path.to(DEV, torch.int32),
                                 torch.tensor([2, 2, 2, 1, 4], device=DEV, dtype=torch.int32),
                                 torch.tensor([0, 0, 38, -2, 0], device=DEV))
    cache.qwen3_commit_tree(keys, values, accepted)
    assert attention.read_status() == _native.STATUS_POSITION
    assert torch.equal(keys, before)


@pytest.mark.parametrize("tag", ["bf16", "f32"])
@pytest.mark.parametrize("heads_first,layers,heads,dim,length,budget,sink,recent", [
    (False, 1, 8, 128, 1024, 512, 4, 64), (False, 2, 2, 64, 100, 33, 0, 0),
    (True, 1, 6, 64, 448, 200, 3, 197), (False, 1, 1, 128, 5000, 4999, 0, 1),
    (False, 1, 2, 64, 20000, 777, 5, 70), (True, 1, 3, 64, 300, 1, 0, 0),
    (True, 3, 20, 64, 448, 200, 3, 7), (False, 2, 16, 128, 1024, 1000, 1, 1)])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_evict(tag, heads_first, layers, heads, dim, length, budget, sink, recent, kind):
    rng = np.random.default_rng(length)
    lengths = np.array([length, budget, budget + 1 if budget < length else 0, 0, length - 1])
    batch = len(lengths)
    weights = rng.random((layers, batch, heads, length)).astype(np.float32) ** 4
    if kind == "ties":
        weights = np.floor(weights * 3).astype(np.float32)
    elif kind == "odd":
        odd = rng.choice([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.5, 1e-42], weights.shape)
        weights = np.where(rng.random(weights.shape) < 0.4, odd, weights).astype(np.float32)
    kept = oracle.evict(weights, lengths, budget, sink, recent)
    base = torch.randn((2, layers, batch, length, heads, dim), device=DEV).to(DTYPES[tag])
    caches = [(c.transpose(2, 3) if heads_first else c).contiguous().clone() for c in base]
    w = torch.from_numpy(weights.copy()).to(DEV)
    evict = cache.whisper_evict if heads_first else cache.qwen3_evict
    n, k = evict(caches[0], caches[1], w, _gpu(lengths, torch.int64), budget, sink, recent)
    np.testing.assert_array_equal(n.cpu(), np.minimum(lengths, budget))
    np.testing.assert_array_equal(k.cpu(), kept)
    after = [c.transpose(2, 3) if heads_first else c for c in caches]
    for layer in range(layers):
        for b in range(batch):
            for h in range(heads):
                slots = torch.from_numpy(kept[layer, b, h]).to(DEV)
                slots = slots[slots >= 0]
                for c, old in zip(after, base):
                    assert torch.equal(c[layer, b, :len(slots), h], old[layer, b][slots, h])
                    assert torch.equal(c[layer, b, len(slots):, h], old[layer, b, len(slots):, h])
                want = weights[layer, b, h].copy()
                want[:len(slots)] = want[slots.cpu().numpy()]
                np.testing.assert_array_equal(w[layer, b, h].cpu().numpy().view(np.int32),
                                              want.view(np.int32))
    assert attention.read_status() == 0


@pytest.mark.parametrize("length,budget,sink,recent", [
    (1025, 1000, 3, 9), (2049, 64, 0, 64), (4096, 2048, 0, 0), (4097, 4000, 100, 100),
    (16384, 4096, 8, 1024), (16385, 1, 0, 0), (33000, 20000, 4, 0)])
@pytest.mark.parametrize("distinct", [0, 2, 7])
def test_evict_long_rows(length, budget, sink, recent, distinct):
    """Rows that several CTAs share, some of them with slots of few distinct
    weights, some that end in the first CTA's."""
    rng = np.random.default_rng(length + distinct)
    lengths = np.array([length, budget + 1, (length + budget) // 2, length - 1])
    weights = rng.random((1, 4, 2, length)).astype(np.float32)
    if distinct:
        weights = np.floor(weights ** 3 * distinct).astype(np.float32)
    keys = torch.arange(length, device=DEV, dtype=torch.float32)[None, :, None, None].expand(
        4, length, 2, 64).contiguous()
    values, w = -keys, torch.from_numpy(weights[0].copy()).to(DEV)
    n, kept = cache.qwen3_evict(keys, values, w, _gpu(lengths, torch.int64), budget, sink, recent)
    want = oracle.evict(weights, lengths, budget, sink, recent)[0]
    np.testing.assert_array_equal(n.cpu(), budget)
    np.testing.assert_array_equal(kept.cpu(), want)
    np.testing.assert_array_equal(keys[:, :budget, :, 0].cpu(), want.transpose(0, 2, 1))
    np.testing.assert_array_equal(values[:, :budget, :, 63].cpu(), -want.transpose(0, 2, 1))
    np.testing.assert_array_equal(w[:, :, :budget].cpu(), np.take_along_axis(weights[0], want, -1))
    np.testing.assert_array_equal(w[:, :, budget:].cpu(), weights[0, :, :, budget:])
    assert attention.read_status() == 0


@pytest.mark.parametrize("family,heads,kv_heads,dim,nodes", [
    ("qwen3", 16, 8, 128, 4), ("qwen3", 16, 8, 128, 16), ("whisper", 4, 4, 64, 40)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_score_that_is_not_finite_stays_in_its_row(family, heads, kv_heads, dim, nodes, bad):
    """A cached key that makes scores NaN or infinite (of either sign): only the
    batch row's outputs of that head change, and a NaN is seen in all of them."""
    x = _inputs(3, family, "bf16", 3, nodes, 400, heads, kv_heads, dim, [300, 300, 300])
    good = _call(x)[0]
    position = (1, 70, 1, 5) if family == "qwen3" else (1, 1, 70, 5)
    x["keys"][position] = bad
    out = _call(x)[0].view(3, nodes, heads, dim)
    group = heads // kv_heads
    if np.isnan(bad):
        assert torch.isnan(out[1, :, group:2 * group]).all()
    good = good.view(3, nodes, heads, dim)
    for b, first, last in ((0, 0, heads), (2, 0, heads), (1, 0, group), (1, 2 * group, heads)):
        assert torch.equal(out[b, :, first:last], good[b, :, first:last])


def test_evict_skips_rows_out_of_range():
    keys, values = torch.randn((2, 3, 50, 2, 64), device=DEV)
    before, weights = keys.clone(), torch.rand((3, 2, 50), device=DEV)
    n, kept = cache.qwen3_evict(keys, values, weights, torch.tensor([51, -1, 1 << 40], device=DEV), 20)
    assert attention.read_status() == _native.STATUS_POSITION
    assert torch.equal(keys, before) and n.tolist() == [51, -1, 1 << 40] and (kept == -1).all()


# ------------------------------------------------------ the operators together


class _Decoder:
    """A small float32 decoder on the package's ops: two layers of Qwen3
    attention and a tied output layer."""

    def __init__(self, batch, length, seed=0):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        draw = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
        self.heads, self.kv_heads, self.dim, width = 4, 2, 64, 128
        self.embed = draw(50, width)
        self.qkv = [draw(width, (4 + 2 * 2) * 64) / 11 for _ in range(2)]
        self.out = [draw(4 * 64, width) / 16 for _ in range(2)]
        self.norms = torch.ones(64, device=DEV)
        cos, sin = oracle_attention.rope_tables(1e4, 64, 2 * length)
        self.cos, self.sin = _gpu(cos, torch.float32), _gpu(sin, torch.float32)
        self.keys = torch.zeros((2, batch, length, 2, 64), device=DEV)
        self.values = torch.zeros_like(self.keys)
        self.weights = torch.zeros((2, batch, 2, length), device=DEV)

    def __call__(self, tokens, tree, positions, lengths, keep_weights=False):
        x = self.embed[tokens]
        for layer in range(2):
            a = attention.qwen3_attention_tree(
                x @ self.qkv[layer], self.norms, self.norms, 1e-6, self.cos, self.sin, positions,
                tree, self.keys[layer], self.values[layer], 4, 2, lengths=lengths,
                weights=self.weights[layer] if keep_weights else None)
            x = x + a @ self.out[layer]
        return x


def _fresh_state(batch, length, first):
    return dict(tokens=first.clone(), position=torch.zeros(batch, dtype=torch.int64, device=DEV),
                end=torch.full((batch,), 60, dtype=torch.int64, device=DEV),
                finished=torch.zeros(batch, dtype=torch.bool, device=DEV),
                sum_logprobs=torch.zeros(batch, device=DEV),
                generated=torch.zeros((batch, length), dtype=torch.int64, device=DEV))


def test_speculative_decoding_gives_the_greedy_tokens():
    """Drafts, partly right, over trees: the tokens, positions and sums of
    plain greedy steps, in fewer steps."""
    batch, length, nodes = 5, 128, 12
    rng = np.random.default_rng(0)
    first = torch.arange(batch, device=DEV)
    eos = [3]
    plain, state = _Decoder(batch, length), _fresh_state(batch, length, first)
    single = attention.draft_tree(torch.full((batch, 1), -1, dtype=torch.int32, device=DEV))
    while not state["finished"].all():
        hidden = plain(state["tokens"][:, None], single, state["position"], None)
        step.greedy_step(hidden[:, 0], plain.embed, *state.values(), eos)
    fast, got = _Decoder(batch, length), _fresh_state(batch, length, first)
    steps = 0
    while not got["finished"].all():
        assert steps < 60
        parents = _parents(rng, batch, nodes, "tree")
        tree = _tree(parents, rng.integers(1, nodes + 1, batch))
        # A node's draft is the true token at its depth, or a wrong one.
        at = (got["position"][:, None] + tree.depths).clamp(max=length - 1)
        drafts = state["generated"].gather(1, at)
        wrong = torch.from_numpy(rng.random((batch, nodes)) < 0.4).to(DEV)
        drafts = torch.where(wrong, (drafts + 1) % 50, drafts)
        drafts[:, 0] = got["tokens"]
        start = got["position"].clone()
        hidden = fast(drafts, tree, start, None)
        accepted = step.greedy_tree_step(hidden, fast.embed, tree, drafts, *got.values(), eos)
        cache.qwen3_commit_tree(fast.keys, fast.values, accepted)
        steps += 1
    assert steps < int(state["position"].max())
    for name in ("tokens", "position", "finished", "generated"):
        assert torch.equal(got[name], state[name]), name
    # Sums over at most 60 float32 log-probabilities of some units each.
    torch.testing.assert_close(got["sum_logprobs"], state["sum_logprobs"], rtol=1e-4, atol=1e-3)
    for b in range(batch):  # the committed caches are those of the plain steps
        m = int(state["position"][b])
        for c, d in ((fast.keys, plain.keys), (fast.values, plain.values)):
            torch.testing.assert_close(c[:, b, :m], d[:, b, :m], rtol=1e-3, atol=1e-3)
    assert attention.read_status() == 0


def test_decoding_with_a_bounded_cache():
    """Single steps that gather weights and evict over the budget, all layers
    in one call, against the oracle's steps on the same inputs."""
    batch, length, budget = 3, 24, 10
    rng = np.random.default_rng(1)
    heads, kv_heads, dim, layers = 4, 2, 64, 2
    keys, values = np.zeros((2, layers, batch, length, kv_heads, dim))
    weights = np.zeros((layers, batch, kv_heads, length))
    dev = [_gpu(x, torch.float32) for x in (keys, values, weights)]
    lengths, positions = np.zeros(batch, np.int64), np.zeros(batch, np.int64)
    dev_lengths, dev_positions = _gpu(lengths, torch.int64), _gpu(positions, torch.int64)
    cos, sin = oracle_attention.rope_tables(1e4, dim, 64)
    cos, sin = cos.astype(np.float32), sin.astype(np.float32)
    ones = np.ones(dim)
    tree = attention.draft_tree(torch.full((batch, 1), -1, dtype=torch.int32, device=DEV))
    for _ in range(30):
        for layer in range(layers):
            qkv = rng.standard_normal((batch, 1, (heads + 2 * kv_heads) * dim)).astype(np.float32)
            out = attention.qwen3_attention_tree(
                _gpu(qkv, torch.float32), _gpu(ones, torch.float32), _gpu(ones, torch.float32), 1e-6,
                _gpu(cos, torch.float32), _gpu(sin, torch.float32), dev_positions, tree,
                dev[0][layer], dev[1][layer], heads, kv_heads, lengths=dev_lengths,
                weights=dev[2][layer])
            q, k, v = np.split(qkv.reshape(batch, 1, -1, dim), (heads, heads + kv_heads), 2)
            want = oracle.tree_attention(
                q, k, v, keys[layer], values[layer], lengths, np.ones((batch, 1, 1), bool),
                np.ones(batch, int), dim ** -0.5, weights[layer],
                (ones, ones, 1e-6, cos, sin, positions, np.zeros((batch, 1), int)))
            keys[layer], values[layer], weights[layer] = (want[n] for n in
                                                          ("keys", "values", "weights"))
            np.testing.assert_allclose(_np(out).reshape(want["out"].shape), want["out"], atol=1e-5)
        lengths, positions = lengths + 1, positions + 1
        dev_lengths += 1
        dev_positions += 1
        kept = oracle.evict(weights, lengths, budget, 1, 3)
        dev_lengths, got = cache.qwen3_evict(dev[0], dev[1], dev[2], dev_lengths, budget, 1, 3)
        np.testing.assert_array_equal(got.cpu(), kept)
        for layer, b, h in np.ndindex(layers, batch, kv_heads):
            slots = kept[layer, b, h]
            slots = slots[slots >= 0]
            keys[layer, b, :len(slots), h] = keys[layer, b, slots, h]
            values[layer, b, :len(slots), h] = values[layer, b, slots, h]
            weights[layer, b, h, :len(slots)] = weights[layer, b, h, slots]
        lengths = np.minimum(lengths, budget)
        np.testing.assert_array_equal(dev_lengths.cpu(), lengths)
        np.testing.assert_allclose(_np(dev[2]), weights, atol=1e-5)
    assert attention.read_status() == 0


def _graph_case(seed, nodes, length, lengths, weights):
    x = _inputs(seed, "qwen3", "bf16", len(lengths), nodes, length, 16, 8, 128, lengths,
                weights=weights)
    parents = _gpu(x["parents"], torch.int32)
    at = _gpu(x["lengths"], torch.int64)
    keys, values = x["keys"].clone(), x["values"].clone()
    held = None if x["weights"] is None else x["weights"].clone()
    results = []

    def run():
        if held is not None:
            held.copy_(x["weights"])
        tree = attention.draft_tree(parents)
        out = attention.qwen3_attention_tree(x["qkv"], x["wq"], x["wk"], 1e-6, x["cos"], x["sin"],
                                             at, tree, keys, values, 16, 8, weights=held)
        results[:] = [out, held]

    return x, run, results


def test_captured_graphs_replay_side_by_side():
    """Two graphs on one pool each, replayed at once on two streams, with eager
    calls beside them: no workspace is shared."""
    cases = [_graph_case(1, 8, 4096, [4000, 3000], True), _graph_case(2, 20, 2048, [2000] * 3, False)]
    graphs = [CapturedGraph(run) for _, run, _ in cases]
    captured = [list(results) for _, _, results in cases]
    wants = [_call(x) for x, _, _ in cases]
    for out, held in captured:
        out.zero_()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            beside = _call(cases[0][0])
    torch.cuda.synchronize()
    for (out, held), want in zip(captured, wants):
        assert torch.equal(out, want[0])
        assert held is None or torch.equal(held, want[3])
    assert torch.equal(beside[0], wants[0][0]) and torch.equal(beside[3], wants[0][3])
    assert attention.read_status() == 0


def test_a_captured_step_replays():
    """Acceptance and commit in a graph, replayed on new drafts."""
    batch, nodes, length = 6, 10, 128
    parents, counts, drafts, chosen, logprob, state = _accept_case(2, batch, nodes, length)
    dev, p = _device_state(state), _gpu(parents, torch.int32)
    start = {n: v.clone() for n, v in dev.items()}
    d, c, lp = _gpu(drafts, torch.int64), _gpu(chosen, torch.int64), _gpu(logprob, torch.float32)
    keys, values = torch.randn((2, 2, batch, length, 2, 64), device=DEV)
    before = _np(keys)
    results = []

    def run():
        accepted = step.accept_tree(attention.draft_tree(p), d, c, lp, *dev.values(), [5])
        cache.qwen3_commit_tree(keys, values, accepted)
        results[:] = [accepted]

    graph = CapturedGraph(run)
    keys.copy_(torch.from_numpy(before))
    other = _accept_case(4, batch, nodes, length)
    p.copy_(torch.from_numpy(other[0]))
    d.copy_(torch.from_numpy(other[2]))
    c.copy_(torch.from_numpy(other[3]))
    lp.copy_(torch.from_numpy(other[4]))
    for n in dev:
        dev[n].copy_(start[n])
    graph.replay()
    want = oracle.accept(other[0], np.full(batch, nodes), other[2], other[3], other[4], state, (5,))
    np.testing.assert_array_equal(results[0].path.cpu(), want[0])
    np.testing.assert_array_equal(dev["generated"].cpu(), want[3]["generated"])
    np.testing.assert_array_equal(_np(keys), oracle.commit(before, want[0], want[1], want[2]))


def test_calls_on_another_stream():
    x = _inputs(8, "qwen3", "bf16", 4, 6, 2000, 16, 8, 128, [1500, 900, 30, 1994], weights=True)
    want = _call(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _call(x)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_strided_vectors():
    """Lengths, positions and counts that are columns of wider tensors (their
    copies have to outlive the call), and a fragmented allocator."""
    x = _inputs(21, "qwen3", "bf16", 40, 3, 300, 16, 8, 128, list(range(0, 240, 6)), ahead=5)
    want = _call(x)
    tree = _tree(x["parents"], x["counts"])
    wide = torch.empty((40, 7), dtype=torch.int64, device=DEV).fill_(1 << 40)
    wide[:, 2], wide[:, 5] = _gpu(x["lengths"], torch.int64), _gpu(x["positions"], torch.int64)
    counts = torch.zeros((40, 2), dtype=torch.int32, device=DEV)
    counts[:, 1] = tree.counts
    for _ in range(20):
        held = [torch.empty(n, dtype=torch.uint8, device=DEV) for n in (512, 1024, 512, 40960)]
        del held[::2]
        keys, values = x["keys"].clone(), x["values"].clone()
        out = attention.qwen3_attention_tree(
            x["qkv"], x["wq"], x["wk"], 1e-6, x["cos"], x["sin"], wide[:, 5],
            tree._replace(counts=counts[:, 1]), keys, values, 16, 8, lengths=wide[:, 2])
        assert torch.equal(out, want[0]) and torch.equal(keys, want[1])
    assert attention.read_status() == 0


@pytest.mark.parametrize("length,nodes,heads,kv_heads", [
    (1, 1, 2, 2), (17, 17, 4, 2), (40, 40, 2, 2), (64, 64, 2, 1), (70, 33, 4, 2), (127, 50, 2, 2)])
def test_caches_shorter_than_a_tile(length, nodes, heads, kv_heads):
    x = _inputs(length, "qwen3", "bf16", 2, nodes, length, heads, kv_heads, 128,
                [0, length - nodes])
    _check(x, _call(x), _want(x))


def test_a_captured_eviction_replays():
    """Rows that a cluster shares, captured with the commit before it."""
    keys = torch.randn((2, 5000, 2, 64), device=DEV)
    weights, lengths = torch.rand((2, 2, 5000), device=DEV), torch.tensor([5000, 4100], device=DEV)
    accepted = step.AcceptedPath(torch.tensor([[0, 2, -1], [0, 1, 2]], device=DEV).int(),
                                 torch.tensor([2, 3], device=DEV).int(),
                                 torch.tensor([4990, 7], device=DEV))
    first = [t.clone() for t in (keys, -keys, weights)]

    def run(k, v, w):
        cache.qwen3_commit_tree(k, v, accepted, weights=w)
        return (k, v, w, *cache.qwen3_evict(k, v, w, lengths, 1000, sink=3, recent=30))

    want = [t.clone() for t in run(*(t.clone() for t in first))]
    state = [t.clone() for t in first]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*(t.clone() for t in first))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(*state)
    for _ in range(3):
        for t, start in zip(state, first):
            t.copy_(start)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert attention.read_status() == 0


# ----------------------------------------------------------------- refusals


def test_refusals():
    x = _inputs(9, "qwen3", "bf16", 2, 3, 64, 16, 8, 128, [5, 9])
    tree = _tree(x["parents"], x["counts"])
    at = _gpu(x["lengths"], torch.int64)
    good = dict(qkv=x["qkv"], q_norm_weight=x["wq"], k_norm_weight=x["wk"], eps=1e-6, cos=x["cos"],
                sin=x["sin"], positions=at, tree=tree, keys=x["keys"], values=x["values"], heads=16,
                kv_heads=8)
    attention.qwen3_attention_tree(**good)
    w = torch.zeros((2, 8, 64), device=DEV)
    for change, error in [
            (dict(qkv=x["qkv"][:, :, :-128]), ValueError), (dict(qkv=x["qkv"].float()), TypeError),
            (dict(qkv=x["qkv"].half()), TypeError), (dict(positions=at.int()), ValueError),
            (dict(lengths=at[:1]), ValueError), (dict(keys=x["keys"][:1]), ValueError),
            (dict(values=x["values"][:, :32]), ValueError), (dict(weights=w[:, :, :9]), ValueError),
            (dict(weights=w.bfloat16()), ValueError), (dict(cos=x["cos"][:, :64]), ValueError),
            (dict(tree=_tree(x["parents"][:, :2], np.array([2, 2]))), ValueError),
            (dict(tree=tree._replace(depths=tree.depths.long())), ValueError),
            (dict(positions=at.cpu()), ValueError), (dict(keys=x["keys"].cpu()), ValueError)]:
        with pytest.raises(error):
            attention.qwen3_attention_tree(**{**good, **change})
    nine = _inputs(9, "qwen3", "bf16", 2, 9, 64, 16, 8, 128, [5, 9], weights=True)
    with pytest.raises(_native.NativeError, match="at most 16 query rows"):
        _call(nine)
    with pytest.raises(ValueError):
        attention.draft_tree(torch.zeros((2, 65), dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        attention.draft_tree(torch.zeros((2, 5), dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError):
        cache.qwen3_evict(x["keys"], x["values"], w, at, 10, sink=6, recent=5)
    with pytest.raises(ValueError):
        cache.qwen3_evict(x["keys"], x["values"], w, at, 65)
    with pytest.raises(ValueError):
        cache.whisper_evict(x["keys"], x["values"], w, at, 10)
    odd = torch.zeros((2, 64, 8, 136), dtype=torch.bfloat16, device=DEV)[..., 1:129]
    with pytest.raises(_native.NativeError, match="16-byte"):
        cache.qwen3_evict(odd, odd, w, at, 10)
    assert attention.read_status() == 0
