"""Calls of the draft-tree operators that other tests do not make: from several
threads and streams, on views, at the edges of the cache."""

from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from asrback_b200 import _native, attention, cache, step
from asrback_b200.transcription import CapturedGraph
from oracle import tree as oracle
from tests.test_gpu_tree import (DEV, _accept_case, _call, _Decoder, _device_state, _fresh_state, _gpu,
                                 _inputs, _np, _parents, _tree, _want)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status():
    attention.read_status()
    yield


def _recorded(monkeypatch, name, call):
    """A function that makes ``call``'s call of entry point ``name`` over again,
    on the same buffers, with no work in Python; and ``call``'s result."""
    made, held, empty = [], [], torch.empty

    def record(entry, *args):
        if entry == name:
            made.append(args)
        return real(entry, *args)

    def hold(*args, **kwargs):
        held.append(empty(*args, **kwargs))
        return held[-1]

    packed = name in _native._PACKED
    real = _native.call_packed if packed else _native.call
    with monkeypatch.context() as m:
        m.setattr(_native, real.__name__, record)
        m.setattr(torch, "empty", hold)
        result = call()
    (args,), lib = made, _native.load()
    if packed:
        entry, args = getattr(lib, name + "_packed"), (_native._PACKED[name](*args),)
    else:
        entry = getattr(lib, name)

    def again(held=held):
        if entry(*args) != _native.OK:
            raise _native.NativeError(lib.asrback_last_error().decode())

    return again, result


def _in_threads(calls, times):
    """Every call ``times`` times in a thread of its own, all at once; raises
    what one of them raised."""
    errors, start = [], threading.Barrier(len(calls))

    def work(call):
        start.wait()
        try:
            for _ in range(times):
                call()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(call,)) for call in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    if errors:
        raise errors[0]


def test_float32_attention_from_two_threads(monkeypatch):
    """Calls of few and of many rows, whose kernels ask for less and for more
    shared memory."""
    calls, outs = [], []
    for batch in (1, 1024):
        x = _inputs(batch, "whisper", "f32", batch, 1, 64, 2, 2, 64, np.arange(batch) % 64)
        tree, at = _tree(x["parents"], x["counts"]), _gpu(x["lengths"], torch.int64)
        again, out = _recorded(
            monkeypatch, "asrback_tree_attention",
            lambda x=x, tree=tree, at=at: attention.whisper_self_attention_tree(
                x["q"], x["k"], x["v"], x["keys"], x["values"], at, tree))
        calls.append(again)
        outs.append((out, out.clone(), x, tree, at))  # what the call reads stays alive
    _in_threads(calls, 5000)
    assert all(torch.equal(out, want) for out, want, *_ in outs)
    assert attention.read_status() == 0


def test_float32_choice_from_two_threads(monkeypatch):
    """As above, for the step's choice of tokens: few and many hidden elements."""
    calls, outs = [], []
    gen = torch.Generator(device=DEV).manual_seed(0)
    for batch, width in ((1, 64), (50, 1024)):
        hidden = torch.randn((batch, width), generator=gen, device=DEV)
        weight = torch.randn((500, width), generator=gen, device=DEV)
        again, out = _recorded(monkeypatch, "asrback_greedy_step",
                               lambda hidden=hidden, weight=weight: step.greedy_choose(hidden, weight))
        calls.append(again)
        outs.append((*out, out[0].clone(), out[1].clone(), hidden, weight))
    _in_threads(calls, 5000)
    for token, logprob, want_token, want_logprob, *_ in outs:
        assert torch.equal(token, want_token) and torch.equal(logprob, want_logprob)
    assert attention.read_status() == 0


def _step_case(seed, batch, nodes, vocab, width):
    """A step over trees from the nodes' hidden states: a function that starts
    from the same state every time, and the tensors that it writes."""
    parents, counts, drafts, _, _, state = _accept_case(seed, batch, nodes)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    hidden = torch.randn((batch, nodes, width), generator=gen, device=DEV).bfloat16()
    weight = torch.randn((vocab, width), generator=gen, device=DEV).bfloat16()
    tree, drafts = _tree(parents, counts), _gpu(drafts, torch.int64)
    start = _device_state(state)
    dev = {n: v.clone() for n, v in start.items()}
    written = []

    def run():
        for n, v in dev.items():
            v.copy_(start[n])
        accepted = step.greedy_tree_step(hidden, weight, tree, drafts, *dev.values(), [5])
        written[:] = [*accepted, *dev.values()]

    return run, written


def test_tree_steps_run_side_by_side():
    """Steps on two streams at once, called and replayed: none meets the other's
    partial results."""
    cases = [_step_case(2, 16, 16, 30000, 512), _step_case(4, 9, 7, 50000, 256)]
    wants = []
    for run, written in cases:
        run()
        wants.append([t.clone() for t in written])
    streams = [torch.cuda.Stream() for _ in cases]
    graphs = []
    torch.cuda.synchronize()
    for kind in ("called", "replayed"):
        if kind == "replayed":
            graphs = [CapturedGraph(run) for run, _ in cases]
            torch.cuda.synchronize()
        for _ in range(100):
            for i, stream in enumerate(streams):
                with torch.cuda.stream(stream):
                    graphs[i].replay() if graphs else cases[i][0]()
        torch.cuda.synchronize()
        for (_, written), want in zip(cases, wants):
            assert all(torch.equal(a, b) for a, b in zip(written, want)), kind
    assert attention.read_status() == 0


def test_tree_steps_of_two_streams_have_two_workspaces(monkeypatch):
    run, _ = _step_case(2, 2, 3, 1000, 64)
    used, real = [], _native.call

    def record(name, *args):
        used.append(args[-4])
        return real(name, *args)

    monkeypatch.setattr(_native, "call", record)
    for stream in (torch.cuda.Stream(), torch.cuda.Stream()):
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            run()
        torch.cuda.synchronize()
    assert len(set(used)) == 2


def test_a_plan_of_one_transposed_row():
    """A view whose rows are one element apart, which matters to no one: there
    is one row."""
    parents = torch.tensor([[-1], [0], [0], [1]], dtype=torch.int32, device=DEV).t()
    assert parents.shape == (1, 4) and parents.stride() == (1, 1)
    tree = attention.draft_tree(parents)
    assert tree.ancestors.tolist() == [[1, 3, 5, 11]] and tree.depths.tolist() == [[0, 1, 1, 2]]
    assert attention.read_status() == 0


@pytest.mark.parametrize("start", [(1 << 63) - 1, (1 << 63) - 2, 1 << 62, 1 << 32, 40, 39, -1])
def test_commit_skips_starts_out_of_range(start):
    """Starts up to the largest integer, whose sum with a node would pass it."""
    keys = torch.randn((1, 1, 40, 2, 64), device=DEV)
    before, weights = keys.clone(), torch.rand((1, 1, 2, 40), device=DEV)
    old = weights.clone()
    accepted = step.AcceptedPath(torch.tensor([[1, 2, -1]], device=DEV).int(),
                                 torch.tensor([2], device=DEV).int(),
                                 torch.tensor([start], device=DEV))
    cache.qwen3_commit_tree(keys, keys.clone(), accepted, weights=weights)
    assert attention.read_status() == _native.STATUS_POSITION
    assert torch.equal(keys, before) and torch.equal(weights, old)


def test_a_plan_is_cut_to_the_room_in_the_cache():
    nodes, capacity = 6, 40
    parents = _parents(np.random.default_rng(0), 9, nodes, "tree")
    counts = np.array([6, 6, 6, 6, 6, 6, 2, 4, 0])
    lengths = np.array([0, 34, 35, 39, 12, 38, 37, 37, 40])
    fits = np.array([6, 6, 5, 1, 6, 2, 2, 3, 0])
    tree = attention.draft_tree(_gpu(parents, torch.int32), _gpu(counts, torch.int32),
                                _gpu(lengths, torch.int64), capacity)
    assert attention.read_status() == 0  # the last row is full and wants nothing
    want = _tree(parents, fits)
    assert tree.counts.tolist() == fits.tolist()
    assert all(torch.equal(a, b) for a, b in zip(tree[1:], want[1:]))
    for length in (40, 41, -1, 1 << 62, -(1 << 63)):
        tree = attention.draft_tree(_gpu(parents[:2], torch.int32), None,
                                    torch.tensor([5, length], device=DEV), capacity)
        assert attention.read_status() == _native.STATUS_POSITION
        assert tree.counts.tolist() == [6, 0] and not tree.ancestors[1].any()
    two, at = _gpu(parents[:2], torch.int32), torch.tensor([5, 6], device=DEV)
    for lengths, slots in ((at, None), (None, 40), (at, 0), (at.int(), 40), (at[:1], 40), (at.cpu(), 40)):
        with pytest.raises(ValueError):
            attention.draft_tree(two, None, lengths, slots)


class _Varied(_Decoder):
    """A decoder whose tokens follow from what it attends to."""

    def __init__(self, batch, length):
        super().__init__(batch, length)
        gen = torch.Generator(device=DEV).manual_seed(1)
        self.out = [8 * w for w in self.out]
        self.head = torch.randn((50, 128), generator=gen, device=DEV)


def test_speculative_decoding_up_to_a_full_cache():
    """The documented loop: rows decode to the last slot, with drafts right and
    wrong, and give the tokens of single steps."""
    batch, length, nodes = 5, 40, 7
    first = torch.arange(batch, device=DEV)
    plain, state = _Varied(batch, length), _fresh_state(batch, length + 1, first)
    fast, got = _Varied(batch, length), _fresh_state(batch, length + 1, first)
    state["end"].fill_(length)
    got["end"].fill_(length)
    single = attention.draft_tree(torch.full((batch, 1), -1, dtype=torch.int32, device=DEV))
    for _ in range(length):
        hidden = plain(state["tokens"][:, None], single, state["position"], None)
        step.greedy_step(hidden[:, 0], plain.head, *state.values(), [])
    assert state["generated"][:, 1:].unique().numel() > 20  # they do vary
    rng = np.random.default_rng(0)
    steps = 0
    while not got["finished"].all():
        assert steps < length
        counts = torch.where(got["finished"], 0, nodes).int()
        parents = _gpu(_parents(rng, batch, nodes, "chain" if steps % 2 else "tree"), torch.int32)
        tree = attention.draft_tree(parents, counts, got["position"], length)
        at = (got["position"][:, None] + tree.depths).clamp(max=length)
        drafts = state["generated"].gather(1, at)
        wrong = torch.from_numpy(rng.random((batch, nodes)) < 0.2).to(DEV)
        drafts = torch.where(wrong, (drafts + 1) % 50, drafts)
        drafts[:, 0] = got["tokens"]
        hidden = fast(drafts, tree, got["position"].clone(), None)
        accepted = step.greedy_tree_step(hidden, fast.head, tree, drafts, *got.values(), [])
        cache.qwen3_commit_tree(fast.keys, fast.values, accepted)
        steps += 1
    assert steps < length and attention.read_status() == 0
    for name in ("tokens", "position", "finished", "generated"):
        assert torch.equal(got[name], state[name]), name
    for c, d in ((fast.keys, plain.keys), (fast.values, plain.values)):
        torch.testing.assert_close(c, d, rtol=1e-3, atol=1e-3)


@pytest.mark.parametrize("family,tag,heads,kv_heads,dim,nodes,weights", [
    ("whisper", "bf16", 6, 6, 64, 5, True), ("whisper", "f32", 6, 6, 64, 5, True),
    ("qwen3", "bf16", 4, 2, 128, 8, True), ("qwen3", "f32", 4, 2, 128, 20, False),
    ("whisper", "bf16", 2, 2, 64, 30, False), ("qwen3", "bf16", 4, 2, 128, 40, False)])
@pytest.mark.parametrize("old", [0.25, float("nan")])
def test_a_node_without_a_bit_writes_nothing(family, tag, heads, kv_heads, dim, nodes, weights, old):
    """A caller's own plan, whose node 3 sees nothing: zeros, its slot and the
    slot's weight as they were, whatever lies there; the others as without it."""
    lengths = [70, 3]
    x = _inputs(nodes, family, tag, 2, nodes, 100 + nodes, heads, kv_heads, dim, lengths,
                shape="star", weights=weights)
    tree = _tree(x["parents"], x["counts"])
    tree.ancestors[:, 3] = 0
    caches = [x[n].transpose(1, 2) if family == "whisper" else x[n] for n in ("keys", "values")]
    for b, m in enumerate(lengths):
        for c in caches:
            c[b, m + 3] = old
    out, keys, values, w = _call(x, tree)
    want = _want(x)  # of node 0's children node 3 is no one's ancestor
    others = [i for i in range(nodes) if i != 3]
    assert not out[:, 3].any()
    # The tolerance for the others: scores as in the draft-tree tests' module, one
    # rounding of the probabilities and one of the output.
    full, top = want["reach"][..., 0], want["reach"][..., 1]
    bf16, rotated = tag == "bf16", family == "qwen3"
    d = dim * 2.0 ** -24 * full + 2.0 ** -22 * (1 + full)
    if bf16 and rotated:
        d = d + 2 * 2.0 ** -7 * top + 2.0 ** -17 * full
    shift = np.expm1(2 * d)
    tol = (2.0 ** -8 if bf16 else 2.0 ** -24) * np.abs(want["out"]) + want["mass"] * (
        (2.0 ** -8 if bf16 else 0) + shift[..., None] + 200 * 2.0 ** -24)
    off = np.abs(_np(out).reshape(want["out"].shape) - want["out"])
    assert (off[:, others] <= tol[:, others]).all()
    for b, m in enumerate(lengths):
        for got, before in zip((keys, values), caches):
            torch.testing.assert_close(got[b, m + 3], before[b, m + 3], rtol=0, atol=0,
                                       equal_nan=True)
        if weights:
            assert torch.equal(w[b, :, m + 3], x["weights"][b, :, m + 3])
    if weights and not rotated:  # scores good to d: each weight to its share of what it gained
        above, _ = oracle.plan(x["parents"], x["counts"])
        above[:, 3] = False
        q, k, v = (_np(x[n]).transpose(0, 2, 1, 3) for n in "qkv")
        all_keys, all_values = (np.nan_to_num(_np(c)) for c in caches)
        start = _np(x["weights"])
        full_want = oracle.tree_attention(q, k, v, all_keys, all_values, x["lengths"], above,
                                          x["counts"], dim ** -0.5, start)["weights"]
        slots = np.ones(start.shape, bool)
        for b, m in enumerate(lengths):
            slots[b, :, m + 3] = False
        gained = full_want - start
        tol = (shift.max() + 2.0 ** -20) * np.abs(gained) + 2.0 ** -22 * (1 + np.abs(full_want))
        assert (np.abs(_np(w) - full_want)[slots] <= tol[slots]).all()
    assert attention.read_status() == 0


@pytest.mark.parametrize("tag,nodes", [("bf16", 4), ("bf16", 40), ("f32", 4)])
def test_rows_without_nodes_may_stand_anywhere(tag, nodes):
    """Lengths and positions of rows without nodes are not looked at."""
    lengths, counts = [50, 101, -1, 1 << 40, 7], [nodes, 0, 0, 0, 3]
    x = _inputs(nodes, "qwen3", tag, 5, nodes, 100, 16, 8, 128, lengths, counts)
    x["positions"] = np.array([50, 1 << 40, 3, -5, 7])
    got = _call(x)
    assert attention.read_status() == 0
    near = dict(x, lengths=np.array([50, 0, 0, 0, 7]), positions=np.array([50, 0, 0, 0, 7]))
    assert all(torch.equal(a, b) for a, b in zip(got[:3], _call(near)[:3]))
    x["counts"] = np.array([nodes, 1, 0, 0, 3])  # one that has a node is flagged
    _call(x)
    assert attention.read_status() == _native.STATUS_POSITION


class _Recorded(_Varied):
    """Keeps each layer's qkv, and runs its attention over an accepted path."""

    def __call__(self, tokens, tree, positions, lengths, keep_weights=False):
        self.kept = []
        x = self.embed[tokens]
        for layer in range(2):
            self.kept.append(x @ self.qkv[layer])
            a = self.attend(layer, self.kept[-1], positions, tree, lengths, keep_weights)
            x = x + a @ self.out[layer]
        return x

    def attend(self, layer, qkv, positions, tree, lengths, keep_weights):
        return attention.qwen3_attention_tree(
            qkv, self.norms, self.norms, 1e-6, self.cos, self.sin, positions, tree,
            self.keys[layer], self.values[layer], 4, 2, lengths=lengths,
            weights=self.weights[layer] if keep_weights else None)

    def gather(self, accepted, before):
        """The documented recipe: the path as a chain, in parts of 8 nodes."""
        part = attention.MAX_WEIGHT_ROWS // 2
        for first in range(0, accepted.path.shape[1], part):
            at = accepted.path[:, first:first + part].long().clamp(min=0)
            chain = attention.draft_tree(
                torch.arange(-1, at.shape[1] - 1, dtype=torch.int32, device=DEV).expand(len(at), -1),
                (accepted.counts - first).clamp(0, at.shape[1]))
            for layer, qkv in enumerate(self.kept):
                self.attend(layer, qkv.gather(1, at[..., None].expand(-1, -1, qkv.shape[2])),
                            before + first, chain, accepted.start + first, True)


def test_accepted_paths_gather_the_weights_of_single_steps():
    """Speculative decoding that gathers weights, with drafts rejected on the way,
    and an eviction by them: as single steps."""
    batch, length, nodes = 4, 64, 12
    first = torch.arange(batch, device=DEV)
    plain, state = _Recorded(batch, length), _fresh_state(batch, length, first)
    fast, got = _Recorded(batch, length), _fresh_state(batch, length, first)
    state["end"].fill_(60)
    got["end"].fill_(60)
    single = attention.draft_tree(torch.full((batch, 1), -1, dtype=torch.int32, device=DEV))
    for _ in range(60):
        hidden = plain(state["tokens"][:, None], single, state["position"], None, True)
        step.greedy_step(hidden[:, 0], plain.head, *state.values(), [])
    rng, steps, longest = np.random.default_rng(0), 0, 0
    while not got["finished"].all():
        assert steps < 60
        counts = torch.where(got["finished"], 0, nodes).int()
        parents = _parents(rng, batch, nodes, "chain" if steps % 3 else "tree")
        tree = attention.draft_tree(_gpu(parents, torch.int32), counts, got["position"], length)
        at = (got["position"][:, None] + tree.depths).clamp(max=length - 1)
        drafts = state["generated"].gather(1, at)
        wrong = torch.from_numpy(rng.random((batch, nodes)) < 0.1).to(DEV)
        drafts = torch.where(wrong, (drafts + 1) % 50, drafts)
        drafts[:, 0] = got["tokens"]
        before = got["position"].clone()
        hidden = fast(drafts, tree, before, None)
        accepted = step.greedy_tree_step(hidden, fast.head, tree, drafts, *got.values(), [])
        fast.gather(accepted, before)
        steps += 1
        longest = max(longest, int(accepted.counts.max()))
    assert steps < 50 and longest > 8 and attention.read_status() == 0
    assert torch.equal(got["generated"], state["generated"])
    ends = torch.full((batch,), 60, device=DEV)
    for layer in range(2):
        # float32 sums of some hundred terms of order one to ten, in another order,
        # through two layers: some 1e-5; a rejected node's share is of order 1e-2.
        for a, b in ((fast.keys[layer][:, :60], plain.keys[layer][:, :60]),
                     (fast.values[layer][:, :60], plain.values[layer][:, :60]),
                     (fast.weights[layer][..., :60], plain.weights[layer][..., :60])):
            torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)
        kept = [cache.qwen3_evict(d.keys[layer], d.values[layer], d.weights[layer], ends, 30, 2, 4)[1]
                for d in (fast, plain)]
        assert torch.equal(*kept)


@pytest.mark.parametrize("family,tag,heads,nodes,weights", [
    ("qwen3", "bf16", 2, 1, True), ("qwen3", "bf16", 2, 40, False), ("qwen3", "f32", 2, 1, True),
    ("whisper", "bf16", 1, 1, False), ("whisper", "f32", 1, 1, False)])
def test_dimensions_of_one_with_any_stride(family, tag, heads, nodes, weights):
    """One row, one node, one key/value head, a cache of one slot: their strides,
    which a view may leave at anything, are not read."""
    length = 1 if nodes == 1 else 100
    x = _inputs(nodes, family, tag, 1, nodes, length, heads, 1, 128 if family == "qwen3" else 64,
                [length - nodes], weights=weights)
    want = _call(x)
    tree, at = _tree(x["parents"], x["counts"]), _gpu(x["lengths"], torch.int64)

    def odd(t):
        t = t.clone(memory_format=torch.contiguous_format)
        return t.as_strided(t.shape, [3 if n == 1 else s for n, s in zip(t.shape, t.stride())])

    keys, values = odd(x["keys"]), odd(x["values"])
    w = odd(x["weights"]) if weights else None
    if family == "whisper":
        out = attention.whisper_self_attention_tree(odd(x["q"]), odd(x["k"]), odd(x["v"]), keys,
                                                    values, at, tree)
        keys, values = keys.transpose(1, 2), values.transpose(1, 2)
    else:
        out = attention.qwen3_attention_tree(odd(x["qkv"]), x["wq"], x["wk"], 1e-6, x["cos"],
                                             x["sin"], at, tree, keys, values, heads, 1, weights=w)
    for got, expected in zip((out, keys, values, w), want):
        assert got is expected is None or torch.equal(got, expected)
    assert attention.read_status() == 0
