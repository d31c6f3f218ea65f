"""Steps over draft trees from the nodes' hidden states, in every type and over
several launches, and the commit past 2^31 elements."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from asrback_b200 import attention, cache, step
from oracle import step as oracle_step
from oracle import tree as oracle
from tests.test_gpu_tree import DEV, DTYPES, _accept_case, _device_state, _gpu, _np, _tree

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status():
    attention.read_status()
    yield
    assert attention.read_status() == 0


@pytest.mark.parametrize("tag,batch,nodes,width", [
    ("bf16", 1, 1, 64), ("bf16", 3, 5, 1024), ("bf16", 8, 16, 128), ("bf16", 43, 3, 64),
    ("bf16", 20, 16, 256), ("f32", 1, 1, 64), ("f32", 5, 30, 64), ("f32", 3, 40, 1500)])
@pytest.mark.parametrize("suppressed", [False, True])
def test_tree_step(tag, batch, nodes, width, suppressed):
    """Hidden states and output weights of -1, 0 and 1: every logit is an integer
    that bf16 holds, so that tokens are exact, ties included."""
    rng = np.random.default_rng(batch * nodes)
    parents, counts, drafts, _, _, state = _accept_case(batch + nodes, batch, nodes)
    vocab = 3000
    hidden = rng.integers(-1, 2, (batch, nodes, width)) * (rng.random((batch, nodes, width)) < 0.2)
    weight = rng.integers(-1, 2, (vocab, width))
    suppress = rng.random(vocab) < 0.3 if suppressed else None
    logits = oracle_step.logits(weight, hidden.reshape(-1, width), tag == "bf16")
    assert np.abs(logits).max() <= 256
    chosen, logprob = (a.reshape(batch, nodes) for a in oracle_step.choose(logits, suppress))
    follow = np.take_along_axis(chosen, np.maximum(parents, 0), 1)
    drafts = np.where(rng.random((batch, nodes)) < 0.7, follow, drafts)
    eos = [int(chosen[0, -1]), 2]
    want = oracle.accept(parents, counts, drafts, chosen, logprob, state, eos)
    dev = _device_state(state)
    got = step.greedy_tree_step(
        _gpu(hidden, DTYPES[tag]), _gpu(weight, DTYPES[tag]), _tree(parents, counts),
        _gpu(drafts, torch.int64), *dev.values(), eos,
        suppress=None if suppress is None else torch.from_numpy(suppress).to(DEV))
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.cpu(), b)
    for name in ("tokens", "position", "finished", "generated"):
        np.testing.assert_array_equal(dev[name].cpu(), want[3][name], err_msg=name)
    # Each log-probability, of a float32 sum over the vocabulary, to 1e-5 at most
    # (3000 terms, 2^-24 of their sum each, and the approximations' 2^-21).
    np.testing.assert_allclose(dev["sum_logprobs"].cpu(), want[3]["sum_logprobs"], rtol=2.0 ** -20,
                               atol=nodes * (3000 * 2.0 ** -24 + 2.0 ** -20))


def test_commit_and_eviction_past_32_bits():
    """A cache of more than 2^31 elements: keys, values and weights of its last row
    move, no other row does."""
    batch, length, heads = 64, 33000, 8
    if torch.cuda.mem_get_info()[0] < 24 * 10 ** 9:
        pytest.skip("needs 24 GB")
    keys = torch.zeros((batch, length, heads, 128), dtype=torch.bfloat16, device=DEV)
    values = torch.zeros_like(keys)
    gen = torch.Generator(device=DEV).manual_seed(0)
    for t in (keys, values):
        t[-1] = torch.randn((length, heads, 128), generator=gen, device=DEV)
        t[-2, -70:] = 7  # what a wrong row's move would bring along
    weights = torch.rand((batch, heads, length), generator=gen, device=DEV)
    path = np.full((batch, 6), -1)
    path[:, 0], path[-1, :4] = 0, [0, 2, 3, 5]
    counts = np.ones(batch, int)
    counts[-1] = 4
    start = np.full(batch, 11)
    start[-1] = length - 6
    want = [oracle.commit(_np(t[-1:])[None], path[-1:], counts[-1:], start[-1:])[0, 0]
            for t in (keys, values, weights.transpose(1, 2))]
    before = [t[-2].clone() for t in (keys, values, weights)]
    accepted = step.AcceptedPath(_gpu(path, torch.int32), _gpu(counts, torch.int32),
                                 _gpu(start, torch.int64))
    cache.qwen3_commit_tree(keys, values, accepted, weights=weights)
    for t, w in zip((keys, values, weights.transpose(1, 2)), want):
        np.testing.assert_array_equal(_np(t[-1]), w)
    lengths = np.full(batch, 5)
    lengths[-1] = length - 2
    kept = oracle.evict(_np(weights[-1:])[None], lengths[-1:], 1000, 3, 10)[0, 0]
    new, got = cache.qwen3_evict(keys, values, weights, _gpu(lengths, torch.int64), 1000, 3, 10)
    assert new.tolist() == [5] * 63 + [1000]
    np.testing.assert_array_equal(got[-1].cpu(), kept)
    for h in range(heads):
        for t, w in zip((keys[-1, :, h], values[-1, :, h], weights[-1, h, :, None]), want):
            w = w[:, h] if w.ndim == 3 else w[:, h, None]
            np.testing.assert_array_equal(_np(t[:1000]), w[kept[h]])
            np.testing.assert_array_equal(_np(t[1000:]), w[1000:])
    for t, b in zip((keys, values, weights), before):
        assert torch.equal(t[-2], b)
    assert not keys[:-2].any() and not values[:-2].any()
