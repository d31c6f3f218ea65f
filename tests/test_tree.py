"""Draft trees and eviction without a GPU: the host's argument checks refuse bad
calls before any launch, and the float64 oracle agrees with independent
restatements (masked softmax attention, one greedy step at a time, a sort)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from asrback_b200 import _native, attention, cache, step
from oracle import tree as oracle

P = 1 << 20  # a pointer that no refused call reads


def _status(name: str, args: dict, **changes) -> int:
    assert set(changes) <= set(args), changes
    values = {**args, **changes}.values()
    rc = getattr(_native.load(), name)(*values)
    error = _native.load().asrback_last_error()
    # The arguments as one array of words: the same answer.
    words = [0 if x is None else ctypes.addressof(x) if isinstance(x, ctypes.Array) else x
             for x in values]
    assert getattr(_native.load(), name + "_packed")(_native._PACKED[name](*words)) == rc
    assert _native.load().asrback_last_error() == error
    return rc


PLAN = dict(batch=2, nodes=5, parents=P, parents_stride=5, counts=None, ancestors=P, depths=P,
            live_counts=P, status=None, stream=None)

ATTENTION = dict(
    dtype=_native.BF16, batch=2, nodes=5, heads=16, kv_heads=8, head_dim=128, cache_length=64,
    query=P, q_b=5 * 4096, q_n=4096, q_h=128, key=P, k_b=5 * 4096, k_n=4096, k_h=128, value=P,
    v_b=5 * 4096, v_n=4096, v_h=128, q_norm=P, k_norm=P, eps=1e-6, cos=P, sin=P, table_stride=128,
    table_length=100, positions=P, ancestors=P, depths=P, counts=P, lengths=P, key_cache=P,
    value_cache=P, c_b=64 * 1024, c_p=1024, c_h=128, out=P, o_b=5 * 2048, o_n=2048, o_h=128,
    weights=None, w_b=8 * 64, w_h=64, scale=0.1, workspace=P, workspace_bytes=1 << 40, status=None,
    stream=None)

ACCEPT = dict(
    batch=2, nodes=5, parents=P, parents_stride=5, counts=P, drafts=P, drafts_stride=5, chosen=P,
    chosen_stride=5, logprob=P, logprob_stride=5, tokens=P, tokens_stride=1, position=P, end=P,
    finished=P, sums=P, generated=P, generated_stride=100, generated_cols=100, lengths=None,
    eos=(ctypes.c_int64 * 2)(1, 2), n_eos=2, path=P, accepted=P, start=P, status=None, stream=None)

COMMIT = dict(
    dtype=_native.BF16, layers=2, batch=2, nodes=5, heads=8, head_dim=128, length=64, key_cache=P,
    value_cache=P, c_l=2 * 64 * 1024, c_b=64 * 1024, c_p=1024, c_h=128, weights=P, w_l=2 * 8 * 64,
    w_b=8 * 64, w_h=64, path=P, counts=P, start=P, status=None, stream=None)

EVICT = dict(
    dtype=_native.BF16, layers=2, batch=2, heads=8, head_dim=128, length=64, key_cache=P,
    value_cache=P, c_l=2 * 64 * 1024, c_b=64 * 1024, c_p=1024, c_h=128, weights=P, w_l=2 * 8 * 64,
    w_b=8 * 64, w_h=64, lengths=P + 64, budget=32, sink=4, recent=8, new_lengths=P, kept=P, status=None,
    stream=None)

_ODD = P + 8  # not on a 16-byte boundary

REFUSED = {
    "asrback_draft_tree": (PLAN, [
        dict(batch=0), dict(nodes=0), dict(nodes=65), dict(parents=None), dict(ancestors=None),
        dict(depths=None), dict(live_counts=None), dict(parents_stride=4),
        dict(parents_stride=-5)]),
    "asrback_tree_attention": (ATTENTION, [
        dict(dtype=7), dict(batch=0), dict(batch=1025), dict(nodes=0), dict(nodes=65),
        dict(heads=12), dict(kv_heads=0), dict(head_dim=96), dict(cache_length=0),
        dict(cache_length=(1 << 24) + 1), dict(query=None), dict(key=None), dict(value=None),
        dict(key_cache=None), dict(value_cache=None), dict(out=None), dict(ancestors=None),
        dict(depths=None), dict(counts=None), dict(lengths=None), dict(k_norm=None),
        dict(cos=None), dict(sin=None), dict(positions=None), dict(table_length=0),
        dict(table_stride=64), dict(q_norm=None), dict(q_b=-8), dict(q_n=4097), dict(k_h=132),
        dict(v_b=12), dict(c_p=64), dict(c_h=64), dict(c_b=0), dict(o_h=64), dict(o_n=0),
        dict(o_b=0), dict(query=_ODD), dict(key_cache=_ODD), dict(cos=_ODD), dict(out=_ODD),
        dict(weights=P, nodes=9), dict(weights=P, w_b=63), dict(weights=P, w_h=0)]),
    "asrback_accept_tree": (ACCEPT, [
        dict(batch=0), dict(nodes=65), dict(parents=None), dict(counts=None), dict(drafts=None),
        dict(chosen=None), dict(logprob=None), dict(tokens=None), dict(position=None),
        dict(end=None), dict(finished=None), dict(sums=None), dict(generated=None),
        dict(path=None), dict(accepted=None), dict(start=None), dict(parents_stride=4),
        dict(drafts_stride=4), dict(chosen_stride=0), dict(logprob_stride=4),
        dict(tokens_stride=0), dict(generated_cols=0), dict(generated_stride=99),
        dict(n_eos=-1), dict(n_eos=99), dict(eos=None)]),
    "asrback_commit_tree": (COMMIT, [
        dict(dtype=7), dict(layers=0), dict(batch=0), dict(batch=65536), dict(nodes=0),
        dict(nodes=65), dict(heads=0), dict(head_dim=32), dict(length=0), dict(key_cache=None),
        dict(value_cache=None), dict(key_cache=_ODD), dict(c_l=0), dict(c_b=0), dict(c_p=64),
        dict(c_h=4), dict(c_p=1028), dict(w_l=0), dict(w_b=32), dict(w_h=63), dict(path=None),
        dict(counts=None), dict(start=None)]),
    "asrback_evict": (EVICT, [
        dict(dtype=7), dict(layers=0), dict(batch=0), dict(heads=0), dict(head_dim=32),
        dict(length=0), dict(budget=0), dict(budget=65), dict(sink=-1), dict(recent=-1),
        dict(sink=25), dict(recent=29), dict(layers=256, batch=256), dict(key_cache=None),
        dict(value_cache=_ODD), dict(c_l=0), dict(c_b=0), dict(c_p=64), dict(c_h=0), dict(w_l=0),
        dict(w_b=32), dict(w_h=0), dict(weights=None), dict(lengths=None),
        dict(new_lengths=None), dict(kept=None), dict(new_lengths=P + 64)]),
}


@pytest.mark.parametrize("name,args,changes", [
    pytest.param(name, args, change, id=f"{name}-{'-'.join(f'{k}={v}' for k, v in change.items())}")
    for name, (args, cases) in REFUSED.items() for change in cases])
def test_bad_arguments_are_refused(name, args, changes):
    assert _status(name, args, **changes) == _native.ERR_ARGUMENT
    assert _native.load().asrback_last_error()


def test_workspace():
    size = _native.load().asrback_tree_workspace_bytes
    need = size(_native.BF16, 2, 5, 16, 8, 128, 64, 1, 0)
    assert need > 0
    assert size(_native.BF16, 2, 5, 16, 8, 128, 64, 1, 1) > need  # the scores
    assert size(_native.BF16, 0, 5, 16, 8, 128, 64, 1, 0) == 0
    assert _status("asrback_tree_attention", ATTENTION,
                   workspace_bytes=need - 1) == _native.ERR_WORKSPACE
    assert _status("asrback_tree_attention", ATTENTION, workspace=None) == _native.ERR_WORKSPACE
    assert _status("asrback_tree_attention", ATTENTION, workspace=P + 4) == _native.ERR_ARGUMENT


def test_tensors_off_the_gpu_are_refused():
    parents = torch.zeros((2, 3), dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        attention.draft_tree(parents)
    tree = attention.DraftTree(parents, parents[:, 0].contiguous(), parents.long(), parents)
    state = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        step.accept_tree(tree, parents.long(), parents.long(), parents.float(), state, state, state,
                         state.bool(), state.float(), state[:, None], [1])
    rows = torch.zeros((2, 8, 2, 64))
    with pytest.raises((ValueError, TypeError)):
        cache.qwen3_evict(rows, rows.clone(), torch.zeros((2, 2, 8)), state, 4)
    with pytest.raises((ValueError, TypeError)):
        attention.qwen3_attention_tree(
            torch.zeros((2, 3, 6 * 64)), rows[0, 0, 0], rows[0, 0, 0], 1e-6, rows[0, :, 0],
            rows[0, :, 0], state, tree, rows, rows.clone(), 2, 2)


# ---------------------------------------------------------------- the oracle


def _random_trees(rng, batch, nodes):
    parents = np.array([[rng.integers(-1, i) if i else -1 for i in range(nodes)]
                        for _ in range(batch)])
    return parents, rng.integers(0, nodes + 1, batch)


@pytest.mark.parametrize("nodes,heads,kv_heads", [(1, 2, 2), (6, 4, 2), (17, 4, 1)])
def test_oracle_attention_is_a_masked_softmax(nodes, heads, kv_heads):
    rng = np.random.default_rng(nodes)
    batch, length, dim = 3, 40, 8
    parents, counts = _random_trees(rng, batch, nodes)
    lengths = np.array([0, 7, length - nodes])
    q = rng.standard_normal((batch, nodes, heads, dim))
    k, v = rng.standard_normal((2, batch, nodes, kv_heads, dim))
    keys, values = rng.standard_normal((2, batch, length, kv_heads, dim))
    above, _ = oracle.plan(parents, counts)
    got = oracle.tree_attention(q, k, v, keys, values, lengths, above, counts, 0.3)
    for b in range(batch):
        n, m = counts[b], lengths[b]
        assert not got["out"][b, n:].any()
        if n == 0:
            continue
        kk = torch.from_numpy(np.concatenate((keys[b, :m], k[b, :n])))
        vv = torch.from_numpy(np.concatenate((values[b, :m], v[b, :n])))
        group = heads // kv_heads
        mask = torch.from_numpy(np.concatenate((np.ones((n, m), bool), above[b, :n, :n]), 1))
        want = torch.nn.functional.scaled_dot_product_attention(
            torch.from_numpy(q[b, :n]).transpose(0, 1),
            kk.transpose(0, 1).repeat_interleave(group, 0),
            vv.transpose(0, 1).repeat_interleave(group, 0), attn_mask=mask, scale=0.3)
        # float64 on both sides: sums of at most 57 terms of order one.
        np.testing.assert_allclose(got["out"][b, :n], want.transpose(0, 1).numpy(), rtol=0,
                                   atol=1e-13)


def test_oracle_plan_follows_the_parents():
    above, depths = oracle.plan(np.array([[-1, 0, 0, 1, 2, -1]]), np.array([5]))
    assert [np.flatnonzero(row).tolist() for row in above[0]] == [
        [0], [0, 1], [0, 2], [0, 1, 3], [0, 2, 4], []]
    assert depths.tolist() == [[0, 1, 1, 2, 2, 0]]


def test_oracle_acceptance_is_greedy_decoding():
    """A model that maps the tokens so far to the next one: the accepted tokens
    are what it says one step at a time, as many as the drafts foresaw."""
    rng = np.random.default_rng(0)
    for _ in range(1000):
        nodes, vocab = int(rng.integers(1, 9)), 3
        parents, counts = _random_trees(rng, 1, nodes)
        drafts = rng.integers(0, vocab, (1, nodes))
        if len({*zip(parents[0], drafts[0])}) < nodes:
            continue  # of two children with one token only the first is walked
        model = {}

        def after(tokens, model=model):
            return model.setdefault(tokens, int(rng.integers(0, vocab)))

        def path_tokens(i, parents=parents, drafts=drafts):
            return () if i < 0 else (*path_tokens(parents[0, i]), int(drafts[0, i]))

        chosen = np.array([[after(path_tokens(i)) for i in range(nodes)]])
        logprob = rng.standard_normal((1, nodes)).astype(np.float32)
        state = dict(tokens=np.array([9]), position=np.array([4]), end=np.array([4 + 5]),
                     finished=np.array([False]), sum_logprobs=np.zeros(1, np.float32),
                     generated=np.zeros((1, 20), np.int64))
        path, taken, start, new, _ = oracle.accept(parents, counts, drafts, chosen, logprob, state,
                                                   [0])
        assert start[0] == 4 and new["position"][0] == 4 + taken[0]
        so_far = () if counts[0] == 0 else (int(drafts[0, 0]),)
        emitted = []
        while counts[0]:
            emitted.append(after(so_far))
            if emitted[-1] == 0 or len(emitted) == 5:
                break
            so_far = (*so_far, emitted[-1])
            if not any(path_tokens(i) == so_far for i in range(counts[0])
                       if _under(parents[0], i)):
                break
        assert new["generated"][0, 5:5 + taken[0]].tolist() == emitted
        assert taken[0] == len(emitted)


def _under(parents, i):
    """Whether node ``i`` lies in the tree of node 0 (others are not walked)."""
    while i > 0:
        i = parents[i]
    return i == 0


def test_oracle_evict_keeps_the_largest():
    weights = np.array([[[[5., 0., np.nan, 2., 2., 9., 1., 7., 0., 3.]]]], np.float32)
    kept = oracle.evict(weights, np.array([9]), 5, 1, 1)
    assert kept.tolist() == [[[[0, 3, 5, 7, 8]]]]  # of the twos the lower slot
    assert oracle.evict(weights, np.array([3]), 5, 1, 1).tolist() == [[[[0, 1, 2, -1, -1]]]]
