"""What speculative decoding and bounded caches cost: attention for a tree of
drafted tokens over a cache, with and without accumulated attention weights,
the acceptance of a tree with its cache commit, and eviction by weight.

``listed()`` and ``draw()`` give cases, ``prepare()`` a case's inputs on the
GPU, ``run()`` one pass (``own``: the package's operators, otherwise plain
torch in float32), ``exact()`` the same results in float64 and ``work()`` the
bytes and operations that a pass cannot do without.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EOS = (151643, 151645)


def listed():
    return [
        # One request, a chain-like tree of a few drafts in the shortest cache
        # bucket: a latency-bound layer call.
        dict(name="qwen3 tree 1x6 L256", op="qwen3", batch=1, nodes=6, length=256, heads=16,
             kv_heads=8, dim=128, dtype="bf16", ragged=False, ahead=0, weights=False),
        # The full serving batch and cache with a 16-node tree per row.
        dict(name="qwen3 tree 64x16 L1024", op="qwen3", batch=64, nodes=16, length=1024, heads=16,
             kv_heads=8, dim=128, dtype="bf16", ragged=False, ahead=0, weights=False),
        # Wide trees over long caches, rows of unequal tree sizes.
        dict(name="qwen3 tree 8x64 L8192", op="qwen3", batch=8, nodes=64, length=8192, heads=16,
             kv_heads=8, dim=128, dtype="bf16", ragged=True, ahead=0, weights=False),
        # Whisper decoder self-attention: the headline batch, eight drafts a row.
        dict(name="whisper tree 64x8 L448", op="whisper", batch=64, nodes=8, length=448, heads=20,
             kv_heads=20, dim=64, dtype="bf16", ragged=True, ahead=0, weights=False),
        # The smallest Whisper in float32, odd sizes.
        dict(name="whisper tree f32 7x5 L448", op="whisper", batch=7, nodes=5, length=448, heads=6,
             kv_heads=6, dim=64, dtype="f32", ragged=True, ahead=0, weights=False),
        # Single-token steps of the full batch that keep the weights for eviction.
        dict(name="qwen3 weights 64x1 L1024", op="qwen3", batch=64, nodes=1, length=1024, heads=16,
             kv_heads=8, dim=128, dtype="bf16", ragged=False, ahead=300, weights=True),
        # A few long rows, a short chain each, positions past evicted slots.
        dict(name="qwen3 weights 3x4 L16384", op="qwen3", batch=3, nodes=4, length=16384, heads=16,
             kv_heads=8, dim=128, dtype="bf16", ragged=True, ahead=1000, weights=True),
        # Acceptance and commit: one request; the Qwen3 batch over all 28
        # layers; Whisper's head-major cache over the turbo model's 4 layers.
        dict(name="accept qwen3 1x6", op="accept", batch=1, nodes=6, length=256, layers=28,
             kv_heads=8, dim=128, dtype="bf16", heads_first=False, ragged=False),
        dict(name="accept qwen3 64x16", op="accept", batch=64, nodes=16, length=512, layers=28,
             kv_heads=8, dim=128, dtype="bf16", heads_first=False, ragged=True),
        dict(name="accept whisper 64x8", op="accept", batch=64, nodes=8, length=448, layers=4,
             kv_heads=20, dim=64, dtype="bf16", heads_first=True, ragged=True),
        # Halving every row of the full batch in one layer.
        dict(name="evict 64 L1024 to 512", op="evict", batch=64, length=1024, budget=512, sink=4,
             recent=64, layers=1, kv_heads=8, dim=128, dtype="bf16", heads_first=False),
        # Two long rows to a quarter.
        dict(name="evict 2 L16384 to 4096", op="evict", batch=2, length=16384, budget=4096, sink=8,
             recent=1024, layers=1, kv_heads=8, dim=128, dtype="bf16", heads_first=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("qwen3", "qwen3", "whisper", "weights", "weights", "accept", "evict"))
    if op in ("qwen3", "whisper", "weights"):
        weights = op == "weights"
        nodes = _log_int(rng, 1, 8 if weights else 64)
        batch = _log_int(rng, 1, 64)
        if op == "whisper":
            kv_heads = heads = rng.choice((6, 8, 12, 16, 20))
            dim, length = 64, _log_int(rng, nodes + 32, 448)
        else:
            kv_heads = rng.choice((1, 2, 4, 8))
            heads = kv_heads * (rng.choice((1, 2)) if weights else rng.choice((1, 2, 4)))
            dim = rng.choice((64, 128))
            length = _log_int(rng, nodes + 32, max(nodes + 33, min(16384 if weights else 8192,
                                                                   49152 // batch)))
        batch = max(1, min(batch, (1 << 22) // (nodes * length)))
        dtype = "f32" if rng.random() < 0.2 else "bf16"
        if dtype == "f32":  # the float32 kernels serve small models
            batch, length = min(batch, 8), min(length, 1024)
        return dict(op="whisper" if op == "whisper" else "qwen3", batch=batch, nodes=nodes,
                    length=length, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                    ragged=rng.random() < 0.5,
                    ahead=0 if op == "whisper" else rng.choice((0, 17, 500)), weights=weights)
    if op == "accept":
        batch, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
        heads_first = rng.random() < 0.5
        return dict(op="accept", batch=batch, nodes=nodes,
                    length=_log_int(rng, nodes + 32, 448), layers=rng.randint(1, 8),
                    kv_heads=rng.choice((2, 6, 8, 20)), dim=rng.choice((64, 128)),
                    dtype=rng.choice(("bf16", "f32")), heads_first=heads_first,
                    ragged=rng.random() < 0.5)
    batch = _log_int(rng, 1, 64)
    length = _log_int(rng, 64, min(16384, 65536 // batch))
    budget = _log_int(rng, 16, length)
    sink = rng.randint(0, budget // 4)
    return dict(op="evict", batch=batch, length=length, budget=budget, sink=sink,
                recent=rng.randint(0, budget - sink), layers=1, kv_heads=rng.choice((1, 4, 8)),
                dim=rng.choice((64, 128)), dtype=rng.choice(("bf16", "f32")),
                heads_first=rng.random() < 0.3)


# ---------------------------------------------------------------- the inputs


def _trees(rng, batch, nodes, ragged):
    """Random trees: ``parents``, ``counts``, the ancestors' bit masks (each
    node its own ancestor) and depths, as arrays over (batch, nodes)."""
    parents = np.full((batch, nodes), -1, np.int64)
    ancestors = np.zeros((batch, nodes), np.uint64)
    depths = np.zeros((batch, nodes), np.int64)
    rows = np.arange(batch)
    counts = rng.integers((nodes + 1) // 2, nodes + 1, batch) if ragged else np.full(batch, nodes)
    for i in range(nodes):
        if i:
            parents[:, i] = rng.integers(max(0, i - 4), i, batch)
            ancestors[:, i] = ancestors[rows, parents[:, i]]
            depths[:, i] = depths[rows, parents[:, i]] + 1
        ancestors[:, i] |= np.uint64(1 << i)
        gone = i >= counts
        ancestors[gone, i] = 0
        depths[gone, i] = 0
    return parents, counts, ancestors.view(np.int64), depths


def _on_gpu(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV, dtype)


def _cache(gen, case, gain=1.0):
    """A cache (layers, batch, ...) in the family's layout."""
    c = case
    shape = ((c["kv_heads"], c["length"]) if c["heads_first"] else (c["length"], c["kv_heads"]))
    shape = (c["layers"], c["batch"], *shape, c["dim"])
    return torch.randn(shape, generator=gen, device=DEV, dtype=DTYPES[c["dtype"]]).mul_(gain)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return {"qwen3": _prepare_attention, "whisper": _prepare_attention, "accept": _prepare_accept,
            "evict": _prepare_evict}[case["op"]](case, rng, gen)


def _prepare_attention(case, rng, gen):
    c = case
    b, n, length, dim = c["batch"], c["nodes"], c["length"], c["dim"]
    dtype = DTYPES[c["dtype"]]
    parents, counts, ancestors, depths = _trees(rng, b, n, c["ragged"])
    lengths = rng.integers(length // 4, length - n + 1, b)
    s = dict(case=c, parents=_on_gpu(parents, torch.int32), counts=_on_gpu(counts, torch.int32),
             ancestors=_on_gpu(ancestors, torch.int64), depths=_on_gpu(depths, torch.int32),
             lengths=_on_gpu(lengths, torch.int64),
             positions=_on_gpu(lengths + c["ahead"], torch.int64))
    layout = dict(c, layers=1, heads_first=c["op"] == "whisper")
    s["keys"], s["values"] = _cache(gen, layout, 1.5)[0], _cache(gen, layout)[0]
    if c["op"] == "whisper":  # views of the (batch, nodes, heads * dim) projections
        for name in ("query", "key", "value"):
            x = torch.randn((b, n, c["heads"] * dim), generator=gen, device=DEV, dtype=dtype)
            s[name] = x.view(b, n, c["heads"], dim).transpose(1, 2)
    else:
        width = (c["heads"] + 2 * c["kv_heads"]) * dim
        s["qkv"] = torch.randn((b, n, width), generator=gen, device=DEV, dtype=dtype)
        for name in ("q_norm", "k_norm"):
            s[name] = (1 + 0.1 * torch.randn(dim, generator=gen, device=DEV)).to(dtype)
        angles = torch.arange(length + c["ahead"], device=DEV, dtype=torch.float64)[:, None] \
            * 1e6 ** (-torch.arange(0, dim, 2, device=DEV, dtype=torch.float64) / dim)
        angles = torch.cat((angles, angles), 1)
        s["cos"], s["sin"] = angles.cos().to(dtype), angles.sin().to(dtype)
    if c["weights"]:
        s["weights"] = torch.rand((b, c["kv_heads"], length), generator=gen, device=DEV)
    return s


def _prepare_accept(case, rng, gen):
    c = case
    b, n = c["batch"], c["nodes"]
    parents, counts, ancestors, depths = _trees(rng, b, n, c["ragged"])
    chosen = rng.integers(0, 150000, (b, n))
    # A draft is its parent's chosen token in three cases of four.
    drafts = np.take_along_axis(chosen, np.maximum(parents, 0), 1)
    drafts = np.where(rng.random((b, n)) < 0.75, drafts, rng.integers(0, 150000, (b, n)))
    stop = rng.random((b, n)) < 0.02
    chosen = np.where(stop, rng.choice(EOS, (b, n)), chosen)
    position = rng.integers(c["length"] // 4, c["length"] - n, b)
    finished = rng.random(b) < (0.1 if c["ragged"] else 0.0)
    # Tokens, positions and the generated tokens lie in one buffer, so that a
    # pass restores them with one copy.
    generated = rng.integers(0, 150000, b * c["length"])
    packed = np.concatenate((drafts[:, 0], position, generated))
    return dict(case=c, parents=_on_gpu(parents, torch.int32), counts=_on_gpu(counts, torch.int32),
                chosen=_on_gpu(chosen, torch.int64), drafts=_on_gpu(drafts, torch.int64),
                logprob=-torch.rand((b, n), generator=gen, device=DEV),
                packed=_on_gpu(packed, torch.int64), start_packed=_on_gpu(packed, torch.int64),
                end=_on_gpu(position + rng.integers(n // 2 + 1, 200, b), torch.int64),
                finished=_on_gpu(finished, torch.bool), start_finished=_on_gpu(finished, torch.bool),
                sums=torch.zeros(b, device=DEV), keys=_cache(gen, c), values=_cache(gen, c))


def _prepare_evict(case, rng, gen):
    c = case
    lengths = rng.integers((c["budget"] + c["length"]) // 2, c["length"] + 1, c["batch"])
    # Few keys gather most of the weight; some ties, as keys that got none.
    weights = torch.rand((c["layers"], c["batch"], c["kv_heads"], c["length"]), generator=gen,
                         device=DEV).pow_(4).sub_(0.01).clamp_(min=0)
    return dict(case=c, lengths=_on_gpu(lengths, torch.int64), weights=weights.clone(),
                start_weights=weights, keys=_cache(gen, c), values=_cache(gen, c))


# ------------------------------------------------------------------ one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return {"qwen3": _own_qwen3, "whisper": _own_whisper, "accept": _own_accept,
                "evict": _own_evict}[op](state)
    return {"qwen3": _plain_attention, "whisper": _plain_attention, "accept": _plain_accept,
            "evict": _plain_evict}[op](state)


def _own_tree(s):
    from asrback_b200 import attention

    return attention.DraftTree(s["parents"], s["counts"], s["ancestors"], s["depths"])


def _attention_outputs(s, out):
    got = dict(out=out, keys=s["keys"], values=s["values"])
    return dict(got, weights=s["weights"]) if s["case"]["weights"] else got


def _own_qwen3(s):
    from asrback_b200 import attention

    c = s["case"]
    out = attention.qwen3_attention_tree(
        s["qkv"], s["q_norm"], s["k_norm"], 1e-6, s["cos"], s["sin"], s["positions"], _own_tree(s),
        s["keys"], s["values"], c["heads"], c["kv_heads"], lengths=s["lengths"],
        weights=s.get("weights"))
    return _attention_outputs(s, out)


def _own_whisper(s):
    from asrback_b200 import attention

    out = attention.whisper_self_attention_tree(
        s["query"], s["key"], s["value"], s["keys"], s["values"], s["lengths"], _own_tree(s),
        weights=s.get("weights"))
    return _attention_outputs(s, out)


def _unpacked(s):
    b = s["case"]["batch"]
    return s["packed"][:b], s["packed"][b:2 * b], s["packed"][2 * b:].view(b, -1)


def _own_accept(s):
    from asrback_b200 import attention, cache, step

    s["packed"].copy_(s["start_packed"])  # every pass starts from the same state
    s["finished"].copy_(s["start_finished"])
    s["sums"].zero_()
    tree = attention.draft_tree(s["parents"], s["counts"])
    tokens, position, generated = _unpacked(s)
    accepted = step.accept_tree(tree, s["drafts"], s["chosen"], s["logprob"], tokens, position,
                                s["end"], s["finished"], s["sums"], generated, EOS)
    commit = (cache.whisper_commit_tree if s["case"]["heads_first"]
              else cache.qwen3_commit_tree)
    commit(s["keys"], s["values"], accepted)
    return dict(depths=tree.depths, ancestors=tree.ancestors, path=accepted.path,
                counts=accepted.counts, state=s["packed"], finished=s["finished"], sums=s["sums"],
                keys=s["keys"], values=s["values"])


def _own_evict(s):
    from asrback_b200 import cache

    c = s["case"]
    s["weights"].copy_(s["start_weights"])  # every pass evicts by the same weights
    evict = cache.whisper_evict if c["heads_first"] else cache.qwen3_evict
    lengths, kept = evict(s["keys"], s["values"], s["weights"], s["lengths"], c["budget"],
                          sink=c["sink"], recent=c["recent"])
    return dict(lengths=lengths, kept=kept, keys=s["keys"], values=s["values"],
                weights=s["weights"])


def _rotate(x, weight, cos, sin):
    """Per-head RMS norm, then rotation by halves (``x`` (b, n, h, d))."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight
    first, second = x.chunk(2, -1)
    return x * cos[:, :, None] + torch.cat((-second, first), -1) * sin[:, :, None]


def _plain_attention(s):
    c = s["case"]
    b, n, kvh, dim, length = c["batch"], c["nodes"], c["kv_heads"], c["dim"], c["length"]
    g = c["heads"] // kvh
    node = torch.arange(n, device=DEV)
    live = node < s["counts"][:, None]
    rows = torch.arange(b, device=DEV)[:, None].expand(b, n)[live]
    slots = (s["lengths"][:, None] + node)[live]
    if c["op"] == "whisper":
        q, k, v = (s[name].transpose(1, 2).float() for name in ("query", "key", "value"))
        keys, values = s["keys"].transpose(1, 2), s["values"].transpose(1, 2)
    else:
        q, k, v = s["qkv"].float().view(b, n, -1, dim).split((c["heads"], kvh, kvh), 2)
        at = (s["positions"][:, None] + s["depths"]).clamp(max=s["cos"].shape[0] - 1)
        cos, sin = s["cos"][at].float(), s["sin"][at].float()
        q, k = _rotate(q, s["q_norm"].float(), cos, sin), _rotate(k, s["k_norm"].float(), cos, sin)
        keys, values = s["keys"], s["values"]
    keys[rows, slots] = k[live].to(keys.dtype)
    values[rows, slots] = v[live].to(values.dtype)
    # Node i sees slot j if it is older than the tree or holds an ancestor.
    ancestor = (s["ancestors"][:, :, None] >> node) & 1 == 1
    age = torch.arange(length, device=DEV) - s["lengths"][:, None]
    inside = ancestor.gather(2, age.clamp(0, n - 1)[:, None].expand(b, n, length))
    visible = torch.where(age[:, None] < 0, live[:, :, None], inside & (age < n)[:, None])
    q = q.reshape(b, n, kvh, g, dim).permute(0, 2, 3, 1, 4).reshape(b, kvh, g * n, dim)
    scores = torch.matmul(q, keys.float().permute(0, 2, 3, 1)).mul_(dim ** -0.5)
    seen = visible[:, None, None].expand(b, kvh, g, n, length).reshape(b, kvh, g * n, length)
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    scores.div_(torch.where(total == 0, 1.0, total))
    out = torch.matmul(scores, values.float().transpose(1, 2))
    out = out.view(b, kvh, g, n, dim).permute(0, 3, 1, 2, 4).reshape(b, n, -1)
    if c["weights"]:
        gained = scores.sum(2)
        fresh = ((age >= 0) & (age < s["counts"][:, None]))[:, None]
        s["weights"].masked_fill_(fresh, 0).add_(gained)
    return _attention_outputs(s, out.to(keys.dtype))


def _move(cache, source, moved, heads_first):
    """Rows of ``cache`` (layers, batch, length, ...) replaced by the rows
    ``source`` (batch or layers x batch, heads, length) where ``moved``."""
    view = cache.transpose(2, 3) if not heads_first else cache
    at = source[..., None].expand(view.shape)
    view.copy_(torch.where(moved[..., None], view.gather(3, at), view))


def _plain_accept(s):
    c = s["case"]
    b, n, length = c["batch"], c["nodes"], c["length"]
    s["packed"].copy_(s["start_packed"])
    s["finished"].copy_(s["start_finished"])
    s["sums"].zero_()
    tokens, position, generated = _unpacked(s)
    node = torch.arange(n, device=DEV)
    live = node < s["counts"][:, None]
    # Ancestors: powers of the parent relation, squared until all are joined.
    parent = s["parents"][:, :, None] == node
    above = ((parent & live[:, :, None]) | torch.eye(n, dtype=torch.bool, device=DEV)).float()
    above = torch.matmul(above, above).clamp_(max=1)
    above = torch.matmul(above, above).clamp_(max=1)
    above = torch.matmul(above, above).clamp_(max=1)
    above = torch.matmul(above, above).clamp_(max=1)
    above = torch.matmul(above, above).clamp_(max=1)
    above = (torch.matmul(above, above) > 0) & live[:, :, None]
    depths = (above.sum(-1) - 1).clamp_(min=0)
    ancestors = (above.long() << node).sum(-1)
    # A child stands if it holds its parent's token and no elder sibling does.
    at = s["parents"].long().clamp(min=0)
    fits = live & (s["parents"] >= 0) & (s["drafts"] == s["chosen"].gather(1, at))
    elder = (node[:, None] > node) & (s["parents"][:, :, None] == s["parents"][:, None])
    fits &= ~(elder & fits[:, None]).any(-1)
    fits[:, 0] = live[:, 0] & ~s["finished"]
    # The walk ends behind a node whose token ends the row.
    eos = torch.isin(s["chosen"], torch.tensor(EOS, device=DEV))
    ends = eos | (position[:, None] + depths + 1 >= s["end"][:, None])
    before = above & ~torch.eye(n, dtype=torch.bool, device=DEV)
    taken = live & above[:, :, 0] & ~(above & ~fits[:, None]).any(-1)
    taken &= ~(before & ends[:, None]).any(-1)
    counts = taken.sum(-1)
    order = torch.where(taken, depths, n).argsort(dim=1, stable=True)
    path = torch.where(node < counts[:, None], order, -1)
    start = position.clone()
    last = order.gather(1, (counts - 1).clamp(min=0)[:, None])[:, 0]
    tokens.copy_(torch.where(counts > 0, s["chosen"].gather(1, last[:, None])[:, 0], tokens))
    rows = torch.arange(b, device=DEV)[:, None].expand(b, n)[taken]
    generated[rows, (start[:, None] + depths + 1)[taken]] = s["chosen"][taken]
    s["sums"].add_((s["logprob"] * taken).sum(-1))
    position.add_(counts)
    s["finished"].logical_or_((taken & ends).any(-1))
    # The accepted nodes' cache rows close up behind the row's old end.
    age = torch.arange(length, device=DEV) - start[:, None]
    moved = (age >= 0) & (age < counts[:, None])
    source = start[:, None] + path.gather(1, age.clamp(0, n - 1))
    source = torch.where(moved, source, 0)
    shape = (c["layers"], b, c["kv_heads"], length)
    source, moved = (x[None, :, None].expand(shape) for x in (source, moved))
    _move(s["keys"], source, moved, c["heads_first"])
    _move(s["values"], source, moved, c["heads_first"])
    return dict(depths=depths.int(), ancestors=ancestors, path=path.int(), counts=counts.int(),
                state=s["packed"], finished=s["finished"], sums=s["sums"], keys=s["keys"],
                values=s["values"])


def _plain_evict(s):
    c = s["case"]
    length, budget = c["length"], c["budget"]
    s["weights"].copy_(s["start_weights"])
    weights, lengths = s["weights"], s["lengths"][:, None, None]
    slot = torch.arange(length, device=DEV)
    rank = torch.where(torch.isnan(weights), -math.inf, weights)
    rank = torch.where((slot < c["sink"]) | (slot >= lengths - c["recent"]), math.inf, rank)
    # Slots past the row's end come last, behind the lowest weights too.
    inside = (slot < lengths).expand(rank.shape)
    order = torch.where(inside, rank, -math.inf).sort(stable=True, dim=-1, descending=True).indices
    full = torch.where(inside.gather(-1, order), 0, 1).sort(stable=True, dim=-1).indices
    kept = order.gather(-1, full)[..., :budget]
    whole = (lengths <= budget).expand(kept.shape)
    kept = torch.where(whole, slot[:budget], kept.sort(-1).values)
    filled = slot[:budget] < lengths
    moved = torch.zeros(weights.shape, dtype=torch.bool, device=DEV)
    moved[..., :budget] = ~whole
    source = torch.zeros(weights.shape, dtype=torch.int64, device=DEV)
    source[..., :budget] = kept
    weights.copy_(torch.where(moved, weights.gather(-1, source), weights))
    _move(s["keys"], source, moved, c["heads_first"])
    _move(s["values"], source, moved, c["heads_first"])
    return dict(lengths=s["lengths"].clamp(max=budget), keys=s["keys"], values=s["values"],
                kept=torch.where(filled, kept, -1).int(), weights=weights)


# ----------------------------------------------------------- float64 results


def exact(case, seed):
    s = prepare(case, seed)
    return {"qwen3": _exact_attention, "whisper": _exact_attention, "accept": _exact_accept,
            "evict": _exact_evict}[case["op"]](s)


def _exact_attention(s):
    c = s["case"]
    n, heads, kvh, dim = c["nodes"], c["heads"], c["kv_heads"], c["dim"]
    dtype, g = DTYPES[c["dtype"]], heads // kvh
    turned = c["op"] == "whisper"
    keys, values = s["keys"].double(), s["values"].double()
    weights = s["weights"].double() if c["weights"] else None
    out = torch.zeros((c["batch"], n, heads, dim), dtype=torch.float64, device=DEV)
    lengths, counts = s["lengths"].tolist(), s["counts"].tolist()
    positions, depths = s["positions"].tolist(), s["depths"].tolist()
    for b in range(c["batch"]):
        if turned:
            q, k, v = (s[x][b].double().transpose(0, 1) for x in ("query", "key", "value"))
        else:
            x = s["qkv"][b].double().reshape(n, -1, dim)
            at = [min(positions[b] + d, s["cos"].shape[0] - 1) for d in depths[b]]
            cos, sin = s["cos"][at].double()[:, None], s["sin"][at].double()[:, None]
            half, turnings = dim // 2, []
            for y, w in ((x[:, :heads], s["q_norm"]), (x[:, heads:heads + kvh], s["k_norm"])):
                y = y / (y.pow(2).sum(-1, keepdim=True) / dim + 1e-6).sqrt() * w.double()
                low, high = y[..., :half], y[..., half:]
                turnings.append(torch.cat((low * cos[..., :half] - high * sin[..., :half],
                                           high * cos[..., half:] + low * sin[..., half:]), -1))
            (q, k), v = turnings, x[:, heads + kvh:]
        m, start = counts[b], lengths[b]
        kb = keys[b].transpose(0, 1) if turned else keys[b]
        vb = values[b].transpose(0, 1) if turned else values[b]
        kb[start:start + m], vb[start:start + m] = k[:m].to(dtype).double(), v[:m].to(dtype).double()
        masks = [[(a >> j) & 1 == 1 for j in range(m)] for a in s["ancestors"][b, :m].tolist()]
        hidden = torch.zeros((m, start + m), dtype=torch.bool, device=DEV)
        hidden[:, start:] = ~torch.tensor(masks, dtype=torch.bool, device=DEV).reshape(m, m)
        for h in range(kvh):
            logits = torch.tensordot(q[:m, h * g:(h + 1) * g], kb[:start + m, h], ([2], [1]))
            logits = (logits / math.sqrt(dim)).masked_fill(hidden[:, None], -math.inf)
            p = torch.softmax(logits, -1)
            out[b, :m, h * g:(h + 1) * g] = torch.tensordot(p, vb[:start + m, h], ([2], [0]))
            if weights is not None:
                weights[b, h, start:start + m] = 0
                weights[b, h, :start + m] += p.sum((0, 1))
    got = dict(out=out.reshape(c["batch"], n, heads * dim), keys=keys, values=values)
    return got if weights is None else dict(got, weights=weights)


def _exact_accept(s):
    chosen, drafts, logprob = (s[x].tolist() for x in ("chosen", "drafts", "logprob"))
    parents, counts, end = (s[x].tolist() for x in ("parents", "counts", "end"))
    done, size = s["start_finished"].tolist(), s["case"]["batch"]
    position = s["start_packed"][size:2 * size].tolist()
    sums = [0.0] * len(done)
    for b, over in enumerate(done):
        at, place = (None if over or not counts[b] else 0), position[b]
        while at is not None:
            token, place = chosen[b][at], place + 1
            sums[b] += logprob[b][at]
            if token in EOS or place >= end[b]:
                break
            at = next((i for i in range(at + 1, counts[b])
                       if parents[b][i] == at and drafts[b][i] == token), None)
    return dict(depths=None, ancestors=None, path=None, counts=None, state=None, finished=None,
                sums=torch.tensor(sums, dtype=torch.float64), keys=None, values=None)


def _exact_evict(s):
    c = s["case"]
    weights = s["start_weights"].double().cpu().numpy()
    for b, m in enumerate(s["lengths"].tolist()):
        if m <= c["budget"]:
            continue
        old = set(range(min(c["sink"], m))) | set(range(max(0, m - c["recent"]), m))
        middle = np.array([j for j in range(m) if j not in old], np.int64)
        for layer in range(c["layers"]):
            for h in range(c["kv_heads"]):
                row = weights[layer, b, h]
                best = middle[np.lexsort((middle, -row[middle]))][:c["budget"] - len(old)]
                kept = np.sort(np.concatenate((best, np.array(sorted(old), np.int64))))
                row[:c["budget"]] = row[kept].copy()
    return dict(lengths=None, kept=None, keys=None, values=None, weights=torch.from_numpy(weights))


# ------------------------------------------------- what a pass cannot do without


def work(case):
    c = case
    size = 2 if c["dtype"] == "bf16" else 4
    b, d, kvh = c["batch"], c["dim"], c["kv_heads"]
    if c["op"] in ("qwen3", "whisper"):
        n, h = c["nodes"], c["heads"]
        live = n * (0.75 if c["ragged"] else 1.0)
        cached = (c["length"] // 4 + c["length"] - n) / 2
        moved = 2 * cached * kvh * d + n * (h + 2 * kvh) * d + n * h * d + 2 * live * kvh * d
        held = 8 * (cached + live) * kvh if c["weights"] else 0
        return dict(bytes=b * (moved * size + held + 20 * n),
                    flops=4.0 * b * h * live * (cached + live / 2) * d)
    if c["op"] == "accept":  # the accepted rows' keys and values once in and out
        n = c["nodes"]
        taken = 1 + min(2.0, 0.4 * (n - 1))
        return dict(bytes=b * n * 48.0 + 4 * size * b * c["layers"] * kvh * d * (taken - 1),
                    flops=0)
    held = ((c["budget"] + c["length"]) / 2 + c["length"]) / 2
    rows = b * c["layers"] * kvh
    return dict(bytes=rows * (4 * held + 12 * c["budget"] + 4 * c["budget"] * d * size), flops=0)
