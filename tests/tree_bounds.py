"""How far the draft-tree attention's results may be from the definition, for
inputs on which a fault shows.

The oracle gets the keys that the call wrote, checked apart, as they lie in the
cache: what is left is the query's own error, the float32 sums, and the roundings
of probabilities and outputs. The inputs of :func:`coded` have values that are
not negative, so that an output is the sum of its terms' magnitudes and a bound
relative to these is one relative to the output; each value column counts for
some tiles only, so that one tile left out shows in its column.

With u = 2^-24, half a float32 step:

- a rotated element is a difference of two products of some dozen roundings: 2^-18
  of their magnitudes, and over a row 1.5 * 2^-18 * |q| * |k| (Cauchy-Schwarz;
  the root of 2 for the two products, and bf16 tables); two bf16 parts of it 2^-17;
- a score: (dim + 4) * 2u of its terms' magnitudes, their largest sum ``full``;
- its exponential: 2^-22 (the approximation) and 2^-22 of the exponent, which is
  at most full + log2 of the keys' number, 24 at most;
- d, the sum of these, moves a probability by e^(2 d) (itself and its sum) and
  the sum's own float32 additions by keys * u;
- in bf16, probabilities are rounded (2^-8) and so is the output (2^-8).
"""

from __future__ import annotations

import numpy as np
import torch

from oracle import tree as oracle

TILE = 64


def f64(t):
    return t.detach().double().cpu().numpy()


def position_major(x, t):
    """A cache as (B, L, KVH, D)."""
    return t.transpose(1, 2) if x["family"] == "whisper" else t


def coded(x):
    """``x`` with values that are not negative, key p's in the columns c with
    c = p // 64 (mod D) only: each column tells of every D-th tile."""
    x = dict(x)
    dim = x["dim"]
    values = position_major(x, x["values"]).abs() + 0.5
    tile = torch.arange(values.shape[1], device=values.device) // TILE % dim
    values = values * (torch.arange(dim, device=values.device) == tile[:, None])[None, :, None]
    values = values.to(x["keys"].dtype)
    x["values"] = values.transpose(1, 2).contiguous() if x["family"] == "whisper" else values
    if x["family"] == "whisper":
        x["v"] = x["v"].abs()
    else:
        x["qkv"] = x["qkv"].clone()
        x["qkv"][..., -x["kv_heads"] * dim:].abs_()
    return x


def definition(x, keys=None):
    """The results in float64, given the cache's new ``keys`` (B, L, KVH, D) as the
    call wrote them (None: those of the definition, rounded to the type), and the
    bounds ``d`` (B, N, H) of the scores."""
    heads, kv_heads, dim, bf16 = x["heads"], x["kv_heads"], x["dim"], x["tag"] == "bf16"
    counts, lengths = x["counts"], x["lengths"]
    above, depths = oracle.plan(x["parents"], counts)
    old_keys, old_values = (f64(position_major(x, x[n])) for n in ("keys", "values"))
    rotated = x["family"] == "qwen3"
    if rotated:
        qkv = f64(x["qkv"])
        q, k, v = np.split(qkv.reshape(*qkv.shape[:2], -1, dim), (heads, heads + kv_heads), 2)
        at = np.minimum(x["positions"][:, None] + depths, x["cos"].shape[0] - 1)
        turn = [f64(x[n])[at][:, :, None] for n in ("cos", "sin")]
        q = oracle.norm_rotate(q, f64(x["wq"]), *turn, 1e-6)
        plain = k / np.sqrt((k * k).mean(-1, keepdims=True) + 1e-6) * f64(x["wk"])
        k = oracle.norm_rotate(k, f64(x["wk"]), *turn, 1e-6)
        terms = np.abs(plain * turn[0]) + np.abs(np.roll(plain, dim // 2, -1) * turn[1])
    else:
        q, k, v = (f64(x[n]).transpose(0, 2, 1, 3) for n in "qkv")
        terms = np.zeros_like(k)
    half = 2.0 ** -8 if bf16 else 2.0 ** -24
    if keys is None:
        new = torch.from_numpy(k).to(x["keys"].dtype).double().numpy()
    else:
        new = np.zeros_like(k)
        for b, (n, m) in enumerate(zip(counts, lengths)):
            new[b, :n] = keys[b, m:m + n]
            # One rounding of a float32 norm and rotation (none: the input itself).
            tol = half * np.abs(k[b, :n]) * (1 + 2.0 ** -9) + 2.0 ** -18 * terms[b, :n] \
                if rotated else np.zeros_like(k[b, :n])
            assert (np.abs(new[b, :n] - k[b, :n]) <= tol).all(), "new keys"
    weights = None if x["weights"] is None else f64(x["weights"])
    want = oracle.tree_attention(q, new, v, old_keys, old_values, lengths, above, counts,
                                 dim ** -0.5, weights)
    full = want["reach"][..., 0]
    d = (dim + 4) * 2.0 ** -23 * full + 2.0 ** -22 * (full + 25)
    if rotated:
        reach = np.sqrt((want["keys"] ** 2).sum(-1)).max(1).repeat(heads // kv_heads, 1)[:, None]
        d = d + 1.5 * 2.0 ** -18 * np.sqrt((q * q).sum(-1)) * reach * dim ** -0.5
        if bf16:
            d = d + 2.0 ** -17 * full
    return want, d


def check(x, got):
    """Asserts that ``got`` (out, keys, values, weights; caches (B, L, KVH, D))
    is what a call on ``x`` may give."""
    out, keys, values, weights = got
    keys, values = f64(keys), f64(values)
    want, d = definition(x, keys)
    bf16 = x["tag"] == "bf16"
    half = 2.0 ** -8 if bf16 else 2.0 ** -24
    n_keys = int(x["lengths"].max()) + 64
    share = np.expm1(2 * d) + n_keys * 2.0 ** -24  # of a probability
    tol = half * np.abs(want["out"]) + want["mass"] * (1 + half) * (
        (2.0 ** -8 if bf16 else 0.0) + share[..., None] + n_keys * 2.0 ** -24) * (1 + 2.0 ** -7)
    off = np.abs(f64(out).reshape(want["out"].shape) - want["out"])
    assert (off <= tol).all(), f"outputs: {np.nanmax(off / (tol + 1e-300)):.2f} of the bound"
    np.testing.assert_array_equal(keys, want["keys"], err_msg="keys")
    np.testing.assert_array_equal(values, want["values"], err_msg="values")
    if weights is None:
        return
    before = f64(x["weights"])
    group = x["heads"] // x["kv_heads"]
    batch, nodes, heads = share.shape
    # Of a batch row and key/value head: the largest share among its query rows.
    worst = share.reshape(batch, nodes, -1, group).max((1, 3))
    for b, (n, m) in enumerate(zip(x["counts"], x["lengths"])):
        got_w, want_w = f64(weights)[b], want["weights"][b]
        np.testing.assert_array_equal(got_w[:, m + n:], before[b, :, m + n:], err_msg="weights behind")
        if n == 0:
            np.testing.assert_array_equal(got_w, before[b], err_msg="weights of an empty row")
            continue
        start = before[b].copy()
        start[:, m:m + n] = 0  # new slots are assigned
        gained = want_w - start
        tol = worst[b][:, None] * gained + (n * group + 2) * 2.0 ** -24 * (gained + want_w)
        off = np.abs(got_w - want_w)[:, :m + n]
        assert (off <= tol[:, :m + n]).all(), \
            f"weights: {np.max(off / (tol[:, :m + n] + 1e-300)):.2f} of the bound"
