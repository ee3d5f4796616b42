"""Attention over the paged 4-bit cache with scores and biases of any size: biases that are masks of the type's lowest values, scores far
beyond where a softmax still weighs."""
import numpy as np
import pytest
import torch

import forms_ref
import kv_ref
from test_attention_forms_gpu import ctx, i32, make_bias  # noqa: F401  (ctx: the fixture)
from test_attention_gpu import dev, make_cache, numpy_cache, tell, wide

pytestmark = pytest.mark.gpu

MOST = float(np.finfo(np.float32).max)
SHAPES = [  # dim, page, kv heads, group, [(tokens, rows)], reach
    (64, 16, 2, 2, [(400, 70), (90, 90), (5, 2)], 60),
    (128, 64, 2, 4, [(300, 1), (65, 1), (1, 1)], 128),
    (128, 32, 1, 3, [(500, 40), (70, 90)], 3),                     # more rows than tokens
    (64, 16, 1, 2, [(100, 40), (30, 50), (0, 3)], 0),              # one bias a head: tiles that are out of reach and not seen
    (96, 32, 1, 3, [(500, 40)], 20),
    (256, 16, 1, 4, [(400, 33)], 30),
    (64, 64, 1, 2, [(20000, 3)], 128),                             # many parts, joined by a launch of their own
    (64, 64, 64, 1, [(200, 200), (129, 129)], 100),                # waves with rows of their own
    (96, 64, 64, 1, [(200, 200), (129, 129)], 30),
]


def make(shape, seed):
    dim, page, kv_heads, group, seqs, reach = shape
    rng = np.random.default_rng(seed)
    lens = [n for n, _ in seqs]
    kv, pages = make_cache(rng, lens, page, kv_heads, dim)
    q_start = np.cumsum([0] + [m for _, m in seqs])
    q = rng.standard_normal((q_start[-1], kv_heads * group, dim)).astype(np.float32)
    return rng, kv, pages, q, q_start, lens, reach


def decoded(kv, pages, lens, part):
    """what a sequence's tokens hold, float64 [tokens, kv heads, dim]"""
    codes, scales = numpy_cache(kv)[2 * part: 2 * part + 2]
    for s, n in enumerate(lens):
        t = np.arange(n)
        where, at = pages[s][t // kv.page_tokens], t % kv.page_tokens
        yield kv_ref.decode((kv_ref.unpack_values if part else kv_ref.unpack_keys)(codes[where, :, at]), scales[where, :, at])


def between(kv, pages, q_start, lens, heads, causal):
    """The least and the largest value of every dimension among the tokens that a row sees, [rows, heads, dim], zeros where it sees none, and how far
    a mean of them, its weights rounded and summed as kv_ref.allowed says, may be outside."""
    low, high = (np.zeros((q_start[-1], heads, kv.head_dim)) for _ in "lh")
    for s, v in enumerate(decoded(kv, pages, lens, 1)):
        v = np.repeat(v, heads // v.shape[1], 1)
        p = lens[s] - (q_start[s + 1] - np.arange(q_start[s], q_start[s + 1])) if causal else np.full(q_start[s + 1] - q_start[s], lens[s] - 1)
        rows, p = np.arange(q_start[s], q_start[s + 1])[p >= 0], p[p >= 0]
        if rows.size:
            low[rows], high[rows] = np.minimum.accumulate(v, 0)[p], np.maximum.accumulate(v, 0)[p]
    most = np.maximum(np.abs(low), np.abs(high))
    return low, high, most * (2.0 ** -21 + (max(lens) / 8 + 64) * 2.0 ** -24) + 2.0 ** -36 * max(lens) * most.max(-1, keepdims=True)


def tables(kv, pages):
    return (wide(pages, kv), pages)


# ---- biases ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_a_large_negative_bias_is_a_mask(ctx, shape, causal):
    """at single distances, at all beyond reach on either side, at all but a row's own: rows that see another token are what -infinity gives
    (a weight of exp(-6e7) is zero in 64 bits too), rows that see none are a mean of what they see"""
    tell("masks", shape, causal)
    rng, kv, pages, q, q_start, lens, reach = make(shape, 71)
    bias, _ = make_bias(rng, q.shape[1], reach)
    low, high, slip = between(kv, pages, q_start, lens, q.shape[1], causal)
    for cut in (slice(0, 1), slice(2 * reach, None), slice(0, 2 * reach + 1, 2), np.r_[0:reach, reach + 1:2 * reach + 1]):
        hidden = bias.copy()
        hidden[:, cut] = -np.inf
        want, sizes = forms_ref.attention(numpy_cache(kv), q, q_start, lens, pages, kv.head_dim ** -0.5, sees_all=not causal, bias=hidden)
        bound, some = forms_ref.allowed(sizes, kv.head_dim, max(lens)), sizes[2].any(-1)
        for size in (-1e6, -6e7, -1e8, -1e9, -1e10, -1e30, -2.5e38, -MOST):
            bias_now = hidden.copy()
            bias_now[:, cut] = size
            for table in tables(kv, pages):
                got = ctx.attention_biased(kv, dev(q), i32(q_start), i32(lens), dev(table), dev(bias_now), causal=causal, max_q=int(np.diff(q_start).max())).cpu().numpy()
                assert np.isfinite(got).all(), size
                assert (np.abs(got - want)[some] <= bound[some]).all(), size
                assert ((low - slip <= got) & (got <= high + slip))[~some].all(), size


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_biases_of_any_size_weigh_alike(ctx, shape, causal):
    """scores of next to nothing: the tokens with the largest bias that a row sees have the same weight, others none"""
    tell("alike", shape, causal)
    rng, kv, pages, q, q_start, lens, reach = make(shape, 72)
    for size in (6e7, 7e7, 1e8, 3.3e8, 1e9, 1e10, 1e30, 2.3e38, 2.5e38, MOST):
        for sign in (1, -1):
            bias = np.full((q.shape[1], 2 * reach + 1), sign * size, np.float32)
            bias[:, rng.random(2 * reach + 1) < 0.5] *= np.float32(0.95 if sign > 0 else 1.0 if size == MOST else 1.05)
            args = numpy_cache(kv), q, q_start, lens, pages, 1e-30
            want, sizes = forms_ref.attention(*args, sees_all=not causal, bias=bias)
            bound = kv_ref.allowed(sizes[:3], kv.head_dim, max(lens))      # (equal biases are rounded alike)
            for table in tables(kv, pages):
                got = ctx.attention_biased(kv, dev(q), i32(q_start), i32(lens), dev(table), dev(bias), causal=causal, scale=1e-30,
                                           max_q=int(np.diff(q_start).max())).cpu().numpy()
                assert (np.abs(got - want) <= bound).all(), (size, sign)


@pytest.mark.parametrize("dim,page,kv_heads,group,lens", [(64, 64, 2, 4, [1024, 640, 128]), (128, 32, 8, 4, [4096, 192]), (256, 16, 1, 2, [448]), (64, 64, 1, 2, [20480])])
def test_a_bias_that_all_tokens_have_changes_nothing(ctx, dim, page, kv_heads, group, lens):
    """tiles that are out of reach take their one bias off without rounding scores beside it, as long as steps of fp32 there are under what a score may pass
    the row's largest by: (largest, rounded by 2) up to 2^26 in powers of two"""
    rng, kv, pages, q, q_start, lens, reach = make((dim, page, kv_heads, group, [(n, 1) for n in lens], 64), 75)
    bias = np.full((q.shape[1], 2 * reach + 1), -np.inf, np.float32)      # the last 64 tokens, a tile, are not seen
    bias[:, 0] = 0
    want, sizes = forms_ref.attention(numpy_cache(kv), q, q_start, lens, pages, dim ** -0.5, bias=bias)
    bound = kv_ref.allowed(sizes[:3], dim, max(lens))
    for size in (0, 300, 1e5, 8e5, 1e6, 3e6, 1e7, 3e7, 4.6e7):
        for sign in (1, -1):
            bias[:, 0] = sign * size
            for table in tables(kv, pages):
                got = ctx.attention_biased(kv, dev(q), i32(q_start), i32(lens), dev(table), dev(bias), max_q=1).cpu().numpy()
                assert (np.abs(got - want) <= bound).all(), sign * size


def test_biases_that_are_not_finite_reach_who_meets_them(ctx):
    """among others of any size: +infinity and NaN make the rows that see their tokens not finite, no others"""
    rng = np.random.default_rng(73)
    kv, pages = make_cache(rng, [300], 16, 1, 64)
    q = dev(rng.standard_normal((20, 2, 64)).astype(np.float32))
    for ordinary in (1.0, -1e8, -MOST):
        bias = np.full((2, 101), ordinary, np.float32)
        base = ctx.attention_biased(kv, q, i32([0, 20]), i32([300]), dev(pages), dev(bias)).cpu().numpy()
        for bad in (np.inf, np.nan):
            for at in (0, 30, 49):
                now = bias.copy()
                now[0, at] = bad
                got = ctx.attention_biased(kv, q, i32([0, 20]), i32([300]), dev(pages), dev(now)).cpu().numpy()
                assert not np.isfinite(got[:, 0]).any()
                np.testing.assert_array_equal(got[:, 1], base[:, 1])


# ---- scores ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["causal", "window", "cross", "biased", "shared"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scores_of_every_size(ctx, shape, kind):
    """as large as fp32 holds them: a row whose largest score leads by more than scores are off by is its token's value, any row a mean of what it sees"""
    tell("scores", shape, kind)
    _, kv, pages, q, q_start, lens, reach = make(shape, 74)
    heads, dim = q.shape[1:]
    most_q = int(np.diff(q_start).max())
    if kind == "shared":
        q_start = np.arange(len(lens) + 1)
        q, most_q = q[:len(lens)], 1
    window = 100 if kind == "window" else 0
    low, high, slip = between(kv, pages, q_start, lens, heads, kind != "cross")
    want, lead, steep = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    scales = numpy_cache(kv)[1]
    for s, (k, v) in enumerate(zip(decoded(kv, pages, lens, 0), decoded(kv, pages, lens, 1))):
        if not lens[s]:
            continue
        t = np.arange(lens[s])
        most = 8 * np.repeat(np.abs(scales[pages[s][t // kv.page_tokens], :, t % kv.page_tokens].astype(np.float64)), 32, -1)
        r = np.arange(q_start[s], q_start[s + 1])
        p = lens[s] - (q_start[s + 1] - r)
        for h in range(heads):
            a = q[r, h].astype(np.float64) @ k[:, h // (heads // kv.n_head)].T
            if kind != "cross":
                a = np.where((t[None] <= p[:, None]) & ((t[None] > p[:, None] - window) if window else True), a, -np.inf)
            order = np.sort(a, -1)
            with np.errstate(invalid="ignore"):
                lead[r, h] = np.nan_to_num(order[:, -1] - order[:, -2] if lens[s] > 1 else np.inf, nan=0.0)
            want[r, h] = v[a.argmax(-1), h // (heads // kv.n_head)]
            steep[r, h] = (np.abs(q[r, h]).astype(np.float64) @ most[:, h // (heads // kv.n_head)].T).max(-1)
    # kv_ref.allowed's: a score is off by this times the scale
    off = steep * (2.0 ** -21 + (dim + 16) * 2.0 ** -24)
    for power in (16, 19, 20, 21, 22, 23, 24, 25, 26, 27, 30, 60, 118):
        scale = 2.0 ** power / dim ** 0.5
        clear = lead > 2 * off + 60 / scale
        assert clear.mean() > 0.5
        for table in tables(kv, pages):
            args = kv, dev(q), i32(q_start), i32(lens), dev(table)
            if kind in ("causal", "window"):
                got = ctx.attention(*args, max_q=most_q, scale=scale, window=window)
            elif kind == "cross":
                got = ctx.cross_attention(*args, max_q=most_q, scale=scale)
            elif kind == "shared":
                got = ctx.attention_shared(*args, i32([0, len(lens)]), i32([0]), max_q=1, scale=scale)
            else:
                got = ctx.attention_biased(*args, torch.zeros((heads, 2 * reach + 1), device="cuda"), max_q=most_q, scale=scale)
            got = got.cpu().numpy()
            assert np.isfinite(got).all(), power
            assert ((low - slip <= got) & (got <= high + slip)).all(), power
            # (others' weights are under exp(-60), their sum's share of a value far under its own error)
            assert (np.abs(got - want) <= slip + 1e-20)[clear].all(), power
