"""Attention over the paged 4-bit cache in its other forms on the GPU, against plain statements in 64 bits (forms_ref.py)."""
import numpy as np
import pytest
import torch

import forms_ref
from test_attention_gpu import dev, make_cache, numpy_cache, tell, wide

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from magnitude_amd import Context
    assert torch.cuda.is_available(), "these tests need the MI355X"
    c = Context(0)
    yield c
    c.close()


def i32(a):
    return dev(np.asarray(a, np.int32))


def compare(got, want, plain, sizes, dim, tokens):
    """`got` against the statement in 64 bits: every value within what is derived for it, all of them within half as much again as the statement
    in fp32, or 16 steps of an fp32 number"""
    mine = ~np.isnan(want).all(-1)
    assert (got[~mine] == 7.5).all()                       # rows of no sequence stay as they were
    got, want, plain, bound = got[mine], want[mine], plain[mine], forms_ref.allowed(sizes, dim, tokens)[mine]
    if not want.size:
        return
    err, norm = np.abs(got - want), max(1e-30, np.linalg.norm(want))
    worst, rel, usual = np.max(err / bound), np.linalg.norm(err) / norm, np.linalg.norm(plain - want) / norm
    tell(f"   worst {worst:.3g} of what is allowed, {rel:.3g} of the norm, in fp32 {usual:.3g}")
    assert worst <= 1.0 and rel <= max(1.5 * usual, 2.0 ** -20)


# ---- rows that see everything ---------------------------------------------------------------------------------------------
def check_cross(ctx, kv, pages, q, q_start, kv_len, scale=None, **kw):
    """of the call in both its forms: 16 and 32 rows at a time"""
    s = kv.head_dim ** -0.5 if scale is None else scale
    want, sizes = forms_ref.attention(numpy_cache(kv), q, q_start, kv_len, pages, s, sees_all=True)
    plain = forms_ref.attention(numpy_cache(kv), q, q_start, kv_len, pages, s, sees_all=True, dtype=np.float32)[0]
    for table in (wide(pages, kv), pages):
        out = torch.full(q.shape, 7.5, device="cuda")
        got = ctx.cross_attention(kv, dev(q), i32(q_start), i32(kv_len), dev(table), scale=scale, out=out, **kw).cpu().numpy()
        compare(got, want, plain, sizes, kv.head_dim, max([1] + list(kv_len)))
    return got


CROSS = [  # dim, page, kv heads, group, [(states, rows)]
    (64, 64, 1, 1, [(1, 1)]),
    (64, 64, 12, 1, [(1500, 1)]),
    (128, 16, 8, 4, [(500, 1), (64, 1), (63, 1), (65, 1)]),
    (96, 32, 2, 5, [(257, 3), (1, 7), (0, 2), (90, 0), (128, 1)]),
    (128, 64, 2, 4, [(1601, 187)]),
    (128, 64, 2, 4, [(5, 300), (200, 40)]),               # more rows than states
    (256, 128, 1, 8, [(700, 3), (100, 50)]),
    (64, 256, 1, 71, [(100, 2)]),
    (128, 64, 1, 4, [(20000, 1)]),                        # many parts, joined by a launch of their own
    (128, 64, 8, 4, [(1 + 700 * i, 1) for i in range(8)]),
    (64, 16, 8, 1, [(1 + 37 * i % 301, 1 + i % 3) for i in range(150)]),
    (96, 16, 1, 3, [(1300, 400)]),
]


APART = [  # of heads of 64, so many rows of short sequences that every wave has some of its own: page, kv heads, group, [(tokens, rows)]
    (64, 64, 1, [(200, 200), (129, 129), (60, 60), (190, 130)]),
    (16, 64, 2, [(100, 250), (1, 130), (0, 140), (65, 65), (64, 33)]),       # more rows than tokens, none at all
    (256, 32, 5, [(500, 500)]),                                               # 6 of 32 rows a token
    (32, 128, 1, [(90 + 7 * i, 130 + 3 * i) for i in range(3)]),
    (128, 1, 71, [(200, 1000)]),
    (128, 64, 1, [(900 - 10 * i, 600) for i in range(5)]),
]
APART_WIDE = [APART[i] for i in (0, 1, 3, 4)]      # of wider heads too
CROSS += [(64, page, kv_heads, group, seqs) for page, kv_heads, group, seqs in APART]
CROSS += [(dim, page, kv_heads, group, seqs) for dim in (96, 128) for page, kv_heads, group, seqs in APART_WIDE]


@pytest.mark.parametrize("dim,page,kv_heads,group,seqs", CROSS)
def test_cross_attention(ctx, dim, page, kv_heads, group, seqs):
    tell("cross", dim, page, kv_heads, group, seqs)
    rng = np.random.default_rng(dim + page + len(seqs))
    lens = [n for n, _ in seqs]
    kv, pages = make_cache(rng, lens, page, kv_heads, dim)
    q_start = np.cumsum([0] + [m for _, m in seqs])
    q = rng.standard_normal((q_start[-1], kv_heads * group, dim)).astype(np.float32)
    check_cross(ctx, kv, pages, q, q_start, lens)
    check_cross(ctx, kv, pages, q, q_start, lens, scale=1.0, max_q=max(m for _, m in seqs))


def test_cross_rows_of_no_sequence_stay_and_rows_without_states_are_zeros(ctx):
    rng = np.random.default_rng(21)
    lens, q_start = [3, 0, 40, 0], [2, 10, 14, 14, 15]
    kv, pages = make_cache(rng, lens, 16, 2, 64)
    q = rng.standard_normal((20, 8, 64)).astype(np.float32)
    got = check_cross(ctx, kv, pages, q, q_start, lens)
    assert got[2:10].any(-1).all() and not got[10:15].any()


def test_cross_blocks_that_are_not_finite_reach_every_row_of_their_sequence(ctx):
    rng = np.random.default_rng(22)
    kv, pages = make_cache(rng, [200, 90], 16, 2, 128)
    q = rng.standard_normal((40, 8, 128)).astype(np.float32)
    args = kv, dev(q), i32([0, 30, 40]), i32([200, 90]), dev(pages)
    base = ctx.cross_attention(*args).cpu().numpy()
    last = int(pages[0, 199 // 16]), 199 % 16
    kv.tensors[3][last[0], 1, last[1], 1] = float("nan")          # a block of a value of head 1
    for at in range(last[1] + 1, 16):                             # what lies behind the end is seen by nobody
        kv.tensors[1][last[0], :, at] = float("nan")
        kv.tensors[3][last[0], :, at] = float("nan")
    got = ctx.cross_attention(*args).cpu().numpy()
    assert np.isnan(got[:30, 4:, 32:64]).all()
    np.testing.assert_array_equal(got[30:], base[30:])
    np.testing.assert_array_equal(got[:30, :4], base[:30, :4])
    np.testing.assert_array_equal(got[:30, 4:, :32], base[:30, 4:, :32])


def test_cross_bad_pages_and_bounds_are_reported(ctx):
    from magnitude_amd import QprojError
    rng = np.random.default_rng(23)
    kv, pages = make_cache(rng, [100, 60], 16, 1, 64)
    q = rng.standard_normal((5, 4, 64)).astype(np.float32)
    ok = ctx.cross_attention(kv, dev(q), i32([0, 3, 5]), i32([100, 60]), dev(pages)).cpu().numpy()
    wrong = pages.copy()
    wrong[0, 2] = kv.n_pages
    out = torch.full(q.shape, 7.5, device="cuda")
    with pytest.raises(QprojError, match="page"):
        ctx.cross_attention(kv, dev(q), i32([0, 3, 5]), i32([100, 60]), dev(wrong), out=out)
    want, sizes = forms_ref.attention(numpy_cache(kv), q, [0, 3, 5], [100, 60], wrong, 64 ** -0.5, sees_all=True)
    assert (np.abs(out.cpu().numpy() - want) <= forms_ref.allowed(sizes, 64, 100)).all()
    for q_start, lens, max_q, left in (([0, 3, 6], [100, 60], 5, [0, 1, 2]), ([0, 3, 5], [-1, 60], 5, [3, 4]), ([0, 3, 5], [100, 1 << 20], 5, [0, 1, 2]), ([0, 3, 5], [100, 60], 2, [3, 4])):
        out = torch.full(q.shape, 7.5, device="cuda")
        with pytest.raises(QprojError, match="q_start or kv_len"):
            ctx.cross_attention(kv, dev(q), i32(q_start), i32(lens), dev(pages), max_q=max_q, out=out)
        got = out.cpu().numpy()
        np.testing.assert_allclose(got[left], ok[left], rtol=1e-5, atol=1e-6)
        assert (got[[i for i in range(5) if i not in left]] == 7.5).all()
    ctx.sync()


# ---- a bias of the distance -------------------------------------------------------------------------------------------------
def make_bias(rng, heads, reach, n_buckets=None, both=True, size=3.0):
    """(by distance, and where there are buckets the table)"""
    from magnitude_amd import relative_buckets
    if n_buckets is None:
        return (rng.standard_normal((heads, 2 * reach + 1)) * size).astype(np.float32), None
    table = (rng.standard_normal((n_buckets, heads)) * size).astype(np.float32)
    return np.ascontiguousarray(table[relative_buckets(n_buckets, reach, both)].T), table


def check_biased(ctx, kv, pages, q, q_start, kv_len, bias, causal, scale=None, **kw):
    s = kv.head_dim ** -0.5 if scale is None else scale
    args = numpy_cache(kv), q, q_start, kv_len, pages, s
    want, sizes = forms_ref.attention(*args, sees_all=not causal, bias=bias)
    plain = forms_ref.attention(*args, sees_all=not causal, bias=bias, dtype=np.float32)[0]
    for table in (wide(pages, kv), pages):
        out = torch.full(q.shape, 7.5, device="cuda")
        got = ctx.attention_biased(kv, dev(q), i32(q_start), i32(kv_len), dev(table), dev(bias), causal=causal, scale=scale, out=out, **kw).cpu().numpy()
        compare(got, want, plain, sizes, kv.head_dim, max([1] + list(kv_len)))
    return got


BIASED = [  # dim, page, kv heads, group, [(tokens, rows)], reach
    (64, 64, 1, 1, [(1, 1)], 128),
    (64, 64, 12, 1, [(300, 1), (64, 1), (65, 1), (1, 1)], 128),
    (64, 16, 2, 1, [(200, 200), (33, 33), (1, 1)], 20),
    (64, 64, 2, 1, [(700, 700)], 128),
    (128, 32, 1, 8, [(500, 90), (40, 40)], 128),
    (128, 64, 2, 3, [(1000, 1), (90, 7), (0, 0), (0, 3), (5, 9)], 64),
    (96, 128, 1, 16, [(600, 20)], 40),
    (256, 16, 1, 4, [(400, 70)], 30),
    (64, 256, 1, 71, [(100, 2)], 128),                    # as many heads an item as there is room for
    (64, 32, 1, 5, [(3000, 40)], 500),
    (128, 64, 1, 2, [(2500, 33)], 1703),
    (64, 64, 1, 1, [(9000, 1)], 0),
    (64, 64, 1, 2, [(20000, 3)], 128),                    # many parts, joined by a launch of their own
    (128, 16, 4, 4, [(1 + 37 * i % 301, 1) for i in range(90)], 10),
]


BIASED += [(64, page, kv_heads, group, seqs, reach) for (page, kv_heads, group, seqs), reach in zip(APART, (128, 30, 400, 128, 1, 200))]
BIASED += [(96, page, kv_heads, group, seqs, reach) for (page, kv_heads, group, seqs), reach in zip(APART_WIDE, (128, 30, 128, 500))]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,page,kv_heads,group,seqs,reach", BIASED)
def test_biased_attention(ctx, dim, page, kv_heads, group, seqs, reach, causal):
    tell("biased", dim, page, kv_heads, group, seqs, reach, causal)
    rng = np.random.default_rng(dim + page + len(seqs) + causal)
    lens = [n for n, _ in seqs]
    kv, pages = make_cache(rng, lens, page, kv_heads, dim)
    q_start = np.cumsum([0] + [m for _, m in seqs])
    q = rng.standard_normal((q_start[-1], kv_heads * group, dim)).astype(np.float32)
    bias, _ = make_bias(rng, kv_heads * group, reach)
    check_biased(ctx, kv, pages, q, q_start, lens, bias, causal)
    check_biased(ctx, kv, pages, q, q_start, lens, bias, causal, scale=0.25, max_q=max(m for _, m in seqs))


@pytest.mark.parametrize("both", [True, False])
@pytest.mark.parametrize("n_buckets,reach,heads", [(32, 128, 12), (8, 20, 1), (64, 500, 3)])
def test_bias_by_distance(ctx, n_buckets, reach, heads, both):
    from magnitude_amd import QprojError, relative_buckets
    rng = np.random.default_rng(n_buckets)
    bias, table = make_bias(rng, heads, reach, n_buckets, both)
    buckets = relative_buckets(n_buckets, reach, both)
    assert np.array_equal(ctx.bias_by_distance(dev(table), dev(buckets)).cpu().numpy(), bias)
    for bad in (-1, n_buckets, 2147483647):
        wrong = buckets.copy()
        wrong[3] = bad
        out = torch.full(bias.shape, 7.5, device="cuda")
        with pytest.raises(QprojError, match="bucket"):
            ctx.bias_by_distance(dev(table), dev(wrong), out=out)
        got = out.cpu().numpy()
        assert not got[:, 3].any() and np.array_equal(np.delete(got, 3, 1), np.delete(bias, 3, 1))
    ctx.sync()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("reach", [3, 60, 128])
def test_a_bias_of_minus_infinity_hides_tokens(ctx, reach, causal):
    """at single distances, at all beyond reach on either side, at all but a row's own, at all: as masks; rows that see nothing are zeros"""
    rng = np.random.default_rng(reach)
    lens, q_start = [400, 90, 5], [0, 70, 160, 162]
    kv, pages = make_cache(rng, lens, 16, 2, 64)
    q = rng.standard_normal((162, 4, 64)).astype(np.float32)
    whole, _ = make_bias(rng, 4, reach)
    for cut in (slice(0, 1), slice(2 * reach, None), slice(0, 2 * reach + 1, 2), np.r_[0:reach, reach + 1:2 * reach + 1]):
        bias = whole.copy()
        bias[:, cut] = -np.inf
        check_biased(ctx, kv, pages, q, q_start, lens, bias, causal)
    bias = whole.copy()
    bias[2] = -np.inf
    got = check_biased(ctx, kv, pages, q, q_start, lens, bias, causal)
    assert not got[:, 2].any() and got[:, 1].any(-1).all()


def test_biased_what_is_not_seen_is_not_looked_at(ctx):
    """blocks that are not finite, hidden by the bias or by the rows' own positions"""
    rng = np.random.default_rng(31)
    kv, pages = make_cache(rng, [300], 16, 1, 64)
    q = dev(rng.standard_normal((20, 2, 64)).astype(np.float32))
    bias, _ = make_bias(rng, 2, 50)
    bias[:, :30] = -np.inf                      # more than 20 tokens back: not seen, from 29 on by distances of their own
    args = kv, q, i32([0, 20]), i32([300]), dev(pages), dev(bias)
    base = ctx.attention_biased(*args).cpu().numpy()
    for t in list(range(0, 259)):               # 280 - 21 and before: out of every row's sight
        for plane in (1, 3):
            kv.tensors[plane][int(pages[0, t // 16]), :, t % 16] = float("nan")
    np.testing.assert_array_equal(ctx.attention_biased(*args).cpu().numpy(), base)
    bias[0, 50 - 1] = np.nan                    # met by the rows that have a token before them
    got = ctx.attention_biased(kv, q, i32([0, 20]), i32([300]), dev(pages), dev(bias)).cpu().numpy()
    assert np.isnan(got[:, 0]).all()
    np.testing.assert_array_equal(got[:, 1], base[:, 1])


def test_a_bias_of_nothing_changes_nothing(ctx):
    rng = np.random.default_rng(32)
    kv, pages = make_cache(rng, [700, 20], 64, 2, 128)
    q = dev(rng.standard_normal((41, 8, 128)).astype(np.float32))
    args = kv, q, i32([0, 40, 41]), i32([700, 20]), dev(pages)
    none = torch.zeros((8, 257), device="cuda")
    assert (ctx.attention_biased(*args, none) - ctx.attention(*args)).abs().max() < 1e-5
    assert (ctx.attention_biased(*args, none, causal=False) - ctx.cross_attention(*args)).abs().max() < 1e-5
    same = torch.full((8, 257), 7.25, device="cuda")       # softmax does not see what all tokens have
    assert (ctx.attention_biased(*args, same) - ctx.attention(*args)).abs().max() < 1e-5


# ---- sequences that share their first tokens ----------------------------------------------------------------------------------
def share(pages, lens, groups, page):
    """The table with whole pages of `shared` tokens the same in every group [(shared, sequences)], (table, group_start, shared_len)"""
    pages, at = pages.copy(), 0
    for shared, n in groups:
        for s in range(at + 1, at + n):
            whole = min(shared, lens[at]) // page
            pages[s, :whole] = pages[at, :whole]
        at += n
    return pages, np.cumsum([0] + [n for _, n in groups]).astype(np.int32), np.array([min(m, lens[s]) // page * page for (m, _), s in
                                                                                       zip(groups, np.cumsum([0] + [n for _, n in groups]))], np.int32)


def check_shared(ctx, kv, pages, q, q_start, kv_len, group_start, shared, scale=None, **kw):
    s = kv.head_dim ** -0.5 if scale is None else scale
    want, sizes = forms_ref.attention(numpy_cache(kv), q, q_start, kv_len, pages, s)
    plain = forms_ref.attention(numpy_cache(kv), q, q_start, kv_len, pages, s, dtype=np.float32)[0]
    for table in (wide(pages, kv), pages):
        out = torch.full(q.shape, 7.5, device="cuda")
        got = ctx.attention_shared(kv, dev(q), i32(q_start), i32(kv_len), dev(table), i32(group_start), i32(shared), scale=scale, out=out, **kw).cpu().numpy()
        compare(got, want, plain, sizes, kv.head_dim, max([1] + list(kv_len)))
    return got


SHARED = [  # dim, page, kv heads, group, [(shared, [(tokens, rows)])], the most rows
    (128, 64, 1, 4, [(64, [(65, 1), (100, 1)])], 1),
    (128, 64, 8, 4, [(1024, [(1024 + 37 * i % 300 + 1, 1) for i in range(20)])], 1),
    (64, 16, 2, 7, [(80, [(90, 2), (83, 3), (400, 1)]), (16, [(33, 2), (17, 1)]), (0, [(50, 1), (3, 2)])], 3),
    (96, 32, 2, 1, [(320, [(320 + i, 1) for i in range(1, 41)])], 1),             # 32 sequences an item
    (256, 128, 1, 2, [(384, [(400, 2), (700, 2), (385, 1)]), (128, [(129, 1), (130, 2)])], 2),
    (128, 16, 1, 16, [(160, [(200, 1), (170, 1), (300, 1)])], 1),                 # two sequences fill an item
    (128, 64, 2, 4, [(8192, [(8200 + 11 * i, 1) for i in range(9)])], 1),         # many parts
    (64, 64, 1, 4, [(20032, [(20040, 1), (20400, 4), (21000, 2)])], 4),           # many parts, joined by a launch of their own
    (128, 64, 4, 2, [(128 * (i % 4), [(130 + 128 * (i % 4) + 7 * j, 1 + (i + j) % 2) for j in range(1 + i % 6)]) for i in range(40)], 2),
    (128, 256, 2, 4, [(512, [(600, 1), (520, 0), (513, 1), (0, 0)]), (256, []), (256, [(300, 0)]), (256, [(299, 1), (700, 4)])], 4),
    (64, 32, 8, 1, [(96, [(97 + 5 * i, 1) for i in range(150)])], 1),             # far more items than can stay whole
    (128, 32, 2, 4, [(640, [(650, 8), (700, 5)])], 8),                            # nothing to gain: the causal kernel
]


@pytest.mark.parametrize("dim,page,kv_heads,group,groups,most", SHARED)
def test_shared_attention(ctx, dim, page, kv_heads, group, groups, most):
    tell("shared", dim, page, kv_heads, group, [(m, len(g)) for m, g in groups], most)
    rng = np.random.default_rng(dim + page + len(groups))
    seqs = [s for _, g in groups for s in g]
    lens, q_start = [n for n, _ in seqs], np.cumsum([0] + [m for _, m in seqs])
    kv, pages = make_cache(rng, lens, page, kv_heads, dim)
    table, group_start, shared = share(np.pad(pages, ((0, 1), (0, 0))), lens + [0], [(m, len(g)) for m, g in groups], page)
    table = table[:len(lens)]
    q = rng.standard_normal((q_start[-1], kv_heads * group, dim)).astype(np.float32)
    sizes = dict(max_q=most, max_group=max(len(g) for _, g in groups))
    check_shared(ctx, kv, table, q, q_start, lens, group_start, shared, **sizes)
    check_shared(ctx, kv, table, q, q_start, lens, group_start, shared, scale=0.3, max_q=most)      # any number a group
    for other in (0, 1, 63, 64, 65):      # less shared than could be
        if group_start[-1] < 20:
            check_shared(ctx, kv, table, q, q_start, lens, group_start, np.minimum(shared, other), **sizes)


def test_shared_tokens_that_reach_into_the_newest_are_each_row_s_own(ctx):
    """shared_len up to and past the sequences' ends: what lies at and behind the rows is not taken as seen"""
    rng = np.random.default_rng(41)
    lens, q_start = [200, 130, 129, 64, 5], [0, 2, 3, 5, 6, 8]
    kv, pages = make_cache(rng, lens, 16, 2, 64)
    pages[:, :] = pages[0]                       # the same pages from the first to the last
    q = rng.standard_normal((8, 8, 64)).astype(np.float32)
    for shared in (64, 128, 129, 200, 100000, 2147483647):
        check_shared(ctx, kv, pages, q, q_start, lens, [0, 5], [shared], max_q=2)
        check_shared(ctx, kv, pages, q, q_start, lens, [0, 3, 5], [shared, shared], max_q=2)


def test_shared_rows_of_no_sequence_stay_and_rows_that_see_nothing_are_zeros(ctx):
    rng = np.random.default_rng(42)
    lens, q_start = [3, 0, 300, 290, 0], [2, 6, 8, 10, 11, 12]        # four rows of three tokens
    kv, pages = make_cache(rng, lens, 16, 1, 128)
    q = rng.standard_normal((20, 4, 128)).astype(np.float32)
    pages[3, :16] = pages[2, :16]
    got = check_shared(ctx, kv, pages, q, q_start, lens, [0, 2, 4, 5], [0, 256, 0], max_q=4)
    assert not got[2].any() and got[3:6].any(-1).all() and not got[6:8].any() and got[8:11].any(-1).all() and not got[11].any()


def test_shared_blocks_that_are_not_finite(ctx):
    """shared ones reach all rows of the group, a sequence's own its rows, others nobody"""
    rng = np.random.default_rng(43)
    lens, q_start = [300, 280, 270, 100], [0, 1, 3, 4, 5]
    kv, pages = make_cache(rng, lens, 16, 2, 128)
    pages[1, :16], pages[2, :16] = pages[0, :16], pages[0, :16]
    q = dev(rng.standard_normal((5, 8, 128)).astype(np.float32))
    args = kv, q, i32(q_start), i32(lens), dev(pages), i32([0, 3, 4]), i32([256, 0])
    base = ctx.attention_shared(*args, max_q=2).cpu().numpy()
    clean = [t.clone() for t in kv.tensors]
    for s, t, rows in ((0, 255, [0, 1, 2, 3]), (0, 299, [0]), (1, 279, [2]), (1, 270, [1, 2]), (2, 256, [3]), (3, 99, [4])):
        for u, c in zip(kv.tensors, clean):
            u.copy_(c)
        p = int(pages[s, t // 16])
        kv.tensors[1][p, 0, t % 16, 0] = float("nan")         # a key of head 0
        kv.tensors[3][p, 1, t % 16, 1] = float("inf")         # a block of a value of head 1
        for i in range(t % 16 + 1, 16):                       # and what lies behind the last token
            if t + i - t % 16 >= lens[s]:
                kv.tensors[1][p, :, i] = float("nan")
        got = ctx.attention_shared(*args, max_q=2).cpu().numpy()
        assert np.isnan(got[rows, :4]).all() and not np.isfinite(got[rows, 4:, 32:64]).any()
        others = [r for r in range(5) if r not in rows]
        np.testing.assert_array_equal(got[others], base[others])
        np.testing.assert_array_equal(got[rows, 4:, :32], base[rows, 4:, :32])


def test_shared_bad_pages_bounds_and_groups_are_reported(ctx):
    from magnitude_amd import QprojError
    rng = np.random.default_rng(44)
    lens, q_start = [200, 180, 190, 90, 60], [0, 1, 2, 3, 4, 5]
    kv, pages = make_cache(rng, lens, 16, 1, 64)
    pages[1, :10], pages[2, :10] = pages[0, :10], pages[0, :10]
    q = rng.standard_normal((5, 4, 64)).astype(np.float32)
    call = lambda p=pages, s=q_start, n=lens, g=(0, 3, 5), m=(160, 0), out=None, **kw: ctx.attention_shared(
        kv, dev(q), i32(s), i32(n), dev(p), i32(g), i32(m), out=out, **{"max_q": 1, "max_group": 3, **kw}).cpu().numpy()
    ok = call()
    for bad in (-1, kv.n_pages, 2147483647, -2147483648):
        wrong = pages.copy()
        wrong[:3, 2] = bad                    # of what is shared (a sequence's tokens of a bad page are not seen)
        wrong[4, 1] = bad
        out = torch.full(q.shape, 7.5, device="cuda")
        with pytest.raises(QprojError, match="page"):
            call(wrong, out=out)
        want, sizes = forms_ref.attention(numpy_cache(kv), q, q_start, lens, wrong, 64 ** -0.5)
        assert (np.abs(out.cpu().numpy() - want) <= forms_ref.allowed(sizes, 64, 200)).all()
    for kw, what, left in ((dict(s=[0, 1, 2, 3, 4, 6]), "q_start", [0, 1, 2, 3]), (dict(s=[0, 1, 0, 3, 4, 5]), "q_start", [0, 3, 4]), (dict(n=[200, -1, 190, 90, 60]), "q_start", [0, 2, 3, 4]),
                           (dict(n=[1 << 20, 180, 190, 90, 60]), "q_start", [1, 2, 3, 4]), (dict(s=[-1, 1, 2, 3, 4, 5]), "q_start", [1, 2, 3, 4]),
                           (dict(g=(0, 3, 6)), "group_start", [0, 1, 2]), (dict(g=(1, 3, 5)), "group_start", [1, 2, 3, 4]), (dict(g=(0, 3, 4)), "group_start", [0, 1, 2, 3]),
                           (dict(g=(0, 3, 2)), "group_start", [0, 1, 2]), (dict(g=(-1, 3, 5)), "group_start", [3, 4]), (dict(m=(-1, 0)), "group_start", [3, 4]),
                           (dict(g=(0, 2, 5), m=(160, 0), max_group=2), "group_start", [0, 1])):
        out = torch.full(q.shape, 7.5, device="cuda")
        with pytest.raises(QprojError, match=what):
            call(out=out, **kw)
        got = out.cpu().numpy()
        np.testing.assert_allclose(got[left], ok[left], rtol=1e-5, atol=1e-6)
        assert (got[[i for i in range(5) if i not in left]] == 7.5).all()
    ctx.sync()
    np.testing.assert_array_equal(call(), ok)


def test_shared_rows_that_lie_apart_and_the_same_bits(ctx):
    rng = np.random.default_rng(45)
    lens = [3000, 2900, 2600, 70, 3100, 2700]
    kv, pages = make_cache(rng, lens, 64, 2, 128)
    pages[[1, 2, 4, 5], :40] = pages[0, :40]
    order = [0, 1, 2, 4, 5, 3]
    pages, lens = pages[order], [lens[i] for i in order]
    wide_rows = rng.standard_normal((9, 12 * 128)).astype(np.float32)
    q = dev(wide_rows)[:, 256: 256 + 1024].unflatten(1, (8, 128))
    out = torch.full((9, 1100), 7.5, device="cuda")
    y = out[:, 8: 8 + 1024].unflatten(1, (8, 128))
    args = i32([0, 1, 3, 4, 6, 8, 9]), i32(lens), dev(pages), i32([0, 5, 6]), i32([2560, 0])
    ctx.attention_shared(kv, q, *args, max_q=2, max_group=5, out=y)
    first = ctx.attention_shared(kv, q.contiguous(), *args, max_q=2, max_group=5)
    assert torch.equal(y, first) and (out[:, :8] == 7.5).all() and (out[:, 8 + 1024:] == 7.5).all()
    for _ in range(5):
        assert torch.equal(first, ctx.attention_shared(kv, q, *args, max_q=2, max_group=5))
    want = ctx.attention(kv, q, *args[:3], max_q=2)
    assert (first - want).abs().max() < 1e-5
