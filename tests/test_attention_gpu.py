"""Rotary positions, the paged 4-bit cache and attention over it on the GPU, against plain statements in 64 bits (kv_ref.py)."""
import numpy as np
import pytest
import torch

import kv_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from magnitude_amd import Context
    assert torch.cuda.is_available(), "these tests need the MI355X"
    c = Context(0)
    yield c
    c.close()


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def tell(*a):
    print(*a, flush=True)


# ---- rotation -----------------------------------------------------------------------------------------------------------
ROPE = [  # tokens, heads, dim, n_dims, mode, first position, gap between rows, in place
    (1, 32, 128, 128, "pairs", 0, 0, False),
    (1, 1, 8, 8, "halves", 5, 0, False),
    (7, 5, 128, 64, "halves", 1000003, 64, False),
    (33, 3, 80, 32, "pairs", 77, 4, True),
    (33, 3, 80, 40, "halves", 77, 4, True),
    (5, 2, 96, 24, "halves", 123456, 0, True),
    (4, 71, 64, 64, "pairs", 2147483640, 0, False),
    (300, 2, 256, 256, "halves", 0, 0, False),
    (3, 2, 1024, 1024, "pairs", 9, 0, True),
]


@pytest.mark.parametrize("tokens,heads,dim,n_dims,mode,first,gap,in_place", ROPE)
def test_rope(ctx, tokens, heads, dim, n_dims, mode, first, gap, in_place):
    from magnitude_amd import rope_frequencies
    tell("rope", tokens, heads, dim, n_dims, mode, first, gap, in_place)
    rng = np.random.default_rng(tokens * dim + heads)
    freqs, _ = rope_frequencies(n_dims)
    wide = rng.standard_normal((tokens, heads * dim + gap)).astype(np.float32)
    pos = (first + np.arange(tokens)).astype(np.int32)
    whole = dev(wide)
    x = whole[:, : heads * dim].unflatten(1, (heads, dim))
    want = kv_ref.rotate(wide[:, : heads * dim].reshape(tokens, heads, dim), pos, freqs, mode, 1.25)
    y = ctx.rope(x, dev(pos), dev(freqs), mode=mode, magnitude=1.25, out=x if in_place else None)
    got = y.cpu().numpy()
    # rounded once (half a step of fp32), at an angle that is off by a few 2^-53 of itself
    size = np.abs(wide[:, : heads * dim].reshape(tokens, heads, dim)).max(-1, keepdims=True) * 1.25
    angle = (np.abs(pos)[:, None, None] + 1.0) * 2.0 ** -50
    assert (np.abs(got - want) <= np.abs(want) * 2.0 ** -24 * 1.0001 + 2 * size * angle + 1e-30).all()
    assert np.array_equal(got[..., n_dims:], wide[:, : heads * dim].reshape(tokens, heads, dim)[..., n_dims:])
    assert np.array_equal(whole.cpu().numpy()[:, heads * dim:], wide[:, heads * dim:])     # what lies between the rows stays


# ---- append and read ----------------------------------------------------------------------------------------------------
def numpy_cache(kv):
    return tuple(t.cpu().numpy() for t in kv.tensors)


def filled(kv, rng):
    """random codes and scales everywhere, so that what a call must leave alone can be told"""
    for t in kv.tensors:
        if t.dtype == torch.uint8:
            t.copy_(dev(rng.integers(0, 256, tuple(t.shape), dtype=np.uint8)))
        else:
            t.copy_(dev((rng.standard_normal(tuple(t.shape)) * 0.25).astype(np.float16)))


def special_rows(dim):
    """rows of one head where the scale can go wrong"""
    rng = np.random.default_rng(dim)
    rows = [np.zeros(dim), np.full(dim, -0.0), np.full(dim, 3.0), np.full(dim, -3.0), np.where(np.arange(dim) % 2, 5.0, -5.0),
            np.where(np.arange(dim) % 2, -5.0, 5.0), np.arange(dim) - dim / 2 + 0.5, rng.standard_normal(dim) * 1e-8, rng.standard_normal(dim) * 1e-30,
            rng.standard_normal(dim) * 1e-42, rng.standard_normal(dim) * 2e5, rng.standard_normal(dim) * 1e6, rng.standard_normal(dim) * 1e38]
    for bad in (np.inf, -np.inf, np.nan):
        r = rng.standard_normal(dim)
        r[dim - 5] = bad
        rows.append(r)
    r = np.zeros(dim)
    r[31] = 1.0
    rows.append(r)
    return np.stack(rows).astype(np.float32)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_append_without_a_rotation_has_the_definitions_codes(ctx, dim):
    from magnitude_amd import KvCache
    rows = special_rows(dim)
    n = len(rows)
    tell("append special rows", dim)
    kv = KvCache.zeros(3, 16, 2, dim)
    filled(kv, np.random.default_rng(1))
    before = numpy_cache(kv)
    k = np.stack((rows, rows[::-1]), 1)
    v = np.stack((rows[::-1] * np.float32(-1), rows), 1)
    slots = np.random.default_rng(2).permutation(48)[:n].astype(np.int64)
    ctx.kv_append(kv, dev(k), dev(v), dev(slots))
    after = numpy_cache(kv)
    for x, codes, scales, pack in ((k, 0, 1, kv_ref.pack_keys), (v, 2, 3, kv_ref.pack_values)):
        want_n, want_d = kv_ref.quantize(x)
        got_n, got_d = after[codes][slots // 16, :, slots % 16], after[scales][slots // 16, :, slots % 16]
        assert np.array_equal(got_n, pack(want_n))
        assert np.array_equal(np.isnan(got_d), np.isnan(want_d)) and np.array_equal(got_d[~np.isnan(want_d)], want_d[~np.isnan(want_d)])
        others = np.setdiff1d(np.arange(48), slots)
        for plane in (codes, scales):
            assert np.array_equal(after[plane][others // 16, :, others % 16], before[plane][others // 16, :, others % 16])
    back_k, back_v = ctx.kv_read(kv, dev(slots))
    for got, x, unpack, codes, scales in ((back_k, k, kv_ref.unpack_keys, 0, 1), (back_v, v, kv_ref.unpack_values, 2, 3)):
        want = kv_ref.decode(unpack(after[codes][slots // 16, :, slots % 16]), after[scales][slots // 16, :, slots % 16])
        np.testing.assert_array_equal(got.cpu().numpy(), want.astype(np.float32))


APPEND = [  # tokens, heads, kv heads, dim, n_dims, mode, page, first position
    (1, 32, 8, 128, 128, "pairs", 16, 700),
    (1, 1, 1, 64, 64, "halves", 256, 0),
    (5, 14, 2, 64, 32, "halves", 32, 131071),
    (48, 8, 8, 128, 64, "pairs", 64, 9000),
    (200, 6, 3, 96, 24, "halves", 128, 31),
    (37, 4, 1, 256, 256, "halves", 16, 1000000),
    (9, 40, 8, 128, 120, "halves", 64, 2147483000),
]


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,n_dims,mode,page,first", APPEND)
def test_append_rotates_keys_and_queries(ctx, tokens, heads, kv_heads, dim, n_dims, mode, page, first):
    from magnitude_amd import KvCache, rope_frequencies
    tell("append", tokens, heads, kv_heads, dim, n_dims, mode, page, first)
    rng = np.random.default_rng(tokens + dim)
    freqs, mag = rope_frequencies(n_dims, freq_scale=0.25, n_ctx_orig=4096, ext_factor=1.0)
    joined = rng.standard_normal((tokens, (heads + 2 * kv_heads) * dim)).astype(np.float32)     # one joined q/k/v product
    cut = [heads * dim, (heads + kv_heads) * dim]
    qh, kh, vh = (a.reshape(tokens, -1, dim) for a in np.split(joined, cut, axis=1))
    jd = dev(joined)
    q, k, v = (jd[:, a:b].unflatten(1, (-1, dim)) for a, b in ((0, cut[0]), (cut[0], cut[1]), (cut[1], None)))
    pos = (first + np.arange(tokens)).astype(np.int32)
    n_pages = 2 * (-(-tokens // page)) + 1
    slots = rng.permutation(n_pages * page)[:tokens].astype(np.int64)
    slots[tokens // 2] = -1 if tokens > 1 else slots[tokens // 2]             # padding
    kv = KvCache.zeros(n_pages, page, kv_heads, dim)
    filled(kv, rng)
    before = numpy_cache(kv)
    got_q = ctx.kv_append(kv, k, v, dev(slots), pos=dev(pos), freqs=dev(freqs), mode=mode, magnitude=mag, q=q)
    alone = ctx.rope(q, dev(pos), dev(freqs), mode=mode, magnitude=mag)
    assert torch.equal(got_q, alone)
    after = numpy_cache(kv)
    live = slots >= 0
    at = slots[live]
    turned = kv_ref.rotate(kh, pos, freqs, mode, mag)
    for x, codes, scales, unpack in ((turned[live], 0, 1, kv_ref.unpack_keys), (vh[live], 2, 3, kv_ref.unpack_values)):
        n, d = kv_ref.quantize(x.astype(np.float32))
        got_n = unpack(after[codes][at // page, :, at % page])
        got_d = after[scales][at // page, :, at % page]
        # Angles agree to a few 2^-52 of the position; the fp32 value may round the other way then, off by 2^-23 of the block's
        # largest, and a code next to a border may be its neighbour: nowhere else.
        off = 2.0 ** -22 + 2.0 ** -49 * np.abs(pos[live]).max() if codes == 0 else 0.0
        with np.errstate(all="ignore"):
            exact = x.reshape(n.shape) / (np.take_along_axis(x.reshape(n.shape), np.abs(x.reshape(n.shape)).argmax(-1)[..., None], -1) / -8) + 8.5
        border = (np.abs(exact - np.round(exact)) < 16 * off + 2.0 ** -20).reshape(got_n.shape)
        assert (np.abs(got_n.astype(int) - n.reshape(got_n.shape)) <= (1 if codes == 0 else 0) * border).all()
        np.testing.assert_allclose(got_d.astype(np.float64), d.astype(np.float64), rtol=2.0 ** -10 if codes == 0 else 0, atol=0)
        assert (got_d != d).mean() <= (0.01 if codes == 0 else 0)
    others = np.setdiff1d(np.arange(n_pages * page), at)
    for a, b in zip(after, before):
        assert np.array_equal(a[others // page, :, others % page], b[others // page, :, others % page])


def test_slots_behind_the_cache_are_reported_and_left_out(ctx):
    from magnitude_amd import KvCache, QprojError
    kv = KvCache.zeros(2, 16, 1, 64)
    filled(kv, np.random.default_rng(3))
    before = numpy_cache(kv)
    x = torch.randn((3, 1, 64), device="cuda")
    slots = dev(np.array([32, -5, 1 << 40], dtype=np.int64))
    with pytest.raises(QprojError, match="slot"):
        ctx.kv_append(kv, x, x, slots)
    ctx.sync()                                  # reported once
    for a, b in zip(numpy_cache(kv), before):
        assert np.array_equal(a, b)
    with pytest.raises(QprojError, match="slot"):
        ctx.kv_read(kv, slots)
    k, v = ctx.kv_read(kv, dev(np.array([-1, 3], dtype=np.int64)))
    assert not k[0].any() and not v[0].any() and k[1].any()


# ---- attention ----------------------------------------------------------------------------------------------------------
def make_cache(rng, lens, page, kv_heads, dim, spare=3, scale=1.0):
    """a cache of random rows, pages of the sequences in any order among `spare` unused ones; (kv, pages)"""
    from magnitude_amd import KvCache
    count = [-(-n // page) for n in lens]
    total = sum(count) + spare
    kv = KvCache.zeros(total, page, kv_heads, dim)
    for part, pack in ((0, kv_ref.pack_keys), (2, kv_ref.pack_values)):
        n, d = kv_ref.quantize((rng.standard_normal((total, kv_heads, page, dim)) * scale).astype(np.float32))
        kv.tensors[part].copy_(dev(pack(n)))
        kv.tensors[part + 1].copy_(dev(d))
    order = rng.permutation(total)
    pages = np.full((len(lens), max(count + [1]) + 1), -7, dtype=np.int32)
    at = 0
    for i, c in enumerate(count):
        pages[i, :c] = order[at:at + c]
        at += c
    return kv, pages


def wide(pages, kv):
    """the same table with room for so many pages that rows are taken 32 at a time (where there are more than 16 of a head at all)"""
    columns = -(-6 * 2 * 256 * 300 // (kv.page_tokens * kv.n_head * len(pages))) + 1
    return np.pad(pages, ((0, 0), (0, columns)), constant_values=-7)


def check(ctx, kv, pages, q, q_start, kv_len, window=0, scale=None, **kw):
    """of the call in both its forms: 16 and 32 rows at a time"""
    dim = kv.head_dim
    s = dim ** -0.5 if scale is None else scale
    want, sizes = kv_ref.attention(numpy_cache(kv), q, q_start, kv_len, pages, s, window)
    mine = ~np.isnan(want).all(-1)
    plain = kv_ref.attention(numpy_cache(kv), q, q_start, kv_len, pages, s, window, dtype=np.float32)[0]
    bound = kv_ref.allowed(sizes, dim, max([1] + list(kv_len)))[mine]
    usual = np.linalg.norm((plain - want)[mine]) / max(1e-30, np.linalg.norm(want[mine])) if mine.any() else 0.0
    for table in (wide(pages, kv), pages):
        out = torch.full(q.shape, 7.5, device="cuda")
        got = ctx.attention(kv, dev(q), dev(np.array(q_start, np.int32)), dev(np.array(kv_len, np.int32)), dev(table), scale=scale, window=window,
                            out=out, **kw).cpu().numpy()
        assert (got[~mine] == 7.5).all()                       # rows of no sequence stay as they were
        err = np.abs(got - want)[mine]
        worst = np.max(err / bound) if err.size else 0.0
        rel = np.linalg.norm(err) / max(1e-30, np.linalg.norm(want[mine])) if err.size else 0.0
        tell(f"   worst {worst:.3g} of what is allowed, {rel:.3g} of the norm, in fp32 {usual:.3g}")
        # over all values: half as much again as the statement in fp32, or 16 steps of an fp32 number
        assert worst <= 1.0 and rel <= max(1.5 * usual, 2.0 ** -20)
    return got


ATTENTION = [  # dim, page, kv heads, group, [(tokens in the cache, new ones)], window
    (128, 16, 1, 1, [(1, 1)], 0),
    (128, 16, 8, 4, [(500, 1)], 0),
    (128, 64, 2, 4, [(63, 1), (64, 1), (65, 1), (1, 1), (129, 1)], 0),
    (64, 32, 2, 7, [(300, 1), (17, 1)], 0),
    (96, 256, 3, 5, [(257, 1), (256, 1), (1000, 2)], 0),
    (256, 128, 1, 8, [(700, 3)], 0),
    (128, 64, 1, 16, [(333, 1)], 0),
    (128, 64, 1, 71, [(100, 2)], 0),                        # many heads on one key/value head
    (64, 16, 1, 128, [(40, 1)], 0),
    (128, 32, 2, 4, [(8, 8), (20, 5), (1500, 8), (3, 1)], 0),
    (128, 64, 2, 4, [(200, 200)], 0),
    (128, 64, 1, 3, [(130, 67), (70, 70), (0, 0), (5, 1)], 0),
    (64, 64, 2, 1, [(515, 140)], 0),
    (96, 16, 1, 6, [(90, 33)], 0),
    (256, 64, 1, 2, [(300, 90)], 0),
    (128, 64, 2, 4, [(2500, 1), (40, 1)], 128),
    (64, 128, 2, 7, [(1500, 187)], 300),
    (128, 16, 1, 4, [(400, 100), (90, 90)], 1),
    (128, 16, 1, 4, [(400, 30)], 64),
    (128, 64, 8, 4, [(700, 700)], 100),
    (64, 128, 4, 7, [(1200, 500)], 200),
    (128, 64, 8, 1, [(9000, 1), (100, 1), (4097, 1)], 0),
    # far more items than workgroups, all short: dealt out whole, several rounds
    (64, 16, 8, 1, [(1 + 37 * i % 301, 1) for i in range(300)], 0),
    (96, 32, 4, 4, [(64 + 11 * i % 190, 64) for i in range(20)], 0),
    (256, 16, 4, 2, [(1 + 13 * i % 97, 1) for i in range(150)], 0),
    # more items than can stay whole, one of them long: cut, also inside what an item's start counts for
    (64, 64, 4, 4, [(3000, 1)] + [(1 + 29 * i % 257, 1) for i in range(200)], 0),
    (128, 64, 4, 4, [(2000, 130)] + [(1 + 29 * i % 257, 1) for i in range(60)], 0),
    # a few parts an item, added by the last of its workgroups, and many, which a launch of its own adds
    (128, 64, 8, 4, [(1 + 700 * i, 1) for i in range(8)], 0),
    (96, 128, 2, 3, [(6000, 1), (5, 1), (2000, 1)], 0),
    (256, 64, 2, 4, [(5000, 20)], 0),
    (256, 64, 1, 4, [(20000, 1)], 0),
    (64, 256, 1, 8, [(30000, 3)], 0),
    (128, 64, 1, 4, [(0, 0), (20000, 1), (0, 0), (5, 1)], 0),
    (96, 256, 1, 1, [(20000, 1)], 5000),
    (64, 64, 2, 8, [(3000, 64)], 0),
    # a prompt among tokens, and no max_q: mostly places without an item
    (64, 64, 2, 4, [(50 + i, 1) for i in range(30)] + [(400, 300)] + [(0, 0)] * 5 + [(90 + i, 1) for i in range(10)], 0),
    # the last page full to its end
    (128, 16, 2, 4, [(256, 1), (64, 2)], 0),
]


@pytest.mark.parametrize("dim,page,kv_heads,group,seqs,window", ATTENTION)
def test_attention(ctx, dim, page, kv_heads, group, seqs, window):
    tell("attention", dim, page, kv_heads, group, seqs, window)
    rng = np.random.default_rng(dim + page + len(seqs))
    lens = [n for n, _ in seqs]
    kv, pages = make_cache(rng, lens, page, kv_heads, dim)
    q_start = np.cumsum([0] + [m for _, m in seqs])
    q = rng.standard_normal((q_start[-1], kv_heads * group, dim)).astype(np.float32)
    check(ctx, kv, pages, q, q_start, lens, window)
    check(ctx, kv, pages, q, q_start, lens, window, max_q=max(m for _, m in seqs))


def test_rows_that_see_nothing_are_zeros_and_rows_of_no_sequence_stay(ctx):
    rng = np.random.default_rng(5)
    # fewer tokens in the cache than rows, none at all, rows before the first and behind the last sequence
    lens, q_start = [3, 0, 40, 0], [2, 10, 14, 14, 15]
    kv, pages = make_cache(rng, lens, 16, 2, 64)
    q = rng.standard_normal((20, 8, 64)).astype(np.float32)
    got = check(ctx, kv, pages, q, q_start, lens)
    assert not got[2:7].any() and got[7:10].any() and not got[10:15].any()


@pytest.mark.parametrize("new", [1, 40])
def test_values_of_every_size(ctx, new):
    """scales from the smallest to the largest fp16, in tiles that follow each other and in one tile"""
    rng = np.random.default_rng(6)
    for order in range(2):
        kv, pages = make_cache(rng, [400], 16, 2, 128)
        size = np.repeat(np.array([2.0 ** e for e in (-24, -14, -3, 4, 12, -10, 0, -20, 15.9, -24, 3, -7)] * 3)[:28, None], 16, 1)
        if order:
            size = 2.0 ** rng.uniform(-22, 14, size.shape)
        d = np.zeros(kv.tensors[3].shape, np.float16)
        for i in range(25):
            d[pages[0, i]] = size[i][None, :, None]
        kv.tensors[3].copy_(dev(d))
        # attention that moves from tile to tile, so that small values have the weight
        q = (rng.standard_normal((new, 4, 128)) * 12).astype(np.float32)
        check(ctx, kv, pages, q, [0, new], [400])


def test_queries_of_every_size(ctx):
    rng = np.random.default_rng(7)
    kv, pages = make_cache(rng, [150], 32, 1, 96)
    q = rng.standard_normal((7, 3, 96)).astype(np.float32)
    for i, size in enumerate((1e-38, 1e-20, 1e-6, 1.0, 30.0)):
        q[i] *= size
    q[5] = 0
    q[6, :, 1:] *= 1e-6                       # one large value among small ones
    check(ctx, kv, pages, q, [0, 7], [150])
    kv.tensors[1].mul_(1e-4)
    check(ctx, kv, pages, (q * 3e4).astype(np.float32), [0, 7], [150])


def test_queries_next_to_nothing(ctx):
    """so small that the unit of their scores would be zero: weights are equal, tokens that are masked stay so"""
    rng = np.random.default_rng(18)
    kv, pages = make_cache(rng, [100, 70], 16, 2, 128)
    for size in (1e-36, 1e-40, 1e-43, 1e-45, 0.0):
        q = (np.sign(rng.standard_normal((40, 8, 128))) * size).astype(np.float32)
        check(ctx, kv, pages, q, [0, 1, 40], [100, 70])


@pytest.mark.parametrize("dim,new,group,rows", [(128, 1, 4, 16), (128, 70, 4, 16), (128, 70, 4, 32), (64, 9, 2, 16), (64, 9, 2, 32), (96, 20, 3, 32), (256, 3, 1, 16)])
def test_blocks_that_are_not_finite_reach_only_who_sees_them(ctx, dim, new, group, rows):
    rng = np.random.default_rng(8)
    length = 200
    kv, pages = make_cache(rng, [length, 90], 16, 2, dim)
    clean = [t.clone() for t in kv.tensors]
    q = rng.standard_normal((new + 1, 2 * group, dim)).astype(np.float32)
    q_start, lens = [0, new, new + 1], [length, 90]
    check(ctx, kv, pages, q, q_start, lens)
    table = dev(wide(pages, kv) if rows == 32 else pages)
    base = ctx.attention(kv, dev(q), dev(np.array(q_start, np.int32)), dev(np.array(lens, np.int32)), table).cpu().numpy()
    page_of = lambda s, t: (int(pages[s, t // 16]), t % 16)

    def poison(t, value, s=0):
        p, at = page_of(s, t)
        kv.tensors[1][p, 0, at, 0] = value       # a key of head 0
        kv.tensors[3][p, 1, at, 1] = value       # a block of a value of head 1

    # the last token: seen by the last row of sequence 0 only; behind sequence 1's end and in unused pages: by nobody
    for value in (float("nan"), float("inf")):
        poison(length - 1, value)
        p, at = int(pages[1, 89 // 16]), 89 % 16
        for j in range(at + 1, 16):
            for plane in (1, 3):
                kv.tensors[plane][p, :, j] = value
        used = set(pages[0, :-(-length // 16)]) | set(pages[1, :-(-90 // 16)])
        for u in range(kv.n_pages):
            if u not in used:
                for plane in (1, 3):
                    kv.tensors[plane][u] = value
        got = ctx.attention(kv, dev(q), dev(np.array(q_start, np.int32)), dev(np.array(lens, np.int32)), table).cpu().numpy()
        hit = np.zeros(got.shape, bool)
        hit[new - 1, :group] = True
        hit[new - 1, group:, 32:64] = True
        if np.isnan(value):
            assert np.isnan(got[hit]).all()
        else:                                     # infinity: not finite, or (a score of minus infinity) the rest alone
            assert not np.isfinite(got[new - 1, group:, 32:64]).any()
        np.testing.assert_array_equal(got[:new - 1], base[:new - 1])
        np.testing.assert_array_equal(got[new], base[new])
        rest = [d for d in range(dim) if not 32 <= d < 64]
        np.testing.assert_array_equal(got[new - 1, group:][:, rest], base[new - 1, group:][:, rest])
        for t, c in zip(kv.tensors, clean):
            t.copy_(c)


def test_bad_pages_and_bad_bounds_are_reported(ctx):
    from magnitude_amd import QprojError
    rng = np.random.default_rng(9)
    kv, pages = make_cache(rng, [100, 60], 16, 1, 64)
    q = rng.standard_normal((5, 4, 64)).astype(np.float32)
    for bad in (-1, kv.n_pages, 2147483647, -2147483648):
        wrong = pages.copy()
        wrong[0, 2] = bad
        out = torch.full(q.shape, 7.5, device="cuda")
        with pytest.raises(QprojError, match="page"):
            check(ctx, kv, wrong, q, [0, 3, 5], [100, 60])
        ctx.attention(kv, dev(q), dev(np.array([0, 3, 5], np.int32)), dev(np.array([100, 60], np.int32)), dev(wrong), out=out, sync=False)
        torch.cuda.synchronize()
        with pytest.raises(QprojError):
            ctx.sync()
        want, _ = kv_ref.attention(numpy_cache(kv), q, [0, 3, 5], [100, 60], wrong, 64 ** -0.5)     # its tokens are not seen
        np.testing.assert_allclose(out.cpu().numpy(), want, rtol=2e-4, atol=2e-5)
    ok = ctx.attention(kv, dev(q), dev(np.array([0, 3, 5], np.int32)), dev(np.array([100, 60], np.int32)), dev(pages)).cpu().numpy()
    for q_start, lens, max_q, left in (([0, 3, 6], [100, 60], 5, [0, 1, 2]), ([0, 3, 5], [100, -1], 5, [0, 1, 2]), ([0, 3, 5], [100, 1 << 20], 5, [0, 1, 2]),
                                       ([0, 3, 5], [100, 60], 2, [3, 4]), ([0, 3, 2], [100, 60], 5, [0, 1, 2]), ([-1, 3, 5], [100, 60], 5, [3, 4])):
        out = torch.full(q.shape, 7.5, device="cuda")
        with pytest.raises(QprojError, match="q_start or kv_len"):
            ctx.attention(kv, dev(q), dev(np.array(q_start, np.int32)), dev(np.array(lens, np.int32)), dev(pages), max_q=max_q, out=out)
        got = out.cpu().numpy()
        np.testing.assert_allclose(got[left], ok[left], rtol=1e-5, atol=1e-6)
        others = [i for i in range(5) if i not in left]
        assert (got[others] == 7.5).all()
    ctx.sync()


def test_rows_that_lie_apart(ctx):
    rng = np.random.default_rng(10)
    kv, pages = make_cache(rng, [77, 200], 16, 2, 128)
    wide = rng.standard_normal((6, 12 * 128)).astype(np.float32)
    q = dev(wide)[:, 256: 256 + 1024].unflatten(1, (8, 128))
    out = torch.full((6, 1100), 7.5, device="cuda")
    y = out[:, 8: 8 + 1024].unflatten(1, (8, 128))
    start, lens = dev(np.array([0, 1, 6], np.int32)), dev(np.array([77, 200], np.int32))
    ctx.attention(kv, q, start, lens, dev(pages), out=y)
    assert torch.equal(y, ctx.attention(kv, q.contiguous(), start, lens, dev(pages)))
    assert (out[:, :8] == 7.5).all() and (out[:, 8 + 1024:] == 7.5).all()


def test_the_same_call_gives_the_same_bits(ctx):
    rng = np.random.default_rng(11)
    kv, pages = make_cache(rng, [3000, 17, 900], 64, 2, 128)
    q = dev(rng.standard_normal((12, 8, 128)).astype(np.float32))
    start, lens, p = dev(np.array([0, 1, 2, 12], np.int32)), dev(np.array([3000, 17, 900], np.int32)), dev(pages)
    first = ctx.attention(kv, q, start, lens, p)
    for _ in range(5):
        assert torch.equal(first, ctx.attention(kv, q, start, lens, p))


def test_a_cache_beyond_32_bits(ctx):
    """planes of more than 4 GiB, pages near their end"""
    from magnitude_amd import KvCache
    page, heads, dim = 256, 8, 128
    n_pages = (1 << 32) // (heads * page * dim // 2) + 40
    tell("cache beyond 32 bits:", n_pages, "pages")
    codes = [torch.empty((n_pages, heads, page, dim // 2), dtype=torch.uint8, device="cuda") for _ in "kv"]
    scales = [torch.empty((n_pages, heads, page, dim // 32), dtype=torch.float16, device="cuda") for _ in "kv"]
    kv = KvCache(codes[0], scales[0], codes[1], scales[1])
    rng = np.random.default_rng(12)
    length = 600
    where = np.array([n_pages - 1, 0, n_pages - 3], np.int64)
    t = np.arange(length)
    slots = where[t // page] * page + t % page
    k, v = (rng.standard_normal((length, heads, dim)).astype(np.float32) for _ in "kv")
    ctx.kv_append(kv, dev(k), dev(v), dev(slots))
    small = KvCache.zeros(3, page, heads, dim)
    ctx.kv_append(small, dev(k), dev(v), dev(t.astype(np.int64)))
    q = dev(rng.standard_normal((2, 8, dim)).astype(np.float32))
    start, lens = dev(np.array([0, 2], np.int32)), dev(np.array([length], np.int32))
    a = ctx.attention(kv, q, start, lens, dev(where.astype(np.int32)[None]))
    b = ctx.attention(small, q, start, lens, dev(np.arange(3, dtype=np.int32)[None]))
    assert torch.equal(a, b) and torch.isfinite(a).all()
    ka, va = ctx.kv_read(kv, dev(slots))
    kb, vb = ctx.kv_read(small, dev(t.astype(np.int64)))
    assert torch.equal(ka, kb) and torch.equal(va, vb)


# ---- together, as they are used -------------------------------------------------------------------------------------------
def test_generation_through_the_projections(ctx):
    """q/k/v projections, rotation and append, attention, output projection, for a prompt and then token by token: the prompt's
    rows and the tokens' agree with the statements in 64 bits on what the cache holds."""
    from magnitude_amd import ACT_F32, TYPE_Q4_K, KvCache, rope_frequencies, synth
    heads, kv_heads, dim, d, page = 8, 2, 64, 512, 16
    weights = [ctx.upload_from_device(TYPE_Q4_K, d, n, synth.random_weight(TYPE_Q4_K, n, d, seed=40 + i, device="cuda"))
               for i, n in enumerate((heads * dim, kv_heads * dim, kv_heads * dim, d))]
    rng = np.random.default_rng(13)
    freqs, mag = rope_frequencies(dim, base=500000.0)
    fd = dev(freqs)
    kv = KvCache.zeros(8, page, kv_heads, dim)
    pages = np.array([[5, 2, 7, 0, 1]], np.int32)
    length = 0
    for new in (37, 1, 1, 3, 1):
        x = dev(rng.standard_normal((new, d)).astype(np.float32))
        q, k, v = ctx.mul_mat_multi(weights[:3], x, ACT_F32, sync=False)
        ctx.sync()
        t = np.arange(length, length + new)
        slots = (pages[0, t // page].astype(np.int64) * page + t % page)
        q = ctx.kv_append(kv, k.unflatten(1, (kv_heads, dim)), v.unflatten(1, (kv_heads, dim)), dev(slots), pos=dev(t.astype(np.int32)), freqs=fd,
                          mode="halves", magnitude=mag, q=q.unflatten(1, (heads, dim)))
        length += new
        got = check(ctx, kv, pages, q.cpu().numpy(), [0, new], [length], max_q=new)
        y = ctx.mul_mat(weights[3], dev(got).flatten(1), ACT_F32)
        assert torch.isfinite(y).all() and y.shape == (new, d)


def test_captured_steps(ctx):
    """append and attention recorded once and replayed with other lengths, eager work of the same context between the replays"""
    from magnitude_amd import Context, KvCache, rope_frequencies
    stream = torch.cuda.Stream()
    own = Context(0, stream=stream.cuda_stream)
    heads, kv_heads, dim, page = 8, 2, 128, 16
    rng = np.random.default_rng(14)
    freqs, _ = rope_frequencies(dim)
    kv = KvCache.zeros(40, page, kv_heads, dim)
    other = KvCache.zeros(40, page, kv_heads, dim)
    order = rng.permutation(40).reshape(2, 20).astype(np.int32)
    lens0 = np.array([150, 7])
    for s, n in enumerate(lens0):
        t = np.arange(n)
        k, v = (dev(rng.standard_normal((n, kv_heads, dim)).astype(np.float32)) for _ in "kv")
        for c in (kv, other):
            own.kv_append(c, k, v, dev(order[s, t // page].astype(np.int64) * page + t % page), pos=dev(t.astype(np.int32)), freqs=dev(freqs))
    qkv = [torch.zeros((2, h, dim), device="cuda") for h in (heads, kv_heads, kv_heads)]
    slots, pos, lens = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), dev(lens0.astype(np.int32))
    start, pages, fd = dev(np.array([0, 1, 2], np.int32)), dev(order), dev(freqs)
    q_out, y = torch.zeros_like(qkv[0]), torch.zeros_like(qkv[0])

    def step(cache, q_out, y):
        own.kv_append(cache, qkv[1], qkv[2], slots, pos=pos, freqs=fd, q=qkv[0], q_out=q_out, sync=False)
        own.attention(cache, q_out, start, lens, pages, max_q=1, out=y, sync=False)

    def load(i):
        now = lens0 + i
        with torch.cuda.stream(stream):
            for t in qkv:
                t.copy_(torch.randn(t.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1000 * i + t.shape[1])))
            pos.copy_(dev(now.astype(np.int32)))
            lens.copy_(dev((now + 1).astype(np.int32)))
            slots.copy_(dev(order[np.arange(2), now // page].astype(np.int64) * page + now % page))
        stream.synchronize()

    load(0)
    step(kv, q_out, y)
    own.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(kv, q_out, y)
    eager_q, eager_y = torch.zeros_like(q_out), torch.zeros_like(y)
    for i in range(0, 12):
        load(i)
        with torch.cuda.stream(stream):
            y.zero_()
            graph.replay()
        step(other, eager_q, eager_y)
        own.sync()
        torch.cuda.synchronize()
        assert torch.equal(y, eager_y) and torch.equal(q_out, eager_q), f"replay {i}"
        want, sizes = kv_ref.attention(numpy_cache(kv), q_out.cpu().numpy(), [0, 1, 2], lens.cpu().numpy(), order, dim ** -0.5)
        assert (np.abs(y.cpu().numpy() - want) <= kv_ref.allowed(sizes, dim, int(lens.max()))).all()
    own.close()


@pytest.mark.parametrize("seqs,group", [(1, 4), (1, 32), (24, 4)])     # joined by a launch of their own, by the last workgroup (of two halves of the heads, of many sequences)
def test_captured_attention_follows_the_lengths(seqs, group):
    """recorded once, replayed with lengths from nothing to full pages: items cut into one part, a few and many"""
    from magnitude_amd import Context
    stream = torch.cuda.Stream()
    own, other = Context(0, stream=stream.cuda_stream), Context(0)
    rng = np.random.default_rng(15)
    page, dim, most = 256, 128, 5000
    kv, pages = make_cache(rng, [most] * seqs, page, 1, dim)
    q, y = dev(rng.standard_normal((seqs, group, dim)).astype(np.float32)), torch.zeros((seqs, group, dim), device="cuda")
    start, lens, p = dev(np.arange(seqs + 1, dtype=np.int32)), torch.full((seqs,), most, dtype=torch.int32, device="cuda"), dev(pages)
    own.attention(kv, q, start, lens, p, max_q=1, out=y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.attention(kv, q, start, lens, p, max_q=1, out=y, sync=False)
    for i in range(12):
        n = rng.integers(0, most + 1, seqs) if i % 3 else np.full(seqs, (0, 1, most, 300)[i // 3])
        with torch.cuda.stream(stream):
            lens.copy_(dev(n.astype(np.int32)))
            y.fill_(7.5)
            graph.replay()
        stream.synchronize()
        assert torch.equal(y, other.attention(kv, q, start, lens, p, max_q=1)), f"replay {i}"
        if i % 2:       # the same context's own work between replays
            own.attention(kv, q, start, lens, p, max_q=1)
        if i == 4:
            want, sizes = kv_ref.attention(numpy_cache(kv), q.cpu().numpy(), np.arange(seqs + 1), n, pages, dim ** -0.5)
            assert (np.abs(y.cpu().numpy() - want) <= kv_ref.allowed(sizes, dim, most)).all()
    own.close()
    other.close()


def test_the_first_call_of_a_context_is_not_captured():
    from magnitude_amd import Context, KvCache, QprojError
    stream = torch.cuda.Stream()
    own = Context(0, stream=stream.cuda_stream)
    kv = KvCache.zeros(2, 16, 1, 64)
    q, y, spare = (torch.zeros((1, 4, 64), device="cuda") for _ in range(3))
    args = dev(np.array([0, 1], np.int32)), dev(np.array([3], np.int32)), dev(np.array([[1]], np.int32))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        spare.add_(1)
        with pytest.raises(QprojError, match="captured"):
            own.attention(kv, q, *args, out=y, sync=False)
    graph.replay()                       # what was recorded beside stays whole
    torch.cuda.synchronize()
    assert (spare == 1).all()
    own.attention(kv, q, *args, out=y)   # and the context does too
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.attention(kv, q, *args, out=y, sync=False)
    y.fill_(7.5)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert not y.any()
    own.close()


def test_two_contexts_at_once():
    """calls of two contexts on streams of their own, one cut into few parts and one into many, do not meet"""
    from magnitude_amd import Context
    rng = np.random.default_rng(16)
    work = []
    for lens, kv_heads in (([9000], 1), ([3000, 10, 700, 2000], 8)):
        stream = torch.cuda.Stream()
        kv, pages = make_cache(rng, lens, 64, kv_heads, 128)
        q = dev(rng.standard_normal((len(lens), 4 * kv_heads, 128)).astype(np.float32))
        args = kv, q, dev(np.arange(len(lens) + 1, dtype=np.int32)), dev(np.array(lens, np.int32)), dev(pages)
        c = Context(0, stream=stream.cuda_stream)
        work.append((c, args, c.attention(*args, max_q=1), [torch.zeros_like(q) for _ in range(20)]))
    torch.cuda.synchronize()
    for i in range(20):
        for c, args, _, outs in work:
            c.attention(*args, max_q=1, out=outs[i], sync=False)
    for c, _, want, outs in work:
        c.sync()
        assert all(torch.equal(o, want) for o in outs)
        c.close()


def test_nothing_to_do(ctx):
    kv, pages = make_cache(np.random.default_rng(17), [30], 16, 2, 64)
    none = torch.zeros((0, 2, 64), device="cuda")
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    assert ctx.attention(kv, none, i32(0, 0), i32(30), dev(pages)).shape == (0, 2, 64)
    y = torch.full((3, 2, 64), 7.5, device="cuda")
    q = torch.zeros_like(y)
    ctx.attention(kv, q, i32(0), i32(), dev(pages)[:0], out=y)                       # no sequence
    assert (y == 7.5).all()
    ctx.attention(kv, q, i32(0, 3), i32(0), dev(pages)[:, :0].contiguous(), out=y)   # no page, no token: rows of zeros
    assert not y.any()
    before = numpy_cache(kv)
    ctx.kv_append(kv, none, none, torch.zeros(0, dtype=torch.int64, device="cuda"))
    ctx.kv_append(kv, q, q, torch.full((3,), -1, dtype=torch.int64, device="cuda"))
    assert all(np.array_equal(a, b) for a, b in zip(before, numpy_cache(kv)))


def test_more_tokens_than_a_launch_has_workgroups(ctx):
    from magnitude_amd import KvCache, rope_frequencies
    n = (1 << 23) + 5
    tell("rope of", n, "tokens")
    x = torch.randn((n, 1, 8), device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    freqs = rope_frequencies(8)[0]
    y = ctx.rope(x, pos, dev(freqs))
    pick = np.r_[0:3, (1 << 23) - 3:n]
    want = kv_ref.rotate(x[pick].cpu().numpy(), pick, freqs, "pairs", 1.0)
    np.testing.assert_allclose(y[pick].cpu().numpy(), want, rtol=0, atol=2.0 ** -22 * np.abs(x[pick].cpu().numpy()).max())
    tell("kv_append and kv_read of", n, "tokens")
    kv = KvCache.zeros(n // 256 + 1, 256, 1, 64)
    rows = torch.randn((n, 1, 64), device="cuda")
    slots = torch.arange(n - 1, -1, -1, device="cuda")
    ctx.kv_append(kv, rows, rows, slots)
    k, v = ctx.kv_read(kv, slots)
    assert torch.equal(k, v)
    some = rows[pick]
    small = KvCache.zeros(1, 16, 1, 64)
    ctx.kv_append(small, some, some, torch.arange(len(pick), device="cuda"))
    assert torch.equal(k[pick], ctx.kv_read(small, torch.arange(len(pick), device="cuda"))[0])


def test_a_call_that_does_not_fit_its_tensors_is_refused(ctx):
    from magnitude_amd import KvCache, rope_frequencies
    kv = KvCache.zeros(4, 16, 2, 64)
    x = torch.randn((3, 2, 64), device="cuda")
    q = torch.randn((3, 8, 64), device="cuda")
    freqs = dev(rope_frequencies(64)[0])
    pos, slots = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.arange(3, device="cuda")
    start, lens, pages = torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda"), torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    bad = [lambda: ctx.rope(x.double(), pos, freqs), lambda: ctx.rope(x, pos[:2], freqs), lambda: ctx.rope(x, pos.long(), freqs), lambda: ctx.rope(x, pos, freqs.float()),
           lambda: ctx.rope(x.transpose(0, 1), pos, freqs), lambda: ctx.rope(x.cpu(), pos, freqs), lambda: ctx.rope(x, pos, freqs, out=q),
           lambda: ctx.kv_append(kv, x, x[:2], slots), lambda: ctx.kv_append(kv, x, x, slots.int()), lambda: ctx.kv_append(kv, q, q, slots),
           lambda: ctx.kv_append(kv, x, x, slots, freqs=freqs), lambda: ctx.kv_append(kv, x, x, slots, q=q), lambda: ctx.kv_append(kv, x, x, slots, pos=pos, freqs=freqs, q=q[:2]),
           lambda: ctx.kv_read(kv, slots, k_out=q), lambda: ctx.kv_read(kv, slots.int()),
           lambda: ctx.attention(kv, q, start, lens.long(), pages), lambda: ctx.attention(kv, q, start[:1], lens, pages), lambda: ctx.attention(kv, q[..., :32], start, lens, pages),
           lambda: ctx.attention(kv, q, start, lens, pages, out=x), lambda: ctx.attention(kv, q, start, lens, pages[0]),
           lambda: KvCache(kv.tensors[0], kv.tensors[1][:1], kv.tensors[2], kv.tensors[3]), lambda: KvCache(kv.tensors[0].int(), *kv.tensors[1:])]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(ValueError):
        ctx.rope(x, pos, freqs, mode="neox")
    from magnitude_amd import QprojError
    with pytest.raises(QprojError):
        ctx.attention(kv, q[:, :7], start, lens, pages)
    ctx.sync()
