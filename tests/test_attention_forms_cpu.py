"""Attention over the paged 4-bit cache in its other forms: what needs no GPU.  Every refusal of the entry points, on a context without a
device whose launches are noted and not made; the buckets of distances."""
import ctypes as C
import re

import numpy as np
import pytest

import forms_ref
from magnitude_amd import qproj
from test_attention_forms_gpu import APART, APART_WIDE
from test_attention_cpu import ATTENTION_BAD, BUF, CACHE_BAD, Dry, cache


def call(dry, name, kv, **kw):
    ref = lambda s: None if s is None else qproj.C.byref(s)
    f = dict(q=BUF, qs=4096, n=5, h=32, seqs=2, start=BUF, len=BUF, max_q=5, pages=BUF, ps=10, scale=0.1, y=2 * BUF, ys=4096)
    f.update(kw)
    head = (dry.ctx, ref(kv), f["q"], f["qs"], f["n"], f["h"], f["seqs"], f["start"], f["len"], f["max_q"], f["pages"], f["ps"])
    if name == "cross":
        return dry.lib.qproj_cross_attention(*head, f["scale"], f["y"], f["ys"])
    if name == "shared":
        g = dict(groups=1, group_start=BUF, shared=BUF, max_group=2, window=0)
        g.update({k: v for k, v in f.items() if k in g})
        return dry.lib.qproj_attention_shared(*head, g["groups"], g["group_start"], g["shared"], g["max_group"], f["scale"], g["window"], f["y"], f["ys"])
    b = dict(by_distance_dev=BUF, reach=128, causal=1)
    b.update(f.get("bias", {}))
    return dry.lib.qproj_attention_biased(*head, ref(qproj.PositionBias(**b)), f["scale"], f["y"], f["ys"])


BIAS_BAD = [dict(by_distance_dev=None), dict(by_distance_dev=BUF + 2), dict(reach=-1), dict(reach=1704), dict(reach=1 << 40)]
SHARED_BAD = [dict(group_start=None), dict(shared=None), dict(groups=-1), dict(groups=0), dict(groups=65537), dict(max_group=-1)]
NO_WINDOW = [b for b in ATTENTION_BAD if "window" not in b]


@pytest.mark.parametrize("name,bad", [(name, b) for name in ("cross", "biased") for b in NO_WINDOW] + [("biased", dict(bias=b)) for b in BIAS_BAD] +
                         [("shared", b) for b in ATTENTION_BAD + SHARED_BAD], ids=str)
def test_bad_arguments_are_refused(name, bad):
    with Dry() as dry:
        assert call(dry, name, cache(), **bad) == 1
        assert dry.error().startswith("qproj_") and ":" in dry.error()
    assert "kernel" not in dry.plan


@pytest.mark.parametrize("ps", [1 << 60, (1 << 60) + 2, (1 << 63) - 1])
def test_page_tables_that_pass_64_bits_are_refused(ps):
    with Dry() as dry:
        for name in ("cross", "biased", "shared"):
            assert call(dry, name, cache(page_tokens=16), ps=ps) == 1 and "2^31" in dry.error()
    assert "kernel" not in dry.plan


@pytest.mark.parametrize("bad", CACHE_BAD, ids=str)
def test_bad_caches_are_refused(bad):
    with Dry() as dry:
        for name in ("cross", "biased", "shared"):
            assert call(dry, name, cache(**bad)) == 1 and call(dry, name, None) == 1
    assert "kernel" not in dry.plan


def test_calls_that_are_taken_note_their_launches():
    with Dry() as dry:
        for page in (16, 32, 64, 128, 256):
            for dim in (64, 96, 128, 256):
                for name in ("cross", "biased"):
                    assert call(dry, name, cache(page_tokens=page, head_dim=dim), h=8, qs=8 * dim, ys=8 * dim) == 0, (page, dim)
        for name in ("cross", "biased"):
            assert call(dry, name, cache(), n=0) == 0 and call(dry, name, cache(), seqs=0) == 0
        assert dry.lib.qproj_bias_by_distance(dry.ctx, BUF, 32, 12, BUF, 128, BUF) == 0
    assert dry.plan.count(", all>:") == 20 and dry.plan.count(", biased>:") == 20 and dry.plan.count("attention_kernel<") == 40
    assert dry.plan.count("bias_by_distance_kernel: 12 heads x 257 distances") == 1


def short(name, page, kv_heads, group, seqs, dim=64, columns=None, **kw):
    """The plan of a call with such sequences [(tokens, rows)] in a table as wide as the tests make it"""
    h, rows = kv_heads * group, [m for _, m in seqs]
    ps = max(-(-n // page) for n, _ in seqs) + 1 if columns is None else columns
    with Dry() as dry:
        assert call(dry, name, cache(page_tokens=page, n_head_kv=kv_heads, head_dim=dim, n_pages=4000), h=h, qs=h * dim, ys=h * dim, n=sum(rows), seqs=len(seqs), max_q=max(rows), ps=ps, **kw) == 0
    return dry.plan


def test_many_rows_of_short_sequences_are_taken_by_waves_of_their_own():
    for page, kv_heads, group, seqs in APART:
        for name in ("cross", "biased"):
            assert "attention_kernel<64, 2, " + {"cross": "all", "biased": "biased"}[name] + ", apart>" in short(name, page, kv_heads, group, seqs), (name, page)
            assert "apart" not in short(name, page, kv_heads, group, seqs, dim=256)
    for page, kv_heads, group, seqs in APART_WIDE:
        assert "attention_kernel<96, 1, biased, apart>" in short("biased", page, kv_heads, group, seqs, dim=96) and "apart" not in short("biased", page, kv_heads, group, seqs, dim=128)
        for dim in (96, 128):
            assert f"attention_kernel<{dim}, 1, all, apart>" in short("cross", page, kv_heads, group, seqs, dim=dim)
            assert "apart" not in short("cross", page, kv_heads, group, seqs, dim=dim, columns=-(-7 * 64 // page))      # (seven tiles)
    many = [(128, 128)] * 64                                            # 512 items of 128 rows
    assert "grid 512 x 256" in short("cross", 64, 8, 1, many, columns=2) and ", apart>" in short("cross", 64, 8, 1, many, columns=11)
    assert "apart" not in short("cross", 64, 8, 1, many, columns=12)    # (twelve tiles: 576 items)
    assert "apart" not in short("cross", 64, 16, 1, [(64, 1)] * 4000, columns=1)       # single rows
    assert "apart" not in short("shared", 64, 8, 1, many, columns=2)


@pytest.mark.parametrize("reach,group,heads", [(0, 16, 16), (128, 16, 8), (128, 9, 5), (128, 4, 4), (500, 8, 3), (1703, 7, 1)])
def test_an_item_has_as_many_heads_as_there_is_room_for_their_biases(reach, group, heads):
    with Dry() as dry:
        assert call(dry, "biased", cache(n_head_kv=2), h=2 * group, qs=256 * group, ys=256 * group, n=1, seqs=1, max_q=1, bias=dict(reach=reach)) == 0
    taken = int(re.search(r"heads in 2 x (\d+) of (\d+)", dry.plan).group(2))
    assert taken == heads and taken * (2 * reach + 193) <= 3600


# ---- groups that share their first tokens -----------------------------------------------------------------------------------
def plan(heads_kv=8, group=4, dim=128, page=64, **kw):
    h = heads_kv * group
    with Dry() as dry:
        assert call(dry, "shared", cache(n_pages=1 << 18, page_tokens=page, n_head_kv=heads_kv, head_dim=dim), h=h, qs=h * dim, ys=h * dim, **kw) == 0
    return dry.plan


def test_calls_with_nothing_to_share_are_the_causal_kernel_s():
    many = dict(seqs=16, n=16, max_q=1, ps=2048, max_group=16)
    assert "attention_kernel<128, 2, prefix>" in plan(**many)
    for kw in (dict(window=100), dict(max_group=1), dict(max_group=0), dict(max_q=5, n=80), dict(max_q=0)):
        assert ", prefix>" not in plan(**{**many, **kw}) and "attention_kernel<128" in plan(**{**many, **kw}), kw
    assert ", prefix>" in plan(**{**many, "max_q": 4, "n": 64}) and ", prefix>" in plan(group=16, **many) and ", prefix>" not in plan(group=17, **many)
    assert "attention_kernel<256, 1, prefix>" in plan(dim=256, **many) and ", prefix>" not in plan(dim=256, **{**many, "max_q": 3, "n": 48})
    assert ", prefix>" in plan(**{**many, "window": 2048 * 64})     # (as long as a sequence can be)
    assert "kernel" not in plan(**{**many, "n": 0}) and "kernel" not in plan(**{**many, "seqs": 0, "groups": 0})


def test_an_item_takes_sequences_alike():
    m = lambda text: tuple(int(v) for v in re.search(r", (\d+) tokens x (\d+) a sequence", text).groups())
    assert m(plan(seqs=48, n=48, max_q=1, ps=2048, max_group=48)) == (8, 6)
    assert m(plan(seqs=9, n=9, max_q=1, ps=2048, max_group=9)) == (5, 2)              # 5 + 4, not 8 + 1
    assert m(plan(heads_kv=2, group=1, seqs=64, n=64, max_q=1, ps=4096, max_group=64)) == (32, 2)
    assert m(plan(seqs=30, n=90, max_q=3, ps=2048, max_group=30)) == (6, 15)          # two sequences of three rows
    assert m(plan(seqs=2, n=2, max_q=1, ps=20, max_group=2)) == (2, 1)


def test_more_places_than_32_bits_hold_are_the_causal_kernel_s():
    most = dict(heads_kv=1, group=2, page=16, seqs=65536, n=65536, max_q=4, ps=4)
    assert ", prefix>" not in plan(groups=65536, max_group=65536, **most)
    assert ", prefix>" in plan(groups=65536, max_group=16, **most) and ", prefix>" in plan(groups=16, max_group=65536, **most)


def test_long_caches_have_items_of_32_columns():
    for ps in (64, 511, 512, 1024):
        kw = dict(seqs=48, n=48, max_q=1, max_group=48, ps=ps)
        assert ("attention_kernel<128, 2, prefix>" in plan(**kw)) == (ps >= 512) and ("attention_kernel<128, 1, prefix>" in plan(**kw)) == (ps < 512), ps
    assert "attention_kernel<128, 2, prefix>" in plan(group=12, seqs=8, n=8, max_q=1, max_group=8, ps=64)      # (16 hold one sequence)


def shared_pieces(q_start, kv_len, max_q, group_start, shared, most_len, together, heads, grid, max_group, later=None, n=None):
    f = qproj.load_library().qproj_internal_attention_shared_pieces
    f.restype, f.argtypes = C.c_int64, [C.c_void_p] * 3 + [C.c_int64] * 3 + [C.c_void_p] * 2 + [C.c_int64] * 6 + [C.c_void_p, C.c_int64]
    a = [np.ascontiguousarray(v, np.int32) for v in (q_start, kv_len, kv_len if later is None else later, group_start, shared)]
    room = 1 << 17
    out = np.zeros((room, 9), np.int32)
    got = f(*[v.ctypes.data for v in a[:3]], len(kv_len), q_start[-1] if n is None else n, max_q, a[3].ctypes.data, a[4].ctypes.data, len(shared), max_group, most_len,
            together, heads, grid, out.ctypes.data, room)
    assert 0 <= got <= room, "a workgroup does not come to an end"
    return out[:got]


def shared_items(q_start, kv_len, group_start, shared, together):
    """{(group, item of it): turns}: whole tiles that lie before the rows of all of an item's sequences that have any, then every sequence's own"""
    got = {}
    for g in range(len(shared)):
        for tile, first in enumerate(range(group_start[g], group_start[g + 1], together)):
            rows = [(kv_len[s], q_start[s + 1] - q_start[s]) for s in range(first, min(first + together, group_start[g + 1])) if q_start[s + 1] > q_start[s]]
            same = max(0, min([shared[g]] + [n - m for n, m in rows])) // 64 if rows else 0
            got[g, tile] = -(-max(1, same + sum(-(-n // 64) - same for n, _ in rows)) // 4)
    return got


@pytest.mark.parametrize("grid", [3, 64, 512])
@pytest.mark.parametrize("heads,together,groups", [   # groups: (shared, [(tokens, rows)])
    (8, 8, [(1000, [(1000 + 30 * i, 1) for i in range(1, 17)])]),
    (1, 2, [(64, [(65, 1), (100, 2), (64, 1)]), (0, [(500, 1)] * 3), (100000, [(4000, 1), (3000, 2), (70, 1), (5, 1), (0, 0)])]),
    (2, 32, [(8192, [(8192 + 7 * i, 1) for i in range(1, 65)])]),
    (4, 3, [(500, [(i, min(i, 2)) for i in range(40)]), (10, []), (300, [(400, 0), (350, 0)]), (77, [(900, 1)])]),
    (1, 5, [(128, [(128 + 300 * (i % 7) + 1, 1) for i in range(5)]) for _ in range(100)]),
])
def test_every_turn_of_groups_has_one_workgroup(heads, together, groups, grid):
    seqs = [s for _, g in groups for s in g]
    lens, q_start = [n for n, _ in seqs], np.cumsum([0] + [m for _, m in seqs]).tolist()
    group_start, shared = np.cumsum([0] + [len(g) for _, g in groups]).tolist(), [n for n, _ in groups]
    max_group = max(len(g) for _, g in groups)
    got = shared_pieces(q_start, lens, 2, group_start, shared, max(lens), together, heads, grid, max_group)
    want = shared_items(q_start, lens, group_start, shared, together)
    taken = {}
    for row in got.tolist():
        taken.setdefault(tuple(row[1:4]), []).append(row)
    assert set(taken) == {(h, s, t) for h in range(heads) for s, t in want} and (got[:, 0] < grid).all()
    for (h, s, t), parts in taken.items():
        parts.sort(key=lambda r: r[4])
        assert parts[0][6] == want[s, t] and parts[0][4] == 0 and parts[-1][5] == want[s, t]
        assert all(a[5] == b[4] for a, b in zip(parts, parts[1:]))
        assert all(r[7:] == parts[0][7:] for r in parts) and len(parts) == parts[0][8] - parts[0][7] + 1
        assert len({r[0] for r in parts}) == len(parts)


@pytest.mark.parametrize("items,grid", [(9, 8), (10, 8), (15, 8), (16, 8), (616, 512), (1025, 512)])
def test_no_workgroup_has_an_item_more_than_the_others(items, grid):
    """items of 20 turns, some grids full and a little more: cut where whole ones would leave workgroups more than two turns from each other"""
    lens, n = [20 * 256] * items, list(range(items + 1))
    got = shared_pieces(n, lens, 1, n, [0] * items, max(lens), 2, 1, grid, 1)
    turns = np.bincount(got[:, 0], weights=got[:, 5] - got[:, 4], minlength=grid)
    assert turns.sum() == 20 * items and turns.max() <= 20 * items / grid + 3 + 2 * -(-items // grid)
    assert (len(got) == items) == (items == 16)


def test_groups_and_lengths_that_are_wrong_come_to_an_end():
    """bounds that do not hold, and lengths that change between the count and the search: pieces are any, but every workgroup ends"""
    rng = np.random.default_rng(3)
    for _ in range(300):
        n_seq, n_groups = int(rng.integers(1, 30)), int(rng.integers(1, 8))
        q_start = np.sort(rng.integers(0, 2 * n_seq, n_seq + 1)) if rng.random() < 0.7 else rng.integers(-3, 2 * n_seq, n_seq + 1)
        lens, later = rng.integers(-2, 3000, n_seq), rng.integers(-2, 3000, n_seq)
        group_start = np.sort(rng.integers(0, n_seq + 1, n_groups + 1)) if rng.random() < 0.5 else rng.integers(-2, n_seq + 3, n_groups + 1)
        shared_pieces(q_start.tolist(), lens, 2, group_start, rng.integers(-5, 4000, n_groups), 2900, int(rng.integers(2, 9)), int(rng.integers(1, 5)), int(rng.integers(1, 200)),
                      int(rng.integers(1, n_seq + 1)), later, n=2 * n_seq)


def test_groups_that_repeat_sequences_are_not_counted_to_their_end():
    n = 3000
    groups = [0, n, n, 0] * 4000                           # every other good one has all sequences
    assert len(shared_pieces(list(range(n + 1)), [100] * n, 1, groups + [0], [0] * len(groups), 100, 2, 1, 8, n)) == 0


# ---- buckets --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("both", [True, False])
@pytest.mark.parametrize("n,reach", [(32, 128), (32, 129), (32, 20), (4, 3), (8, 128), (64, 500), (64, 1703), (320, 800), (6, 7)])
def test_buckets(n, reach, both):
    """against the definition in whole numbers; reach 128 of 32 buckets has powers that meet exactly"""
    got = qproj.relative_buckets(n, reach, both)
    want = [forms_ref.bucket(n, reach, both, d) for d in range(-reach, reach + 1)]
    assert got.dtype == np.int32 and got.tolist() == want
    assert (np.diff(got[:reach + 1]) <= 0).all() and got[reach] == 0 and got.max() < n


def test_buckets_by_hand():
    one = qproj.relative_buckets(32, 128, False)[::-1][128:]        # of 0 .. 128 tokens before the row
    assert one[:17].tolist() == list(range(17)) and one[128] == 31 and one[127] == 31 and one[32] == 21     # 16 + floor(log 2 / log 8 * 16)
    two = qproj.relative_buckets(32, 128)
    assert two[128 - 8] == 8 and two[128 + 8] == 24 and two[128 - 16] == 10 and two[128 + 16] == 26 and two[128 + 3] == 19 and two[0] == 15 and two[-1] == 31


@pytest.mark.parametrize("n,reach,both", [(0, 10, False), (1, 10, False), (2, 10, True), (33, 128, True), (32, 16, False), (32, 8, True), (32, 1704, True), (32, -1, True), (-4, 10, False),
                                          ((1 << 20) + 2, 1000, True)])
def test_bucket_refusals(n, reach, both):
    with pytest.raises(qproj.QprojError) as e:
        qproj.relative_buckets(n, reach, both)
    assert e.value.status == 1


@pytest.mark.parametrize("bad", [dict(table=None), dict(buckets=None), dict(out=None), dict(n=0), dict(n=-1), dict(n=(1 << 20) + 1), dict(h=0), dict(h=4097), dict(reach=-1), dict(reach=1704)], ids=str)
def test_bad_tables_are_refused(bad):
    f = dict(table=BUF, n=32, h=12, buckets=BUF, reach=128, out=BUF)
    f.update(bad)
    with Dry() as dry:
        assert dry.lib.qproj_bias_by_distance(dry.ctx, f["table"], f["n"], f["h"], f["buckets"], f["reach"], f["out"]) == 1
        assert dry.error().startswith("qproj_bias_by_distance: ")
    assert "kernel" not in dry.plan


def test_null_context():
    lib = qproj.load_library()
    assert lib.qproj_cross_attention(None, None, None, 0, 0, 0, 0, None, None, 0, None, 0, 1.0, None, 0) == 1
    assert lib.qproj_attention_biased(None, None, None, 0, 0, 0, 0, None, None, 0, None, 0, None, 1.0, None, 0) == 1
    assert lib.qproj_attention_shared(None, None, None, 0, 0, 0, 0, None, None, 0, None, 0, 0, None, None, 0, 1.0, 0, None, 0) == 1
    assert lib.qproj_bias_by_distance(None, None, 0, 0, None, 0, None) == 1
    assert lib.qproj_relative_buckets(32, 128, 1, None) == 1
