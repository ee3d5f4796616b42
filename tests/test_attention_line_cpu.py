"""How attention's work is shared out among workgroups, on the CPU: the grid from the plan of a call on a context without a device, the
pieces from the kernel's own arithmetic compiled for the host.  Every turn of every item has to be taken by one workgroup."""
import ctypes as C
import re

import numpy as np
import pytest

from test_attention_cpu import Dry, cache, call


def plan(heads_kv, group, n, seqs, max_q, table_pages, page, dim=128, window=0):
    """(tokens of an item, heads of the line, workgroups) of the launch of such a call"""
    m = re.search(r"heads in (\d+) x (\d+) of \d+, (\d+) tokens x (\d+) a sequence of rows, grid (\d+) x", plan_text(heads_kv, group, n, seqs, max_q, table_pages, page, dim, window))
    kv, splits, tokens, _, grid = (int(v) for v in m.groups())
    return tokens, kv * splits, grid


def plan_text(heads_kv, group, n, seqs, max_q, table_pages, page, dim=128, window=0):
    heads = heads_kv * group
    with Dry() as dry:
        assert call(dry, "attention", cache(n_pages=max(1, seqs * table_pages), page_tokens=page, n_head_kv=heads_kv, head_dim=dim), h=heads, qs=heads * dim,
                    ys=heads * dim, n=n, seqs=seqs, max_q=max_q, ps=table_pages, window=window) == 0
    return dry.plan


def pieces(q_start, kv_len, n, max_q, most_len, window, tokens, heads, grid, later=None):
    """[workgroup, head, sequence, row tile, from, to, turns, first stretch, last stretch] of every piece"""
    from magnitude_amd import qproj
    f = qproj.load_library().qproj_internal_attention_pieces
    f.restype, f.argtypes = C.c_int64, [C.c_void_p] * 3 + [C.c_int64] * 8 + [C.c_void_p, C.c_int64]
    start, lens = np.ascontiguousarray(q_start, np.int32), np.ascontiguousarray(kv_len, np.int32)
    later = lens if later is None else np.ascontiguousarray(later, np.int32)
    room = 1 << 17
    out = np.zeros((room, 9), np.int32)
    got = f(start.ctypes.data, lens.ctypes.data, later.ctypes.data, len(lens), n, max_q, most_len, window, tokens, heads, grid, out.ctypes.data, room)
    assert 0 <= got <= room, "a workgroup does not come to an end"
    return out[:got]


def items(q_start, kv_len, tokens, window):
    """{(sequence, row tile): turns}, from the definition: rows at positions lo .. hi see tokens max(0, lo - window + 1) .. hi, 256 of them a turn from
    a multiple of 64 on"""
    got = {}
    for s in range(len(kv_len)):
        count = q_start[s + 1] - q_start[s]
        for tile in range(-(-count // tokens)):
            lo = kv_len[s] - count + tile * tokens
            hi = lo + min(tokens, count - tile * tokens) - 1
            see = max(0, lo - window + 1) if window else 0
            got[s, tile] = 1 if hi < 0 else -(-(hi // 64 - see // 64 + 1) // 4)
    return got


def check(heads_kv, group, seqs, page, spare=0, window=0, max_q=None, dim=128):
    """seqs: (tokens in the cache, new ones)"""
    lens, q_start = [n for n, _ in seqs], np.cumsum([0] + [m for _, m in seqs]).tolist()
    n, max_q = q_start[-1], max_q or max(m for _, m in seqs)
    table = max(-(-v // page) for v in lens) + spare
    tokens, heads, grid = plan(heads_kv, group, n, len(seqs), max_q, table, page, dim, window)
    got = pieces(q_start, lens, n, max_q, table * page, window, tokens, heads, grid)
    want = items(q_start, lens, tokens, window)
    assert (got[:, 0] < grid).all()
    taken = {}
    for row in got.tolist():
        taken.setdefault(tuple(row[1:4]), []).append(row)
    assert set(taken) == {(h, s, t) for h in range(heads) for s, t in want}
    for (h, s, t), parts in taken.items():
        parts.sort(key=lambda r: r[4])
        assert parts[0][6] == want[s, t] and parts[0][4] == 0 and parts[-1][5] == want[s, t]
        assert all(a[5] == b[4] for a, b in zip(parts, parts[1:]))                       # one after the other, nothing between
        assert all(r[7:] == parts[0][7:] for r in parts) and len(parts) == parts[0][8] - parts[0][7] + 1     # as many as the item is said to have
        assert len({r[0] for r in parts}) == len(parts)
    return len(got)


def test_every_stretch_has_one_workgroup():
    """the numbering reaches each of `active` stretches once from any grid that has as many workgroups"""
    for active in range(1, 700):
        # one head, one sequence that needs exactly `active` turns, in a table of exactly its pages
        for grid in {active, active + 1, active + 5, 1024}:
            got = pieces([0, 1], [256 * active - 3], 1, 1, 256 * active, 0, 16, 1, grid)
            assert sorted(got[:, 4]) == list(range(active)) and len(set(got[:, 0])) == active


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("spare", [0, 1, 300])
def test_every_length_of_one_token(page, spare):
    for heads_kv, group in ((1, 4), (1, 32), (2, 7), (3, 1), (4, 8), (5, 3), (7, 2), (8, 4)):
        for length in list(range(1, 4000, 137)) + [255, 256, 257, 512, 513, 1025, 1300, 1537, 2049, 2100, 9000, 22604]:
            check(heads_kv, group, [(length, 1)], page, spare)


@pytest.mark.parametrize("heads_kv", range(1, 9))
def test_shapes(heads_kv):
    rng = np.random.default_rng(heads_kv)
    for group in list(range(1, 17)) + [71]:
        for _ in range(12):
            most = int(np.exp(rng.uniform(0, np.log(9000))))
            rows = int(rng.choice([1, 1, 2, 8, 27, 64]))
            seqs = [(int(rng.integers(0, most + 1)), int(rng.integers(0 if rows > 1 else 1, rows + 1))) for _ in range(rng.integers(1, 7))]
            if rng.random() < 0.5:
                seqs = [(most, rows)] * len(seqs)
            seqs[0] = (max(1, seqs[0][0]), max(1, seqs[0][1]))
            check(heads_kv, group, seqs, int(rng.choice([16, 64, 256])), int(rng.choice([0, 0, 1, 500])), int(rng.choice([0, 0, 1, 100, 5000])),
                  dim=int(rng.choice([64, 128, 256])))


def test_many_sequences():
    """more places than threads, so that the line is searched again for every item"""
    rng = np.random.default_rng(9)
    for n in (255, 256, 257, 700):
        check(2, 4, [(int(v), 1) for v in rng.integers(1, 600, n)], 16)
        check(1, 4, [(30000, 1)] + [(int(v), 1) for v in rng.integers(1, 600, n - 1)], 16, window=7000)
    check(2, 4, [(int(v), 40) for v in rng.integers(0, 600, 30)] + [(2000, 300)], 16, max_q=331)


@pytest.mark.parametrize("window", [1, 2, 1 << 20, (1 << 31) - 2, (1 << 31) - 1])
def test_windows_of_any_size_behind_more_rows_than_tokens(window):
    """rows that stand before the first token: position minus window must not leave 32 bits"""
    q_start, lens = [0, 8, 40, 41], [3, 0, 700]
    for tokens in (1, 4, 16):
        got = pieces(q_start, lens, 41, 32, 1024, window, tokens, 2, 64)
        want = items(q_start, lens, tokens, window)
        for (s, t), turns in want.items():
            for head in range(2):
                mine = got[(got[:, 1:4] == (head, s, t)).all(1)]
                assert (mine[:, 6] == turns).all() and (mine[:, 5] - mine[:, 4]).sum() == turns
        assert len({tuple(r) for r in got[:, 1:4].tolist()}) == 2 * len(want)


@pytest.mark.parametrize("seqs,most", [(300, 400), (300, 20000), (257, 60000), (600, 3000), (40, 9000)])
def test_lengths_that_change_during_a_call(seqs, most):
    """what a workgroup finds where it looks again is not what it counted: it comes to an end all the same, and stays among the stretches there are"""
    rng = np.random.default_rng(seqs + most)
    for i in range(60):
        lens, later = rng.integers(0, most + 1, seqs), rng.integers(0, most + 1, seqs)
        if i % 4 == 1:
            later = np.minimum(later, lens)
        if i % 4 == 2:
            later = np.maximum(later, lens)
        if i % 4 == 3:
            later = np.where(rng.random(seqs) < 0.01, later, lens)
        heads, grid = int(rng.integers(1, 9)), int(rng.choice([7, 64, 256, 512]))
        got = pieces(np.arange(seqs + 1), lens, seqs, 1, most, 0, 4, heads, grid, later)
        assert (got[:, 0] < grid).all() and (got[:, 1] < heads).all() and (got[:, 2] < seqs).all()
        assert (0 <= got[:, 4]).all() and (got[:, 4] < got[:, 5]).all() and (got[:, 5] <= got[:, 6]).all()
        assert (0 <= got[:, 7]).all() and (got[:, 7] <= got[:, 8]).all() and (got[:, 8] < grid).all()


@pytest.mark.parametrize("seqs,rows,most", [(64, 8192, 1 << 23), (33, 100, 1 << 28), (41, 100, 1 << 28), (9, 60000, 1 << 20), (3, 50, 3000)])
def test_sequences_that_share_rows(seqs, rows, most):
    """q_start that falls again and again: the sequences between are within bounds one by one, together they can be more than 32 bits count"""
    for tokens in (1, 4, 8):
        assert len(pieces([rows * (i % 2) for i in range(seqs + 1)], [most] * seqs, rows, rows, most, 0, tokens, 8, 512)) == 0
    # one that falls among others that do not: the others are taken
    start = np.array([0, 3, 2, 5, 9], np.int32)
    got = pieces(start, [700, 700, 300, 900], 9, 9, 1024, 0, 4, 2, 64)
    assert {tuple(r) for r in got[:, 1:4].tolist()} == {(h, s, t) for h in range(2) for s, t in items(start.tolist(), [700, 700, 300, 900], 4, 0)}


def test_which_workgroups_go_first():
    """the second ones of the compute units (256 on a context without a device); all where one item is cut into many parts"""
    assert "first from 256 on" in plan_text(8, 4, 4096, 1, 4096, 64, 64)
    assert "first from 256 on" in plan_text(8, 4, 48, 48, 1, 128, 64)
    assert "first from 0 on" in plan_text(8, 4, 1, 1, 1, 2048, 64)


def test_no_rows_allowed_is_a_launch_that_looks():
    """max_q 0: sequences without rows are fine, one with a row is reported by the kernel"""
    assert "attention_kernel<" in plan_text(8, 4, 5, 3, 0, 10, 64)
    assert len(pieces([0, 0, 0], [100, 0], 5, 0, 640, 0, 4, 8, 64)) == 0
    assert len(pieces([0, 3, 5], [100, 60], 5, 0, 640, 0, 4, 8, 64)) == 0
