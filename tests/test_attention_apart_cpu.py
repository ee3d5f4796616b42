"""How attention's work is shared out where every wave has rows of its own, by the kernel's own arithmetic compiled for the host: items stay whole, every one
has one workgroup."""
import ctypes as C

import numpy as np
import pytest

from magnitude_amd import qproj
from test_attention_apart_gpu import CHUNKS, TEXTS
from test_attention_forms_cpu import short


def pieces(q_start, kv_len, max_q, all_seen, most_len, tokens, heads, grid, later=None, n=None):
    f = qproj.load_library().qproj_internal_attention_apart_pieces
    f.restype, f.argtypes = C.c_int64, [C.c_void_p] * 3 + [C.c_int64] * 3 + [C.c_int32] + [C.c_int64] * 4 + [C.c_void_p, C.c_int64]
    a = [np.ascontiguousarray(v, np.int32) for v in (q_start, kv_len, kv_len if later is None else later)]
    room = 1 << 17
    out = np.zeros((room, 9), np.int32)
    got = f(*[v.ctypes.data for v in a], len(kv_len), q_start[-1] if n is None else n, max_q, all_seen, most_len, tokens, heads, grid, out.ctypes.data, room)
    assert 0 <= got <= room, "a workgroup does not come to an end"
    return out[:got]


def items(q_start, kv_len, tokens, all_seen):
    """{(sequence, row tile): tiles of 64 tokens up to the last one that any of its rows sees}"""
    got = {}
    for s in range(len(kv_len)):
        rows = q_start[s + 1] - q_start[s]
        for tile in range(-(-rows // tokens)):
            last = kv_len[s] - 1 if all_seen else kv_len[s] - rows + min(rows, (tile + 1) * tokens) - 1
            got[s, tile] = max(0, last) // 64 + 1
    return got


SEQS = {"few": [(200, 200), (129, 129), (60, 60), (190, 130)],
        "none": [(100, 250), (1, 130), (0, 140), (65, 65), (0, 0), (64, 0), (3, 1)],
        "255 places": [(64 + i % 65, 20 + i % 45) for i in range(255)],
        "257 places": [(64 + i % 65, 20 + i % 45) for i in range(257)],
        "400": [(64 + 7 * i % 65, 64 + 7 * i % 65) for i in range(400)],
        "mostly without an item": [(90, 1 + i % 40) for i in range(300)] + [(700, 600)]}


@pytest.mark.parametrize("grid", [7, 64, 512])
@pytest.mark.parametrize("all_seen", [0, 1])
@pytest.mark.parametrize("heads,tokens", [(1, 128), (8, 128), (3, 64), (2, 24)])
@pytest.mark.parametrize("seqs", SEQS.values(), ids=SEQS)
def test_every_item_has_one_workgroup(seqs, heads, tokens, all_seen, grid):
    lens, q_start = [n for n, _ in seqs], np.cumsum([0] + [m for _, m in seqs]).tolist()
    got = pieces(q_start, lens, max(m for _, m in seqs), all_seen, max(lens), tokens, heads, grid)
    want = items(q_start, lens, tokens, all_seen)
    assert {tuple(r[1:4]): r[6] for r in got.tolist()} == {(h, s, t): n for h in range(heads) for (s, t), n in want.items()} and len(got) == heads * len(want)
    assert (got[:, 4] == 0).all() and (got[:, 5] == got[:, 6]).all() and (got[:, 0] < grid).all()
    dealt = np.bincount(got[:, 0], minlength=grid)
    assert dealt.max() - dealt.min() <= 1


@pytest.mark.parametrize("seqs,most,rows", [(40, 200, 90), (257, 128, 64), (400, 300, 40)])
def test_lengths_that_change_during_a_call(seqs, most, rows):
    """what a workgroup finds where it looks again is not what it counted: it comes to an end all the same"""
    rng = np.random.default_rng(seqs)
    for i in range(40):
        q_start = np.cumsum(np.r_[0, rng.integers(0, rows + 1, seqs)])
        if i % 4 == 3:
            q_start = rng.integers(-3, seqs * rows, seqs + 1)      # bounds that do not hold
        lens, later = rng.integers(-1, most + 1, seqs), rng.integers(-1, most + 1, seqs)
        got = pieces(q_start.tolist(), lens, rows, i % 2, most, 64, int(rng.integers(1, 9)), int(rng.choice([7, 64, 512])), later, n=seqs * rows)
        assert (0 <= got[:, 4]).all() and (got[:, 4] < got[:, 5]).all() and (got[:, 2] >= 0).all() and (got[:, 2] < seqs).all()


def test_hundreds_of_short_texts_are_taken_so():
    """the calls of the tests on the GPU"""
    for seqs in (TEXTS, CHUNKS):
        for name, kernel in (("cross", "all"), ("biased", "biased")):
            assert f"attention_kernel<64, 2, {kernel}, apart>" in short(name, 64, 4, 1, seqs)
            assert f"attention_kernel<96, 1, {kernel}, apart>" in short(name, 64, 4, 1, seqs, dim=96)
        assert "attention_kernel<128, 1, all, apart>" in short("cross", 64, 4, 1, seqs, dim=128)
