"""Attention over the paged 4-bit cache in its other forms: what needs no GPU.  Every refusal of the entry points, on a context without a
device whose launches are noted and not made; the buckets of distances."""
import re

import numpy as np
import pytest

import forms_ref
from magnitude_amd import qproj
from test_attention_cpu import ATTENTION_BAD, BUF, CACHE_BAD, Dry, cache


def call(dry, name, kv, **kw):
    ref = lambda s: None if s is None else qproj.C.byref(s)
    f = dict(q=BUF, qs=4096, n=5, h=32, seqs=2, start=BUF, len=BUF, max_q=5, pages=BUF, ps=10, scale=0.1, y=2 * BUF, ys=4096)
    f.update(kw)
    head = (dry.ctx, ref(kv), f["q"], f["qs"], f["n"], f["h"], f["seqs"], f["start"], f["len"], f["max_q"], f["pages"], f["ps"])
    if name == "cross":
        return dry.lib.qproj_cross_attention(*head, f["scale"], f["y"], f["ys"])
    b = dict(by_distance_dev=BUF, reach=128, causal=1)
    b.update(f.get("bias", {}))
    return dry.lib.qproj_attention_biased(*head, ref(qproj.PositionBias(**b)), f["scale"], f["y"], f["ys"])


BIAS_BAD = [dict(by_distance_dev=None), dict(by_distance_dev=BUF + 2), dict(reach=-1), dict(reach=1704), dict(reach=1 << 40)]
NO_WINDOW = [b for b in ATTENTION_BAD if "window" not in b]


@pytest.mark.parametrize("name,bad", [(name, b) for name in ("cross", "biased") for b in NO_WINDOW] + [("biased", dict(bias=b)) for b in BIAS_BAD], ids=str)
def test_bad_arguments_are_refused(name, bad):
    with Dry() as dry:
        assert call(dry, name, cache(), **bad) == 1
        assert dry.error().startswith("qproj_") and ":" in dry.error()
    assert "kernel" not in dry.plan


@pytest.mark.parametrize("bad", CACHE_BAD, ids=str)
def test_bad_caches_are_refused(bad):
    with Dry() as dry:
        for name in ("cross", "biased"):
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


@pytest.mark.parametrize("reach,group,heads", [(0, 16, 16), (128, 16, 8), (128, 9, 5), (128, 4, 4), (500, 8, 3), (1703, 7, 1)])
def test_an_item_has_as_many_heads_as_there_is_room_for_their_biases(reach, group, heads):
    with Dry() as dry:
        assert call(dry, "biased", cache(n_head_kv=2), h=2 * group, qs=256 * group, ys=256 * group, n=1, seqs=1, max_q=1, bias=dict(reach=reach)) == 0
    taken = int(re.search(r"heads in 2 x (\d+) of (\d+)", dry.plan).group(2))
    assert taken == heads and taken * (2 * reach + 193) <= 3600


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
    assert lib.qproj_bias_by_distance(None, None, 0, 0, None, 0, None) == 1
    assert lib.qproj_relative_buckets(32, 128, 1, None) == 1
