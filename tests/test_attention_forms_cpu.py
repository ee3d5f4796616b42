"""Attention over the paged 4-bit cache in its other forms: what needs no GPU.  Every refusal of the entry points, on a context without a
device whose launches are noted and not made."""
import pytest

from magnitude_amd import qproj
from test_attention_cpu import ATTENTION_BAD, BUF, CACHE_BAD, Dry, cache


def call(dry, name, kv, **kw):
    ref = lambda s: None if s is None else qproj.C.byref(s)
    f = dict(q=BUF, qs=4096, n=5, h=32, seqs=2, start=BUF, len=BUF, max_q=5, pages=BUF, ps=10, scale=0.1, y=2 * BUF, ys=4096)
    f.update(kw)
    head = (dry.ctx, ref(kv), f["q"], f["qs"], f["n"], f["h"], f["seqs"], f["start"], f["len"], f["max_q"], f["pages"], f["ps"])
    return dry.lib.qproj_cross_attention(*head, f["scale"], f["y"], f["ys"])


NO_WINDOW = [b for b in ATTENTION_BAD if "window" not in b]


@pytest.mark.parametrize("name,bad", [(name, b) for name in ("cross",) for b in NO_WINDOW], ids=str)
def test_bad_arguments_are_refused(name, bad):
    with Dry() as dry:
        assert call(dry, name, cache(), **bad) == 1
        assert dry.error().startswith("qproj_") and ":" in dry.error()
    assert "kernel" not in dry.plan


@pytest.mark.parametrize("bad", CACHE_BAD, ids=str)
def test_bad_caches_are_refused(bad):
    with Dry() as dry:
        for name in ("cross",):
            assert call(dry, name, cache(**bad)) == 1 and call(dry, name, None) == 1
    assert "kernel" not in dry.plan


def test_calls_that_are_taken_note_their_launches():
    with Dry() as dry:
        for page in (16, 32, 64, 128, 256):
            for dim in (64, 96, 128, 256):
                assert call(dry, "cross", cache(page_tokens=page, head_dim=dim), h=8, qs=8 * dim, ys=8 * dim) == 0, (page, dim)
        assert call(dry, "cross", cache(), n=0) == 0 and call(dry, "cross", cache(), seqs=0) == 0
    assert dry.plan.count(", all>:") == 20 and dry.plan.count("attention_kernel<") == 20


def test_null_context():
    lib = qproj.load_library()
    assert lib.qproj_cross_attention(None, None, None, 0, 0, 0, 0, None, None, 0, None, 0, 1.0, None, 0) == 1
