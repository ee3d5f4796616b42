"""Rotary positions, the paged 4-bit cache and attention: what needs no GPU.  The frequency table against formulas in 64 bits,
the plain statements of the cache's layout against each other, and every refusal of the entry points, on a context without
a device whose launches are noted and not made."""
import ctypes as C
import math

import numpy as np
import pytest

import kv_ref
from magnitude_amd import qproj


def test_plain_frequencies():
    f, m = qproj.rope_frequencies(128, base=500000.0)
    assert m == 1.0 and f.dtype == np.float64
    np.testing.assert_allclose(f, 500000.0 ** (-np.arange(64) / 64), rtol=1e-15)
    g, _ = qproj.rope_frequencies(128, base=500000.0, freq_scale=0.25)
    np.testing.assert_allclose(g, f / 4, rtol=1e-15)
    factors = np.linspace(1, 8, 64).astype(np.float32)
    g, _ = qproj.rope_frequencies(128, base=500000.0, factors=factors)
    np.testing.assert_allclose(g, f / factors.astype(np.float64), rtol=1e-15)


@pytest.mark.parametrize("n_dims,base,stretch,trained", [(128, 10000.0, 4.0, 4096), (64, 1000000.0, 32.0, 32768), (96, 10000.0, 16.0, 8192)])
def test_yarn_frequencies(n_dims, base, stretch, trained):
    f, m = qproj.rope_frequencies(n_dims, base=base, freq_scale=1 / stretch, n_ctx_orig=trained, ext_factor=1.0)
    plain = base ** (-2 * np.arange(n_dims // 2) / n_dims)
    turns = trained * plain / (2 * np.pi)
    assert m == pytest.approx(1 + 0.1 * math.log(stretch), rel=1e-6)
    # the ramp's ends are whole pairs: one pair either side of the exact count of turns may be on it
    fast, slow = np.flatnonzero(turns > 32 * base ** (2 / n_dims)), np.flatnonzero(turns < base ** (-2 / n_dims))
    np.testing.assert_allclose(f[fast], plain[fast], rtol=1e-15)
    np.testing.assert_allclose(f[slow], plain[slow] / stretch, rtol=1e-15)
    ratio = plain / f
    assert (np.diff(ratio) >= -1e-12).all() and ratio[0] == pytest.approx(1) and ratio[-1] == pytest.approx(stretch)
    low = max(0, math.floor(n_dims * math.log(trained / (32 * 2 * math.pi)) / (2 * math.log(base))))
    high = min(n_dims - 1, math.ceil(n_dims * math.log(trained / (2 * math.pi)) / (2 * math.log(base))))
    keep = 1 - np.clip((np.arange(n_dims // 2) - low) / max(0.001, high - low), 0, 1)
    np.testing.assert_allclose(f, plain / stretch * (1 - keep) + plain * keep, rtol=1e-14)


@pytest.mark.parametrize("n_dims,kw", [(0, {}), (63, {}), (64, {"base": 1.0}), (64, {"base": float("nan")}), (64, {"freq_scale": 0.0}),
                                       (64, {"ext_factor": 1.0}), (64, {"ext_factor": -1.0}), (64, {"ext_factor": 2.0, "n_ctx_orig": 4096}),
                                       (64, {"ext_factor": 1.0, "n_ctx_orig": 4096, "beta_fast": 0.0})])
def test_frequency_refusals(n_dims, kw):
    with pytest.raises(qproj.QprojError) as e:
        qproj.rope_frequencies(n_dims, **kw)
    assert e.value.status == 1


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_layout_goes_both_ways(dim):
    rng = np.random.default_rng(dim)
    n = rng.integers(0, 16, (3, 5, dim // 32, 32), dtype=np.uint8)
    flat = n.reshape(3, 5, dim)
    assert np.array_equal(kv_ref.unpack_keys(kv_ref.pack_keys(n)), flat)
    assert np.array_equal(kv_ref.unpack_values(kv_ref.pack_values(n)), flat)
    # as the header says it: word w of a row of B blocks holds values 8 * (w / B) .. + 7 of block w % B
    words, blocks = kv_ref.pack_keys(n).view(np.uint32), dim // 32
    for w in range(4 * blocks):
        for j in range(8):
            assert np.array_equal((words[..., w] >> (4 * j)) & 15, n[..., w % blocks, 8 * (w // blocks) + j])


# ---- refusals: a dry context checks arguments and notes launches --------------------------------------------------------
BUF = 1 << 20     # an aligned address that nothing reads


class Dry:
    def __init__(self):
        self.lib = qproj.load_library()
        self.lib.qproj_internal_dry_begin.restype = C.c_void_p
        self.lib.qproj_internal_dry_end.argtypes = [C.c_void_p, C.c_char_p, C.c_size_t]

    def __enter__(self):
        self.ctx = self.lib.qproj_internal_dry_begin()
        return self

    def __exit__(self, *exc):
        buf = C.create_string_buffer(8192)
        assert self.lib.qproj_internal_dry_end(self.ctx, buf, len(buf)) == 0
        self.plan = buf.value.decode()

    def error(self):
        return self.lib.qproj_last_error(self.ctx).decode()


def cache(**kw):
    f = dict(k_codes=BUF, k_scales=BUF, v_codes=BUF, v_scales=BUF, n_pages=100, page_tokens=64, n_head_kv=8, head_dim=128)
    f.update(kw)
    return qproj.KvPlanes(*[f[n] for n, _ in qproj.KvPlanes._fields_])


def rotation(**kw):
    f = dict(pos_dev=BUF, freqs_dev=BUF, n_dims=128, mode=0, magnitude=1.0)
    f.update(kw)
    return qproj.Rotation(*[f[n] for n, _ in qproj.Rotation._fields_])


def call(dry, name, kv=None, rot=None, **kw):
    ref = lambda s: None if s is None else C.byref(s)
    if name == "rope":
        f = dict(x=BUF, xs=4096, n=5, h=32, d=128, y=2 * BUF, ys=4096)
        f.update(kw)
        return dry.lib.qproj_rope(dry.ctx, ref(rot), f["x"], f["xs"], f["n"], f["h"], f["d"], f["y"], f["ys"])
    if name == "append":
        f = dict(k=BUF, ks=1024, v=BUF, vs=1024, n=5, slots=BUF, q=None, qs=0, h=0, qo=None, qos=0)
        f.update(kw)
        return dry.lib.qproj_kv_append(dry.ctx, ref(kv), f["k"], f["ks"], f["v"], f["vs"], f["n"], f["slots"], ref(rot), f["q"], f["qs"],
                                       f["h"], f["qo"], f["qos"])
    if name == "read":
        f = dict(slots=BUF, n=5, k=BUF, v=BUF)
        f.update(kw)
        return dry.lib.qproj_kv_read(dry.ctx, ref(kv), f["slots"], f["n"], f["k"], f["v"])
    f = dict(q=BUF, qs=4096, n=5, h=32, seqs=2, start=BUF, len=BUF, max_q=5, pages=BUF, ps=10, scale=0.1, window=0, y=2 * BUF, ys=4096)
    f.update(kw)
    return dry.lib.qproj_attention(dry.ctx, ref(kv), f["q"], f["qs"], f["n"], f["h"], f["seqs"], f["start"], f["len"], f["max_q"], f["pages"],
                                   f["ps"], f["scale"], f["window"], f["y"], f["ys"])


def test_calls_that_are_taken_note_their_launches():
    with Dry() as dry:
        assert call(dry, "rope", rot=rotation()) == 0
        assert call(dry, "append", cache(), rotation(mode=1, n_dims=64), q=BUF, qs=4096, h=32, qo=BUF, qos=4096) == 0
        assert call(dry, "append", cache(), None) == 0
        assert call(dry, "read", cache()) == 0 and call(dry, "read", cache(), k=None) == 0
        assert call(dry, "attention", cache()) == 0
        for page in (16, 32, 64, 128, 256):
            for dim in (64, 96, 128, 256):
                assert call(dry, "attention", cache(page_tokens=page, head_dim=dim), h=8, qs=8 * dim, ys=8 * dim, window=7) == 0, (page, dim)
        # nothing to do is no error and no launch
        assert call(dry, "rope", rot=rotation(), n=0) == 0 and call(dry, "append", cache(), None, n=0) == 0
        assert call(dry, "read", cache(), n=0) == 0 and call(dry, "read", cache(), k=None, v=None) == 0
        assert call(dry, "attention", cache(), n=0) == 0 and call(dry, "attention", cache(), seqs=0) == 0
    assert dry.plan.count("rope_kv_kernel:") == 3 and dry.plan.count("kv_read_kernel:") == 2 and dry.plan.count("attention_kernel<") == 21


def test_rows_are_taken_sixteen_or_32_at_a_time():
    """few rows of work: 16; many: 32, unless a head is 256 wide"""
    def plan(dim=128, **kw):
        with Dry() as dry:
            assert call(dry, "attention", cache(n_pages=1 << 16, head_dim=dim), qs=32 * dim, ys=32 * dim, **kw) == 0
        return dry.plan.split(":")[0]
    one, token = dict(seqs=1, n=8, max_q=8), dict(seqs=1, n=1, max_q=1)
    assert plan(ps=64, **one) == "attention_kernel<128, 1>" and plan(ps=2048, **one) == "attention_kernel<128, 2>"
    assert plan(ps=2048, **token) == "attention_kernel<128, 1>" and plan(ps=2048, window=1000, **one) == "attention_kernel<128, 1>"
    assert plan(seqs=1, n=4096, max_q=4096, ps=64) == "attention_kernel<128, 2>" and plan(dim=96, seqs=1, n=4096, max_q=4096, ps=64) == "attention_kernel<96, 2>"
    assert plan(dim=256, seqs=1, n=4096, max_q=4096, ps=64) == "attention_kernel<256, 1>"
    # a table that one of many sequences needs, and a max_q that one of them has
    assert plan(seqs=64, n=64 + 100, max_q=100, ps=4) == "attention_kernel<128, 1>"


def test_long_calls_become_launches_that_fit():
    with Dry() as dry:
        assert call(dry, "rope", rot=rotation(), n=(1 << 24) + 1) == 0
        assert call(dry, "read", cache(), n=(1 << 23) + 1) == 0
        # 64 sequences of 131072 tokens, one of them a prompt of 8192, and a token of a million
        assert call(dry, "attention", cache(n_pages=1 << 20), n=8192 + 63, seqs=64, max_q=8192, ps=2048) == 0
        assert call(dry, "attention", cache(n_pages=1 << 20), n=1, seqs=1, max_q=1, ps=1 << 14) == 0
    assert dry.plan.count("rope_kv_kernel: 8388608 tokens") == 2 and dry.plan.count("rope_kv_kernel: 1 tokens") == 1
    assert dry.plan.count("kv_read_kernel: 8388608 places") == 1 and dry.plan.count("kv_read_kernel: 1 places") == 1


ROPE_BAD = [dict(x=None), dict(y=None), dict(x=BUF + 4), dict(y=BUF + 8), dict(xs=4092), dict(xs=4098), dict(ys=100), dict(n=-1), dict(n=1 << 31),
            dict(h=0), dict(h=5000, xs=1 << 20, ys=1 << 20), dict(d=0), dict(d=100), dict(d=2048, xs=1 << 17, ys=1 << 17),
            dict(x=BUF, y=BUF, xs=4096, ys=8192)]
ROTATION_BAD = [dict(pos_dev=None), dict(freqs_dev=None), dict(n_dims=0), dict(n_dims=12), dict(n_dims=136), dict(n_dims=-8), dict(mode=2)]
CACHE_BAD = [dict(k_codes=None), dict(v_scales=None), dict(k_scales=BUF + 2), dict(v_codes=BUF + 8), dict(n_pages=0), dict(n_pages=1 << 31),
             dict(n_pages=1 << 23), dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=512), dict(page_tokens=0), dict(n_head_kv=0), dict(n_head_kv=-1),
             dict(head_dim=80), dict(head_dim=512), dict(head_dim=0)]
APPEND_BAD = [dict(k=None), dict(v=None), dict(slots=None), dict(k=BUF + 4), dict(ks=1020), dict(vs=1026), dict(n=-1),
              dict(q=BUF, qs=4096, h=32, qo=None, qos=4096), dict(q=BUF, qs=4000, h=32, qo=BUF, qos=4096), dict(q=BUF, qs=4096, h=0, qo=BUF, qos=4096),
              dict(q=BUF, qs=4096, h=32, qo=BUF, qos=8192)]
ATTENTION_BAD = [dict(q=None), dict(y=None), dict(start=None), dict(len=None), dict(pages=None), dict(q=BUF + 4), dict(y=BUF + 8), dict(qs=4092), dict(ys=4094),
                 dict(h=33), dict(h=0), dict(h=-8), dict(seqs=-1), dict(seqs=65537), dict(max_q=-1), dict(n=-1), dict(ps=-1), dict(ps=1 << 26), dict(window=-1),
                 dict(y=BUF), dict(n=1 << 30, max_q=1 << 30, seqs=1, ps=1 << 20), dict(n=1 << 20, max_q=1 << 20, seqs=65536)]


@pytest.mark.parametrize("name,bad", [("rope", b) for b in ROPE_BAD] + [("append", b) for b in APPEND_BAD] + [("attention", b) for b in ATTENTION_BAD] +
                         [("read", b) for b in (dict(slots=None), dict(n=-1), dict(k=BUF + 4), dict(v=BUF + 12))], ids=str)
def test_bad_arguments_are_refused(name, bad):
    with Dry() as dry:
        assert call(dry, name, cache(), rotation(), **bad) == 1
        assert dry.error().startswith("qproj_") and ":" in dry.error()
    assert "kernel" not in dry.plan


@pytest.mark.parametrize("bad", CACHE_BAD, ids=str)
def test_bad_caches_are_refused(bad):
    with Dry() as dry:
        for name in ("append", "read", "attention"):
            assert call(dry, name, cache(**bad), rotation()) == 1 and call(dry, name, None, rotation()) == 1
    assert "kernel" not in dry.plan


@pytest.mark.parametrize("bad", ROTATION_BAD, ids=str)
def test_bad_rotations_are_refused(bad):
    with Dry() as dry:
        for name in ("rope", "append"):
            assert call(dry, name, cache(), rotation(**bad)) == 1
        assert call(dry, "rope", rot=None) == 1
        assert call(dry, "append", cache(), None, q=BUF, qs=4096, h=32, qo=BUF, qos=4096) == 1     # queries want a rotation
    assert "kernel" not in dry.plan


def test_null_context():
    lib = qproj.load_library()
    assert lib.qproj_rope(None, None, None, 0, 0, 0, 0, None, 0) == 1
    assert lib.qproj_kv_append(None, None, None, 0, None, 0, 0, None, None, None, 0, 0, None, 0) == 1
    assert lib.qproj_kv_read(None, None, None, 0, None, None) == 1
    assert lib.qproj_attention(None, None, None, 0, 0, 0, 0, None, None, 0, None, 0, 1.0, 0, None, 0) == 1
    assert lib.qproj_rope_frequencies(None, 64, None, None) == 1
