"""Attention over shared prefixes as it is called without sizes: what is shared is shared."""
import re

import numpy as np
import pytest
import torch

import forms_ref
from test_attention_cpu import Dry, cache
from test_attention_forms_gpu import ctx, i32, share  # noqa: F401  (ctx: the fixture)
from test_attention_forms_cpu import call
from test_attention_gpu import dev, make_cache, numpy_cache

pytestmark = pytest.mark.gpu


class Spy:
    """A library whose calls' arguments are kept"""

    def __init__(self, lib):
        self.lib, self.seen = lib, []

    def __getattr__(self, name):
        f = getattr(self.lib, name)

        def call(*args):
            self.seen.append((name, args))
            return f(*args)
        return call if name == "qproj_attention_shared" else f


def launched(max_q, n, seqs, heads, kv_heads, dim, page, columns):
    """the kernel that a call with such sizes launches"""
    with Dry() as dry:
        assert call(dry, "shared", cache(page_tokens=page, n_head_kv=kv_heads, head_dim=dim), h=heads, qs=heads * dim, ys=heads * dim, n=n, seqs=seqs, max_q=max_q, ps=columns,
                    max_group=seqs) == 0
    return re.search(r"attention_kernel<[^>]*>", dry.plan).group()


@pytest.mark.parametrize("rows", [[1] * 48, [1, 2, 0, 4, 3], [0, 0], [1, 5, 40]])
def test_the_most_rows_are_read_from_q_start(ctx, rows, monkeypatch):
    rng = np.random.default_rng(81)
    page, heads, kv_heads, dim = 64, 8, 2, 128
    lens = [512 + 20 * i % 90 + r for i, r in enumerate(rows)]
    kv, pages = make_cache(rng, lens, page, kv_heads, dim)
    pages, group_start, shared = share(np.pad(pages, ((0, 1), (0, 0))), lens + [0], [(512, len(rows))], page)
    pages, q_start = pages[:-1], np.cumsum([0] + rows)
    q = rng.standard_normal((q_start[-1] + 2, heads, dim)).astype(np.float32)      # two rows of no sequence
    args = kv, dev(q), i32(q_start), i32(lens), dev(pages), i32(group_start), i32(shared)
    spy = Spy(ctx.lib)
    monkeypatch.setattr(ctx, "lib", spy)
    out = torch.full(q.shape, 7.5, device="cuda")
    got = ctx.attention_shared(*args, out=out).cpu().numpy()
    max_q, max_group = spy.seen[0][1][9], spy.seen[0][1][15]
    assert (max_q, max_group) == (max(rows), len(rows))
    kernel = launched(max_q, len(q), len(rows), heads, kv_heads, dim, page, pages.shape[1])
    assert (", prefix>" in kernel) == (0 < max(rows) <= 4)
    want, sizes = forms_ref.attention(numpy_cache(kv), q, q_start, lens, pages, dim ** -0.5)
    mine = ~np.isnan(want).all(-1)
    assert (got[~mine] == 7.5).all() and (np.abs(got - want)[mine] <= forms_ref.allowed(sizes, dim, max(lens))[mine]).all()
    assert np.array_equal(got[:-2], ctx.attention_shared(*args, max_q=max(rows), out=torch.full(q.shape, 7.5, device="cuda"))[:-2].cpu().numpy())


def test_bounds_that_do_not_hold_are_still_reported(ctx):
    from magnitude_amd import QprojError
    rng = np.random.default_rng(82)
    kv, pages = make_cache(rng, [100, 90], 16, 1, 64)
    q = dev(rng.standard_normal((2, 4, 64)).astype(np.float32))
    for q_start in ([0, 1, 3], [0, 2, 1], [5, 2, 1], [-1, 0, 1], [-2147483648, 2147483647, 2], [2147483647, -2147483648, 2]):
        with pytest.raises(QprojError, match="q_start"):
            ctx.attention_shared(kv, q, i32(q_start), i32([100, 90]), dev(pages), i32([0, 2]), i32([64]))
    ctx.sync()
    assert ctx.attention_shared(kv, q, i32([0]), i32([]), dev(pages[:0]), i32([0]), i32([])).shape == q.shape
