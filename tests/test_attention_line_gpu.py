"""Attention where the grid has hardly more workgroups than the call has stretches of work, against plain statements in 64 bits (kv_ref.py): tables
of exactly the pages that are needed, few heads, lengths on both sides of what a turn takes."""
import numpy as np
import pytest
import torch

import kv_ref
from test_attention_gpu import check, dev, make_cache, numpy_cache, tell

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    """one context for all calls, one after the other"""
    from magnitude_amd import Context
    assert torch.cuda.is_available(), "these tests need the MI355X"
    c = Context(0)
    yield c
    c.close()


def exact_table(rng, lens, page, kv_heads, dim):
    kv, pages = make_cache(rng, lens, page, kv_heads, dim)
    return kv, np.ascontiguousarray(pages[:, :max(1, max(-(-n // page) for n in lens))])


@pytest.mark.parametrize("length", [257, 513, 1025, 1300, 1537, 2049, 2100, 9000])
@pytest.mark.parametrize("kv_heads,group,dim,page", [(1, 4, 128, 64), (2, 7, 64, 16), (3, 1, 96, 32), (4, 8, 128, 64), (5, 3, 256, 16), (1, 71, 128, 64)])
def test_a_token_in_a_table_of_its_pages(ctx, kv_heads, group, dim, page, length):
    tell("a token", kv_heads, group, dim, page, length)
    rng = np.random.default_rng(length + kv_heads)
    kv, pages = exact_table(rng, [length], page, kv_heads, dim)
    q = rng.standard_normal((1, kv_heads * group, dim)).astype(np.float32)
    check(ctx, kv, pages, q, [0, 1], [length], max_q=1)


@pytest.mark.parametrize("kv_heads,lens,new", [(1, [2100] * 2, 1), (1, [1100] * 3, 1), (2, [1300] * 3, 1), (1, [777] * 5, 1), (3, [1025, 900], 1), (1, [1500], 9),
                                               (2, [700, 650, 600], 4), (4, [1550], 1), (1, [1900], 27)])
def test_few_sequences_of_like_lengths(ctx, kv_heads, lens, new):
    tell("few sequences", kv_heads, lens, new)
    rng = np.random.default_rng(sum(lens) + kv_heads)
    kv, pages = exact_table(rng, lens, 64, kv_heads, 128)
    q_start = np.arange(len(lens) + 1) * new
    q = rng.standard_normal((q_start[-1], kv_heads * 4, 128)).astype(np.float32)
    check(ctx, kv, pages, q, q_start, lens, max_q=new)
    check(ctx, kv, pages, q, q_start, lens, window=500, max_q=new)


def test_two_contexts_at_once_have_the_right_results():
    from magnitude_amd import Context
    rng = np.random.default_rng(16)
    work = []
    for lens, kv_heads in (([9000], 1), ([3000, 10, 700, 2000], 8), ([1300], 2)):
        stream = torch.cuda.Stream()
        kv, pages = exact_table(rng, lens, 64, kv_heads, 128)
        q = rng.standard_normal((len(lens), 4 * kv_heads, 128)).astype(np.float32)
        start = np.arange(len(lens) + 1, dtype=np.int32)
        want, sizes = kv_ref.attention(numpy_cache(kv), q, start, lens, pages, 128 ** -0.5)
        args = kv, dev(q), dev(start), dev(np.array(lens, np.int32)), dev(pages)
        work.append((Context(0, stream=stream.cuda_stream), args, want, kv_ref.allowed(sizes, 128, max(lens)), [torch.zeros_like(args[1]) for _ in range(10)]))
    torch.cuda.synchronize()
    for i in range(10):
        for c, args, _, _, outs in work:
            c.attention(*args, max_q=1, out=outs[i], sync=False)
    for c, _, want, bound, outs in work:
        c.sync()
        for o in outs:
            assert (np.abs(o.cpu().numpy() - want) <= bound).all()
        c.close()


@pytest.mark.parametrize("window", [47, 48, 49, (1 << 31) - 1, 1 << 31, 1 << 62])
def test_windows_of_any_size(ctx, window):
    """as long as a sequence can be and longer, where rows stand before the first token"""
    tell("window", window)
    rng = np.random.default_rng(21)
    lens, q_start = [3, 0, 40, 48], [0, 8, 12, 13, 33]
    kv, pages = exact_table(rng, lens, 16, 2, 128)
    q = rng.standard_normal((33, 8, 128)).astype(np.float32)
    got = check(ctx, kv, pages, q, q_start, lens, window=window)
    assert not got[:5].any() and got[5:8].any() and not got[8:12].any() and got[12:].any()


def test_sequences_that_share_rows_are_reported(ctx):
    from magnitude_amd import QprojError
    rng = np.random.default_rng(22)
    lens = [700, 700, 300, 900]
    kv, pages = exact_table(rng, lens, 64, 2, 128)
    q = rng.standard_normal((9, 8, 128)).astype(np.float32)
    i32 = lambda a: dev(np.array(a, np.int32))
    out = torch.full(q.shape, 7.5, device="cuda")
    tell("q_start falls among others")
    with pytest.raises(QprojError, match="q_start or kv_len"):
        ctx.attention(kv, dev(q), i32([0, 3, 2, 5, 9]), i32(lens), dev(pages), out=out)
    got = out.cpu().numpy()
    for s, rows in ((0, [0, 1]), (2, [3, 4]), (3, [5, 6, 7, 8])):
        a, b = [0, 3, 2, 5, 9][s], [0, 3, 2, 5, 9][s + 1]
        want, sizes = kv_ref.attention(numpy_cache(kv), q[a:b], [0, b - a], lens[s:s + 1], pages[s:s + 1], 128 ** -0.5)
        bound = kv_ref.allowed(sizes, 128, lens[s])
        assert (np.abs(got[rows] - want[[r - a for r in rows]]) <= bound[[r - a for r in rows]]).all()
    # so many shared rows behind so many tokens that 32 bits do not count them: nothing is done
    tell("q_start falls again and again")
    kv, _ = make_cache(rng, [256], 256, 8, 128)
    q = torch.zeros((100, 32, 128), device="cuda")
    out = torch.full(q.shape, 7.5, device="cuda")
    with pytest.raises(QprojError, match="q_start or kv_len"):
        ctx.attention(kv, q, i32([100 * (i % 2) for i in range(42)]), i32([1 << 28] * 41), torch.zeros((41, 1 << 20), dtype=torch.int32, device="cuda"), out=out)
    assert (out == 7.5).all()
    ctx.sync()


def test_rows_of_a_call_that_is_left_out_are_not_joined(ctx):
    """items cut into many parts, then a call with the same places whose sequences share too many rows: what was joined before is not again"""
    from magnitude_amd import QprojError
    rng = np.random.default_rng(25)
    lens = [9000, 9000, 9000]
    kv, pages = exact_table(rng, lens, 64, 1, 128)
    q = rng.standard_normal((40, 4, 128)).astype(np.float32)
    check(ctx, kv, pages, q, [0, 1, 2, 40], lens, max_q=40)
    out = torch.full(q.shape, 7.5, device="cuda")
    with pytest.raises(QprojError, match="q_start or kv_len"):
        ctx.attention(kv, dev(q), dev(np.array([0, 40, 0, 40], np.int32)), dev(np.array(lens, np.int32)), dev(pages), max_q=40, out=out)
    assert (out == 7.5).all()


def test_more_rows_than_none_are_reported(ctx):
    from magnitude_amd import QprojError
    kv, pages = make_cache(np.random.default_rng(23), [100, 60], 16, 1, 64)
    q, out = torch.zeros((5, 4, 64), device="cuda"), torch.full((5, 4, 64), 7.5, device="cuda")
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    ctx.attention(kv, q, i32(0, 0, 0), i32(100, 60), dev(pages), max_q=0, out=out)
    with pytest.raises(QprojError, match="q_start or kv_len"):
        ctx.attention(kv, q, i32(0, 0, 2), i32(100, 60), dev(pages), max_q=0, out=out)
    assert (out == 7.5).all()


def test_everything_that_went_wrong_since_the_last_time_is_named(ctx):
    from magnitude_amd import QprojError
    kv, pages = make_cache(np.random.default_rng(24), [100, 60], 16, 1, 64)
    x, q, out = torch.zeros((1, 1, 64), device="cuda"), torch.zeros((5, 4, 64), device="cuda"), torch.zeros((5, 4, 64), device="cuda")
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    slots, start, lens, wrong, table = torch.tensor([1 << 40], device="cuda"), i32(0, 3, 5), i32(100, 60), i32(100, -1), dev(pages)
    bad = dev(np.full_like(pages, kv.n_pages))
    torch.cuda.synchronize()
    ctx.kv_append(kv, x, x, slots, sync=False)
    ctx.attention(kv, q, start, wrong, table, out=out, sync=False)
    with pytest.raises(QprojError, match="slot.*; q_start or kv_len"):
        ctx.sync()
    ctx.sync()
    ctx.attention(kv, q, start, wrong, table, out=out, sync=False)
    ctx.attention(kv, q, start, lens, bad, out=out, sync=False)
    ctx.kv_append(kv, x, x, slots, sync=False)
    with pytest.raises(QprojError, match="slot.*; a page.*; q_start or kv_len"):
        ctx.sync()
    ctx.sync()


def set_counts(c, words):
    """the counts of parts in a context's workspace, as a call that went wrong could have left them"""
    import ctypes as C
    f = c.lib.qproj_internal_attention_counts
    f.restype, f.argtypes = C.c_int, [C.c_void_p, C.c_void_p, C.c_int64]
    words = np.ascontiguousarray(words, np.uint64)
    assert f(c.handle, words.ctypes.data, len(words)) == 0


@pytest.mark.parametrize("kv_heads,lens,new", [(8, [500], 1), (2, [1300], 1), (4, [900, 2100, 333], 1), (1, [1500] * 24, 1), (2, [1200, 900], 8), (8, [700], 100)])
def test_what_counts_of_parts_an_earlier_call_left_behind_is_nothing(kv_heads, lens, new):
    from magnitude_amd import Context
    tell("counts", kv_heads, lens, new)
    rng = np.random.default_rng(sum(lens) + kv_heads)
    kv, pages = exact_table(rng, lens, 64, kv_heads, 128)
    q_start = np.arange(len(lens) + 1, dtype=np.int32) * new
    q = rng.standard_normal((q_start[-1], 4 * kv_heads, 128)).astype(np.float32)
    want, sizes = kv_ref.attention(numpy_cache(kv), q, q_start, lens, pages, 128 ** -0.5)
    bound = kv_ref.allowed(sizes, 128, max(lens))
    stream = torch.cuda.Stream()
    c = Context(0, stream=stream.cuda_stream)
    args = kv, dev(q), dev(q_start), dev(np.array(lens, np.int32)), dev(pages)
    y = torch.full(q.shape, 7.5, device="cuda")
    torch.cuda.synchronize()

    def right(what):
        c.sync()
        assert (np.abs(y.cpu().numpy() - want) <= bound).all(), what
        y.fill_(7.5)
        torch.cuda.synchronize()

    c.attention(*args, max_q=new, out=y, sync=False)
    right("the first call")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        c.attention(*args, max_q=new, out=y, sync=False)
    number = 0x9e3779b9 + 1        # of the next call.  (Its own number with a count is what only the call itself can have written.)
    for kind in ("zeros", "ones", "random", "the call before, a count that carries into this one's number", "the call to come", "the call before"):
        for how in ("an eager call", "a replay"):
            if kind == "random":
                words = rng.integers(0, 1 << 63, 999, dtype=np.uint64)
            else:
                words = [{"zeros": 0, "ones": (1 << 64) - 1}.get(kind, (number + (1 if "come" in kind else -1) << 32) + (0xffffffff if "carries" in kind else 3))]
            set_counts(c, words)
            if how == "a replay":
                with torch.cuda.stream(stream):
                    graph.replay()
            else:
                c.attention(*args, max_q=new, out=y, sync=False)
            right((kind, how))
            c.attention(*args, max_q=new, out=y, sync=False)
            right((kind, "the call after " + how))
            number += 2
    c.close()


def test_grids_of_many_sizes_in_one_context():
    """a call advances the words of the workgroups that it does not have, too"""
    from magnitude_amd import Context
    rng = np.random.default_rng(30)
    c = Context(0)
    work = []
    for kv_heads, lens, new in ((8, [500], 1), (1, [1500] * 24, 1), (2, [1300], 1), (1, [70], 1), (4, [3000] * 9, 1), (1, [9000], 1), (8, [300], 64)):
        kv, pages = exact_table(rng, lens, 64, kv_heads, 64)
        q_start = np.arange(len(lens) + 1, dtype=np.int32) * new
        q = rng.standard_normal((q_start[-1], 2 * kv_heads, 64)).astype(np.float32)
        want, sizes = kv_ref.attention(numpy_cache(kv), q, q_start, lens, pages, 64 ** -0.5)
        work.append(((kv, dev(q), dev(q_start), dev(np.array(lens, np.int32)), dev(pages)), new, want, kv_ref.allowed(sizes, 64, max(lens))))
    for i in rng.integers(0, len(work), 80):
        args, new, want, bound = work[i]
        got = c.attention(*args, max_q=new)
        assert (np.abs(got.cpu().numpy() - want) <= bound).all(), i
    c.close()


def test_calls_behind_each_other_of_many_grids():
    """no wait between them: each finds the words of counts and the calls' number as the one before left them, eager or replayed"""
    from magnitude_amd import Context
    rng = np.random.default_rng(31)
    stream = torch.cuda.Stream()
    c = Context(0, stream=stream.cuda_stream)
    work = []
    for kv_heads, lens, new in ((8, [500], 1), (1, [1500] * 24, 1), (2, [1300], 1), (1, [70], 1), (4, [3000] * 9, 1), (1, [9000], 1), (8, [300], 64)):
        kv, pages = exact_table(rng, lens, 64, kv_heads, 128)
        q_start = np.arange(len(lens) + 1, dtype=np.int32) * new
        q = rng.standard_normal((q_start[-1], 4 * kv_heads, 128)).astype(np.float32)
        want, sizes = kv_ref.attention(numpy_cache(kv), q, q_start, lens, pages, 128 ** -0.5)
        work.append(((kv, dev(q), dev(q_start), dev(np.array(lens, np.int32)), dev(pages)), new, want, kv_ref.allowed(sizes, 128, max(lens))))
    order = rng.integers(0, len(work), 120)
    outs = [torch.full(work[i][2].shape, 7.5, dtype=torch.float32, device="cuda") for i in order]
    torch.cuda.synchronize()

    def all_right(what):
        c.sync()
        for n, (i, out) in enumerate(zip(order, outs)):
            assert (np.abs(out.cpu().numpy() - work[i][2]) <= work[i][3]).all(), (what, n, i)
            out.fill_(7.5)
        torch.cuda.synchronize()

    def calls():
        for i, out in zip(order, outs):
            c.attention(*work[i][0], max_q=work[i][1], out=out, sync=False)

    calls()
    all_right("eager")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        calls()
    for n in range(3):
        with torch.cuda.stream(stream):
            graph.replay()
        all_right(f"replay {n}")
        calls()
        all_right("eager again")
    c.close()
