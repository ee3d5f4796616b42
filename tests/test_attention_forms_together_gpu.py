"""The forms of attention over the 4-bit cache as they are used: layers of an encoder and a decoder, sequences branching from one prompt,
captured steps, contexts side by side, large caches, calls with nothing to do and calls that are refused."""
import numpy as np
import pytest
import torch

from test_attention_forms_gpu import check_biased, check_cross, check_shared, ctx, i32, make_bias, share  # noqa: F401  (ctx: the fixture)
from test_attention_gpu import check, dev, make_cache, tell

pytestmark = pytest.mark.gpu


def test_an_encoder_and_a_decoder(ctx):
    """projections without a rotation into the cache, an encoder's rows with a bias on both sides, their states' keys and values kept for cross
    attention, a decoder's prompt and tokens with a bias on one side and over the states"""
    from magnitude_amd import ACT_F32, TYPE_Q4_K, KvCache, relative_buckets, synth
    heads, dim, d, page, n_buckets, reach = 8, 64, 512, 32, 32, 128
    weights = [ctx.upload_from_device(TYPE_Q4_K, d, d, synth.random_weight(TYPE_Q4_K, d, d, seed=60 + i, device="cuda")) for i in range(10)]
    rng = np.random.default_rng(51)
    tables = [dev(rng.standard_normal((n_buckets, heads)).astype(np.float32)) for _ in "ed"]
    bias = [ctx.bias_by_distance(t, dev(relative_buckets(n_buckets, reach, both))) for t, both in zip(tables, (True, False))]
    lens = [210, 37, 90]
    start = np.cumsum([0] + lens)
    pages = np.full((3, 8), -1, np.int32)
    at = iter(rng.permutation(12))
    for s, n in enumerate(lens):
        pages[s, :-(-n // page)] = [next(at) for _ in range(-(-n // page))]
    slots = dev(np.concatenate([pages[s, np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page for s, n in enumerate(lens)]))
    rows = lambda t: t.unflatten(1, (heads, dim))

    x = dev(rng.standard_normal((sum(lens), d)).astype(np.float32))
    q, k, v = ctx.mul_mat_multi(weights[:3], x, ACT_F32)
    encoder = KvCache.zeros(12, page, heads, dim)
    ctx.kv_append(encoder, rows(k), rows(v), slots)
    got = check_biased(ctx, encoder, pages, rows(q).cpu().numpy(), start, lens, bias[0].cpu().numpy(), False, scale=1.0 / 16, max_q=max(lens))
    states = x + ctx.mul_mat(weights[3], dev(got).flatten(1), ACT_F32)
    k, v = ctx.mul_mat_multi(weights[4:6], states, ACT_F32)
    cross = KvCache.zeros(12, page, heads, dim)
    ctx.kv_append(cross, rows(k), rows(v), slots)

    own = KvCache.zeros(6, page, heads, dim)
    own_pages, have = np.array([[3, 1], [0, 5], [4, 2]], np.int32), np.zeros(3, np.int64)
    for new in ([5, 1, 30], [1, 1, 1], [1, 0, 2], [1, 1, 1]):
        q_start = np.cumsum([0] + new)
        y = dev(rng.standard_normal((sum(new), d)).astype(np.float32))
        q, k, v = ctx.mul_mat_multi(weights[6:9], y, ACT_F32)
        t = [have[s] + np.arange(n) for s, n in enumerate(new)]
        ctx.kv_append(own, rows(k), rows(v), dev(np.concatenate([own_pages[s, u // page].astype(np.int64) * page + u % page for s, u in enumerate(t)])))
        have += new
        got = check_biased(ctx, own, own_pages, rows(q).cpu().numpy(), q_start, have.tolist(), bias[1].cpu().numpy(), True, scale=1.0 / 16, max_q=max(new))
        y = y + dev(got).flatten(1)
        got = check_cross(ctx, cross, pages, rows(ctx.mul_mat(weights[9], y, ACT_F32)).cpu().numpy(), q_start, lens, max_q=max(new))
        assert got.any(-1).all()


def test_sequences_that_branch_from_one_prompt(ctx):
    """a prompt computed once, its whole pages given to five answers, the rest of it copied to a page of each; answers token by token, one of them
    with drafts; beside them a request of its own"""
    from magnitude_amd import KvCache, rope_frequencies
    heads, kv_heads, dim, page, prompt = 8, 2, 128, 16, 200
    rng = np.random.default_rng(52)
    freqs = dev(rope_frequencies(dim)[0])
    kv = KvCache.zeros(60, page, kv_heads, dim)
    order = rng.permutation(60)
    rows = lambda n, h: dev(rng.standard_normal((n, h, dim)).astype(np.float32))

    def append(t, pages, n):
        """rows of tokens t (a list a sequence) -> queries"""
        slots = np.concatenate([p[u // page].astype(np.int64) * page + u % page for p, u in zip(pages, t)])
        return ctx.kv_append(kv, rows(n, kv_heads), rows(n, kv_heads), dev(slots), pos=i32(np.concatenate(t)), freqs=freqs, mode="halves", q=rows(n, heads))

    first = order[:13].astype(np.int32)
    q = append([np.arange(prompt)], [first], prompt)
    check(ctx, kv, first[None], q.cpu().numpy(), [0, prompt], [prompt], max_q=prompt)
    whole = prompt // page
    pages = np.full((6, 20), -1, np.int32)
    pages[:5, :whole] = first[:whole]
    pages[:5, whole: whole + 3] = order[13:28].reshape(5, 3)
    pages[5, :4] = order[28:32]
    for s in range(5):                       # the prompt's tokens on the last, part page
        for t in kv.tensors:
            t[int(pages[s, whole])] = t[int(first[whole])]
    have = np.array([prompt] * 5 + [0])
    for step in range(8):
        new = np.array([1, 1, 1, 1 + step % 4, 1, 40 if step == 0 else 1]) if step else np.array([1, 1, 1, 1, 1, 40])
        t = [have[s] + np.arange(n) for s, n in enumerate(new)]
        q = append(t, pages, int(new.sum()))
        have = have + new
        check_shared(ctx, kv, pages, q.cpu().numpy(), np.cumsum([0] + new.tolist()), have.tolist(), [0, 5, 6], [whole * page, 0], max_q=int(new.max()), max_group=5)


# ---- calls of every form, alike -------------------------------------------------------------------------------------------
class Case:
    """A call with lengths that may change, rows of one token"""

    def __init__(self, form, rng, lens, kv_heads=2, group=4, dim=128, page=64):
        self.form, self.lens0 = form, list(lens)
        self.kv, pages = make_cache(rng, lens, page, kv_heads, dim)
        n = len(lens)
        half = n // 2
        self.shared0 = min(lens[:half + n % 2]) // page * page
        if form == "shared":
            pages = share(pages, lens, [(self.shared0, half + n % 2), (0, half)], page)[0]
        self.pages_host, self.q_host = pages, rng.standard_normal((n, kv_heads * group, dim)).astype(np.float32)
        self.q, self.pages, self.start, self.lens = dev(self.q_host), dev(pages), i32(np.arange(n + 1)), i32(lens)
        self.groups, self.shared = i32([0, half + n % 2, n]), i32([self.shared0, 0])
        self.bias_host = make_bias(rng, kv_heads * group, 40)[0]
        self.bias = dev(self.bias_host)

    def __call__(self, c, out=None, sync=True):
        args = self.kv, self.q, self.start, self.lens, self.pages
        if self.form == "cross":
            return c.cross_attention(*args, max_q=1, out=out, sync=sync)
        if self.form == "shared":
            return c.attention_shared(*args, self.groups, self.shared, max_q=1, max_group=(len(self.lens0) + 1) // 2, out=out, sync=sync)
        return c.attention_biased(*args, self.bias, causal=self.form == "causal", max_q=1, out=out, sync=sync)

    def check(self, c, lens, groups, shared):
        args = c, self.kv, self.pages_host, self.q_host, np.arange(len(lens) + 1), [int(n) for n in lens]
        if self.form == "cross":
            return check_cross(*args, max_q=1)
        if self.form == "shared":
            return check_shared(*args, groups, shared, max_q=1)
        return check_biased(*args, self.bias_host, self.form == "causal", max_q=1)


FORMS = ["cross", "shared", "causal", "both"]      # (the last two: with a bias)


@pytest.mark.parametrize("seqs,kv_heads,group", [(2, 1, 4), (2, 1, 16), (24, 2, 4)])
@pytest.mark.parametrize("form", FORMS)
def test_captured_calls_follow_the_lengths(form, seqs, kv_heads, group):
    """recorded once, replayed with lengths from nothing to full pages, groups cut elsewhere, the context's own eager calls between"""
    from magnitude_amd import Context
    tell("captured", form, seqs, kv_heads, group)
    stream = torch.cuda.Stream()
    own, other = Context(0, stream=stream.cuda_stream), Context(0)
    rng = np.random.default_rng(53)
    most = 5000
    case = Case(form, rng, [most] * seqs, kv_heads, group, page=256)
    y = torch.zeros_like(case.q)
    torch.cuda.synchronize()
    case(own, out=y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        case(own, out=y, sync=False)
    half = (seqs + 1) // 2
    for i in range(12):
        n = rng.integers(0, most + 1, seqs) if i % 3 else np.full(seqs, (0, 1, most, 300)[i // 3])
        cut, shared = int(rng.integers(seqs - half, half + 1)), [int(rng.integers(0, case.shared0 + 1)), 0]
        with torch.cuda.stream(stream):
            case.lens.copy_(i32(n))
            case.groups.copy_(i32([0, cut, seqs]))
            case.shared.copy_(i32(shared))
            y.fill_(7.5)
            graph.replay()
        stream.synchronize()
        assert torch.equal(y, case(other)), f"replay {i}"
        if i % 2:
            case(own)
        if i in (4, 6):
            case.check(other, n, [0, cut, seqs], shared)
    own.close()
    other.close()


@pytest.mark.parametrize("form", FORMS)
def test_the_first_call_of_a_context_is_not_captured(form):
    from magnitude_amd import Context, QprojError
    stream = torch.cuda.Stream()
    own = Context(0, stream=stream.cuda_stream)
    case = Case(form, np.random.default_rng(54), [100, 70])
    y, spare = torch.zeros_like(case.q), torch.zeros(5, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        spare.add_(1)
        with pytest.raises(QprojError, match="captured"):
            case(own, out=y, sync=False)
    graph.replay()
    torch.cuda.synchronize()
    assert (spare == 1).all()
    want = case(own).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        case(own, out=y, sync=False)
    for _ in range(3):
        y.fill_(7.5)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    own.close()


def test_a_table_of_biases_laid_out_in_a_graph(ctx):
    """the table changes between replays (a program that swaps its weights), with the attention that reads it behind"""
    from magnitude_amd import Context, relative_buckets
    stream = torch.cuda.Stream()
    own = Context(0, stream=stream.cuda_stream)
    rng = np.random.default_rng(55)
    case = Case("both", rng, [900, 33, 150])
    buckets, table = dev(relative_buckets(16, 40, True)), torch.zeros((16, 8), device="cuda")
    y, by_distance = torch.zeros_like(case.q), torch.zeros_like(case.bias)
    case.bias = by_distance
    torch.cuda.synchronize()
    case(own, out=y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        own.bias_by_distance(table, buckets, out=by_distance, sync=False)
        case(own, out=y, sync=False)
    for i in range(4):
        new = (rng.standard_normal((16, 8)) * i).astype(np.float32)
        with torch.cuda.stream(stream):
            table.copy_(dev(new))
            graph.replay()
        stream.synchronize()
        case.bias_host = np.ascontiguousarray(new[buckets.cpu().numpy()].T)
        assert np.array_equal(by_distance.cpu().numpy(), case.bias_host)
        assert torch.equal(y, case(ctx))
        case.check(ctx, [900, 33, 150], None, None)
    own.close()


@pytest.mark.parametrize("form", ["cross", "causal", "both"])
def test_a_captured_encoder_follows_the_lengths(ctx, form):
    """many rows of short sequences, recorded once, replayed with other sequences' lengths and rows, some of none, eager work between"""
    from magnitude_amd import Context, QprojError
    tell("captured encoder", form)
    stream = torch.cuda.Stream()
    own = Context(0, stream=stream.cuda_stream)
    rng = np.random.default_rng(62)
    seqs, heads, most, rows = 8, 64, 180, 600
    kv, pages = make_cache(rng, [most] * seqs, 64, heads, 64)
    q_host, bias_host = rng.standard_normal((rows, heads, 64)).astype(np.float32), make_bias(rng, heads, 100)[0]
    q, bias, table, y = dev(q_host), dev(bias_host), dev(pages), torch.zeros((rows, heads, 64), device="cuda")
    start, lens = i32(np.arange(seqs + 1) * 75), i32([75] * seqs)

    def step(c, out):
        if form == "cross":
            return c.cross_attention(kv, q, start, lens, table, max_q=300, out=out, sync=False)
        return c.attention_biased(kv, q, start, lens, table, bias, causal=form == "causal", max_q=300, out=out, sync=False)

    torch.cuda.synchronize()
    step(own, y)
    own.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(own, y)
    for i in range(6):
        count = [[75] * 8, [300, 0, 1, 299, 0, 0, 0, 0], [128, 129, 31, 32, 33, 96, 97, 54], [0] * 8, [1] * 8, [64, 128, 200, 100, 7, 1, 0, 100]][i]
        n = [most, 0, 1, 64, 65, 128, 33, most] if i % 2 else rng.integers(0, most + 1, seqs)
        with torch.cuda.stream(stream):
            start.copy_(i32(np.cumsum([0] + count)))
            lens.copy_(i32(n))
            y.fill_(7.5)
            graph.replay()
        stream.synchronize()
        other = torch.full_like(y, 7.5)
        torch.cuda.synchronize()
        step(ctx, other)
        ctx.sync()
        assert torch.equal(y, other), f"replay {i}"
        args = ctx, kv, pages, q_host, np.cumsum([0] + count), [int(v) for v in n]
        got = check_cross(*args, max_q=300) if form == "cross" else check_biased(*args, bias_host, form == "causal", max_q=300)
        assert np.abs(got[:sum(count)] - y.cpu().numpy()[:sum(count)]).max(initial=0) < 1e-5
        if i % 2:
            step(own, other)
    ok = y.clone()
    for bad_start, bad_len, what, left in (([64, 128, 200, 100, 7, 1, 0, 101], 33, "q_start", 500), ([64, 128, 200, 100, 7, 1, 0, 100], -1, "q_start", 500)):
        start.copy_(i32(np.cumsum([0] + bad_start)))
        lens[7] = bad_len
        y.fill_(7.5)
        torch.cuda.synchronize()
        step(ctx, y)
        with pytest.raises(QprojError, match=what):
            ctx.sync()
        assert torch.equal(y[:left], ok[:left]) and (y[left:] == 7.5).all()
    own.close()


def test_contexts_of_all_forms_at_once():
    """calls on streams of their own, cut into few parts and into many, do not meet"""
    from magnitude_amd import Context
    rng = np.random.default_rng(56)
    work = []
    for i, form in enumerate(FORMS):
        stream = torch.cuda.Stream()
        case = Case(form, rng, ([9000, 8000], [3000, 10, 700, 2000])[i % 2], (1, 8)[i % 2])
        c = Context(0, stream=stream.cuda_stream)
        torch.cuda.synchronize()
        work.append((c, case, case(c).clone(), [torch.zeros_like(case.q) for _ in range(20)]))
    torch.cuda.synchronize()
    for i in range(20):
        for c, case, _, outs in work:
            case(c, out=outs[i], sync=False)
    for c, _, want, outs in work:
        c.sync()
        assert all(torch.equal(o, want) for o in outs)
        c.close()


def test_the_forms_of_one_context_one_after_the_other():
    """one workspace for all of them: queued without a wait, each as it is alone"""
    from magnitude_amd import Context
    rng = np.random.default_rng(57)
    c = Context(0, stream=torch.cuda.Stream().cuda_stream)
    cases = [Case(form, rng, lens, heads) for form in FORMS for lens, heads in (([9000, 8000], 1), ([300, 10, 70, 200], 8))]
    torch.cuda.synchronize()
    want = [case(c).clone() for case in cases]
    outs = [[torch.zeros_like(case.q) for case in cases] for _ in range(5)]
    torch.cuda.synchronize()
    for turn in outs:
        for case, out in zip(cases, turn):
            case(c, out=out, sync=False)
    c.sync()
    assert all(torch.equal(w, o) for turn in outs for w, o in zip(want, turn))
    c.close()


def test_a_cache_beyond_32_bits(ctx):
    """planes of more than 4 GiB, pages near their end; forms against the same tokens in a small cache"""
    from magnitude_amd import KvCache
    page, heads, dim = 256, 8, 128
    n_pages = (1 << 32) // (heads * page * dim // 2) + 40
    tell("forms on a cache beyond 32 bits:", n_pages, "pages")
    codes = [torch.empty((n_pages, heads, page, dim // 2), dtype=torch.uint8, device="cuda") for _ in "kv"]
    scales = [torch.empty((n_pages, heads, page, dim // 32), dtype=torch.float16, device="cuda") for _ in "kv"]
    case = Case("shared", np.random.default_rng(58), [600, 560, 530, 300], heads, 4, dim, page)
    where = dev(np.concatenate([[n_pages - 1, 0], np.arange(n_pages - 1 - case.kv.n_pages + 2, n_pages - 1)]).astype(np.int64))
    small = case.kv
    for big, t in zip((codes[0], scales[0], codes[1], scales[1]), small.tensors):
        big[where] = t
    case.check(ctx, case.lens0, [0, 2, 4], [512, 0])
    large = KvCache(codes[0], scales[0], codes[1], scales[1])
    for form in FORMS:
        case.form, case.kv, case.pages = form, small, dev(case.pages_host)
        want = case(ctx)
        case.kv, case.pages = large, torch.where(case.pages >= 0, where[case.pages.clamp(min=0).long()].int(), case.pages)
        assert torch.equal(case(ctx), want), form


def test_thousands_of_sequences(ctx):
    """more than workgroups: groups of two and of many, short; against the causal kernel, and a bias of nothing"""
    rng = np.random.default_rng(59)
    n, page = 6000, 16
    kv, pages = make_cache(rng, [40] * 200, page, 1, 64)
    table = np.ascontiguousarray(pages[rng.integers(0, 200, n)])
    table[:, 0] = np.repeat(table[::2, 0], 2)              # pairs share their first page
    lens = rng.integers(17, 41, n)
    q = dev(rng.standard_normal((n, 4, 64)).astype(np.float32))
    args = kv, q, i32(np.arange(n + 1)), i32(lens), dev(table)
    want = ctx.attention(*args, max_q=1)
    for groups, most in ((np.arange(0, n + 1, 2), 2), (np.r_[np.arange(0, 4000, 2), 4000 + np.arange(2001)], 2), (np.arange(n + 1), 5)):
        got = ctx.attention_shared(*args, i32(groups), i32(np.full(len(groups) - 1, 16)), max_q=1, max_group=most)
        assert (got - want).abs().max() < 1e-5
    everything = ctx.cross_attention(*args, max_q=1)
    assert (everything - want).abs().max() < 1e-5          # (rows of one token see all there is)
    none = torch.zeros((4, 7), device="cuda")
    assert (ctx.attention_biased(*args, none, max_q=1) - want).abs().max() < 1e-5


def test_nothing_to_do(ctx):
    case = Case("shared", np.random.default_rng(60), [30, 20], page=16)
    kv, pages, bias = case.kv, case.pages, case.bias
    none = torch.zeros((0, 8, 128), device="cuda")
    calls = {"cross": lambda q, s, n, p, y=None: ctx.cross_attention(kv, q, s, n, p, out=y),
             "shared": lambda q, s, n, p, y=None: ctx.attention_shared(kv, q, s, n, p, i32([0, len(n)] if len(n) else [0]), i32([16] if len(n) else []), out=y),
             "causal": lambda q, s, n, p, y=None: ctx.attention_biased(kv, q, s, n, p, bias, out=y),
             "both": lambda q, s, n, p, y=None: ctx.attention_biased(kv, q, s, n, p, bias, causal=False, out=y)}
    for form, call in calls.items():
        tell("nothing to do:", form)
        assert call(none, i32([0, 0, 0]), i32([30, 20]), pages).shape == (0, 8, 128)
        y = torch.full((3, 8, 128), 7.5, device="cuda")
        q = torch.ones_like(y)
        call(q, i32([0]), i32([]), pages[:0], y)                                 # no sequence
        assert (y == 7.5).all()
        call(q, i32([0, 0, 0]), i32([30, 20]), pages, y)                         # sequences without rows
        assert (y == 7.5).all()
        call(q, i32([0, 2, 3]), i32([0, 0]), pages[:, :0].contiguous(), y)       # no page, no token: rows of zeros
        assert not y.any()


def test_calls_that_do_not_fit_their_tensors_are_refused(ctx):
    from magnitude_amd import QprojError, relative_buckets
    case = Case("shared", np.random.default_rng(61), [100, 90])
    kv, q, start, lens, pages, groups, shared, bias = case.kv, case.q, case.start, case.lens, case.pages, case.groups, case.shared, case.bias
    args = kv, q, start, lens, pages
    table, buckets = torch.randn((16, 8), device="cuda"), dev(relative_buckets(16, 40))
    bad = [lambda: ctx.cross_attention(kv, q.double(), start, lens, pages), lambda: ctx.cross_attention(kv, q, start[:2], lens, pages),
           lambda: ctx.cross_attention(kv, q, start, lens.long(), pages), lambda: ctx.cross_attention(*args, out=q[:1]), lambda: ctx.cross_attention(kv, q.cpu(), start, lens, pages),
           lambda: ctx.cross_attention(kv, q[..., :64], start, lens, pages), lambda: ctx.cross_attention(kv, q, start, lens, pages[0]),
           lambda: ctx.attention_shared(*args, groups[:2], shared), lambda: ctx.attention_shared(*args, groups.long(), shared), lambda: ctx.attention_shared(*args, groups, shared.float()),
           lambda: ctx.attention_shared(*args, groups.cpu(), shared), lambda: ctx.attention_shared(*args, groups, shared, out=q[:1]),
           lambda: ctx.attention_biased(*args, bias[:7]), lambda: ctx.attention_biased(*args, bias[:, :80]), lambda: ctx.attention_biased(*args, bias[0]),
           lambda: ctx.attention_biased(*args, bias.double()), lambda: ctx.attention_biased(*args, bias.cpu()), lambda: ctx.attention_biased(*args, bias[:, 1:80]),
           lambda: ctx.bias_by_distance(table[0], buckets), lambda: ctx.bias_by_distance(table, buckets[:80]), lambda: ctx.bias_by_distance(table, buckets.long()),
           lambda: ctx.bias_by_distance(table.double(), buckets), lambda: ctx.bias_by_distance(table, buckets, out=table), lambda: ctx.bias_by_distance(table.T, buckets),
           lambda: ctx.bias_by_distance(table.cpu(), buckets)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            tell("taken:", i)
    large = [lambda: ctx.attention_biased(*args, torch.zeros((8, 2 * 1704 + 1), device="cuda")), lambda: ctx.cross_attention(kv, q[:, :7], start, lens, pages),
             lambda: ctx.attention_shared(*args, groups, shared, max_group=-1), lambda: ctx.attention_shared(*args, groups, shared, window=-1)]
    for f in large:
        with pytest.raises(QprojError):
            f()
    ctx.sync()
    assert (case(ctx) - ctx.attention(*args, max_q=1)).abs().max() < 1e-5
