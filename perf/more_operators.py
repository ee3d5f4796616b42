"""Attention over the paged 4-bit cache in its other forms, as cases that can be measured.

Three operators, each in its plain form (elementary torch operations) and through the library:

* ``shared`` - causal attention of a batch in groups of sequences that have a long prefix in common: the same first pages.
* ``cross``  - attention of rows that see every token of another length: a decoder's over an encoder's states.
* ``biased`` - attention with a learned bias a head and bucket of the distance between a token and a row, causal (a
               decoder's own tokens) or seeing everything (an encoder's).

The cache is four tensors.  A page holds `page` tokens of every key/value head; a head's row is blocks of 32 values, each
a scale d (fp16) and 32 codes n of four bits that stand for d * (n - 8).  Values' codes lie in order, two a byte, the first
in the low half.  Keys' codes lie in words of eight: word w of a row of B blocks holds values 8 * (w // B) .. + 7 of
block w % B.

Buckets of a distance t - p: seen from both sides, half of them are for tokens behind the row, and of one side of n buckets the
first e = n // 2 are distances of their own, the others grow with the distance's logarithm up to the largest distance.  Causal,
all n are for tokens before the row.
"""
import math

import numpy as np
import torch

own = False

_context = None


def _ctx():
    global _context
    if _context is None:
        from magnitude_amd import Context

        _context = Context(0)
    return _context


# ---- cases ----------------------------------------------------------------------------------------------------------

def _shared(name, groups, seqs, prefix_lo, prefix_hi, past_lo, past_hi, new, heads, kv_heads, dim, page, ragged=False):
    """`groups` groups of `seqs` sequences; a group has prefix_lo to prefix_hi tokens in common (whole pages), a sequence past_lo to
    past_hi of its own behind them, and `new` newest ones (ragged: one to `new`)."""
    return {"name": name, "op": "shared", "groups": groups, "seqs": seqs, "prefix_lo": prefix_lo, "prefix_hi": prefix_hi, "past_lo": past_lo,
            "past_hi": past_hi, "new": new, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "ragged": ragged}


def _cross(name, seqs, states_lo, states_hi, new, heads, kv_heads, dim, page, ragged=False):
    """`seqs` sequences of states_lo to states_hi states, `new` rows each (ragged: one to `new`)."""
    return {"name": name, "op": "cross", "seqs": seqs, "states_lo": states_lo, "states_hi": states_hi, "new": new, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "ragged": ragged}


def _biased(name, seqs, past_lo, past_hi, new, causal, heads, kv_heads, dim, page, buckets, reach, ragged=False):
    """`seqs` sequences with past_lo to past_hi tokens before the `new` newest ones (ragged: one to `new`); `buckets` of distances
    up to `reach`."""
    return {"name": name, "op": "biased", "seqs": seqs, "past_lo": past_lo, "past_hi": past_hi, "new": new, "causal": causal, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "buckets": buckets, "reach": reach, "ragged": ragged}


def listed():
    return [
        # two chats behind one system prompt, a token each: latency
        _shared("shared-token-two", 1, 2, 1024, 1024, 20, 300, 1, 32, 8, 128, 64),
        # a serving step of 48 sequences behind one long system prompt with its tools
        _shared("shared-batch", 1, 48, 8192, 8192, 30, 1500, 1, 32, 8, 128, 64),
        # 32 questions about one very long document
        _shared("shared-document", 1, 32, 65536, 65536, 10, 400, 1, 32, 8, 128, 64),
        # speculative decoding in four groups of a small model: up to four draft tokens a sequence
        _shared("shared-draft-groups", 4, 9, 1500, 6000, 40, 700, 4, 14, 7, 64, 32, ragged=True),
        # one token of a decoder that looks at 1500 frames of an encoder
        _cross("cross-token", 1, 1500, 1500, 1, 20, 20, 64, 64),
        # a serving step of 40 sequences over encoder states of all lengths
        _cross("cross-batch", 40, 90, 6404, 1, 32, 8, 128, 64),
        # the last, ragged chunks of prompts over an image's states
        _cross("cross-prompt-ragged", 5, 1025, 1601, 187, 32, 8, 128, 128, ragged=True),
        # a whole prompt over four images' states
        _cross("cross-prompt", 1, 6404, 6404, 4096, 32, 8, 128, 64),
        # a decoder's tokens behind short answers
        _biased("biased-token", 16, 3, 511, 1, True, 16, 16, 64, 64, 32, 128),
        # a batch of texts through an encoder
        _biased("biased-encoder", 8, 0, 0, 512, False, 16, 16, 64, 64, 32, 128, ragged=True),
        # a long text through an encoder
        _biased("biased-encoder-long", 1, 0, 0, 4096, False, 16, 16, 64, 64, 32, 128),
        # a decoder's forced prefix, grouped heads, far-reaching buckets
        _biased("biased-prompt", 2, 100, 900, 500, True, 24, 8, 96, 16, 64, 400),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = {k: max(w[k], most.get(c["op"], {}).get(k, 0)) for k in w}
    while True:
        op = rng.choice(["shared", "shared", "cross", "biased"])
        dim, page = rng.choice([64, 96, 128, 128, 256]), rng.choice([16, 32, 64, 128, 256])
        kv_heads, group = rng.choice([1, 2, 4, 8, 8, 16]), rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
        ragged = rng.random() < 0.4
        if op == "shared":
            kind = rng.choice(["token", "token", "draft"])
            a, b = sorted((_log(rng, 100, 65536), _log(rng, 100, 65536)))
            lo, hi = sorted((_log(rng, 1, 2048) - 1, _log(rng, 1, 2048) - 1))
            groups = rng.choice([1, 1, 2, 3, 6])
            case = _shared("", groups, max(1, _log(rng, 1, 64) // groups), a, b, lo, hi, 1 if kind == "token" else rng.randint(2, 12), kv_heads * group, kv_heads,
                           dim, page, ragged)
            deep, rows, seqs = b + page, groups * case["seqs"] * case["new"], groups
        elif op == "cross":
            kind = rng.choice(["token", "token", "prompt"])
            lo, hi = sorted((_log(rng, 1, 8192), _log(rng, 1, 8192)))
            case = _cross("", _log(rng, 1, 64) if kind == "token" else rng.randint(1, 6), lo, hi, rng.choice([1, 1, 2, 5]) if kind == "token" else _log(rng, 17, 4096),
                          kv_heads * group, kv_heads, dim, page, ragged)
            deep, rows, seqs = hi, case["seqs"] * case["new"], case["seqs"]
        else:
            causal = rng.random() < 0.5
            lo, hi = sorted((_log(rng, 1, 2048) - 1, _log(rng, 1, 2048) - 1)) if causal else (0, 0)
            new = 1 if causal and rng.random() < 0.5 else _log(rng, 1, 4096)
            buckets = rng.choice([8, 32, 32, 64])
            case = _biased("", _log(rng, 1, 64) if new == 1 else rng.randint(1, 8), lo, hi, new, causal, kv_heads * group, kv_heads, dim, page, buckets,
                           rng.choice([128, 128, _log(rng, buckets, 500)]), ragged)
            deep, rows, seqs = hi + new, case["seqs"] * new, case["seqs"]
        # what the plain form lays out: padded keys and values, and scores
        if seqs * deep * kv_heads * dim > 4.2e8 or rows * deep * kv_heads * group > 5.4e8:
            continue
        del case["name"]
        w = work(case)
        if all(w[k] <= most[op][k] for k in w):
            return case


def _spread(i, lo, hi):
    """The i-th of a sequence of numbers between lo and hi that fills the range evenly."""
    return lo + int(((i * 0.6180339887498949) % 1.0) * (hi - lo + 1)) if i else hi


def _sequences(case):
    """(tokens in the cache, rows) of every sequence, and the tokens that groups have in common"""
    got, prefix = [], []
    if case["op"] == "shared":
        for g in range(case["groups"]):
            prefix.append(-(-_spread(g, case["prefix_lo"], case["prefix_hi"]) // case["page"]) * case["page"])
    for i in range(case["seqs"] * max(1, len(prefix))):
        new = _spread(i, 1, case["new"]) if case["ragged"] else case["new"]
        if case["op"] == "cross":
            got.append((_spread(i, case["states_lo"], case["states_hi"]), new))
        else:
            got.append((_spread(i, case["past_lo"], case["past_hi"]) + new + (prefix[i // case["seqs"]] if prefix else 0), new))
    return got, prefix


def work(case):
    """Inputs and results once each: fp32 rows; 4 bits a value and 2 bytes a block of 32 in the cache."""
    seqs, prefix = _sequences(case)
    rows = sum(new for _, new in seqs)
    kept = sum(n for n, _ in seqs) - (case["seqs"] - 1) * sum(prefix)
    if case["op"] == "cross" or not case.get("causal", True):
        pairs = sum(n * new for n, new in seqs)
    else:
        pairs = sum(new * (n - new) + new * (new + 1) // 2 for n, new in seqs)
    more = 4.0 * case["heads"] * case["buckets"] if case["op"] == "biased" else 0.0
    return {"bytes": kept * 2 * case["kv_heads"] * case["dim"] * 18 / 32 + 8.0 * rows * case["heads"] * case["dim"] + more,
            "flops": 4.0 * pairs * case["heads"] * case["dim"]}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _heads(g, tokens, heads, dim):
    """Rows of heads as projections give them: N(0, 1), one channel in sixteen four times as large."""
    x = torch.randn((tokens, heads, dim), generator=g, device="cuda")
    x[..., torch.randperm(dim, generator=g, device="cuda")[: dim // 16]] *= 4.0
    return x


def _quantize(x):
    """Codes (one a byte, [..., blocks, 32]) and fp16 scales [..., blocks] of rows of values."""
    x = x.unflatten(-1, (-1, 32))
    a = x.abs()
    at = torch.where(a == a.amax(-1, keepdim=True), torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
    d = x.gather(-1, at) / -8.0
    n = (x * (1.0 / d) + 8.5).trunc().clamp(0, 15)
    half = d.half()
    return torch.where(half != 0, n, 8.0).to(torch.uint8), half.squeeze(-1)


def _pack_keys(n):
    """[..., blocks, 32] codes -> bytes of a row, eight codes a word"""
    n = n.unflatten(-1, (4, 4, 2))                             # [..., block, eighth of 32, byte, half]
    b = n[..., 0] | (n[..., 1] << 4)
    return b.transpose(-3, -2).flatten(-3)                     # word = eighth * blocks + block


def _pack_values(n):
    n = n.flatten(-2).unflatten(-1, (-1, 2))
    return n[..., 0] | (n[..., 1] << 4)


def _unpack(b):
    return torch.stack((b & 15, b >> 4), dim=-1)


def _keys(codes, scales):
    n = _unpack(codes.unflatten(-1, (4, -1, 4))).transpose(-4, -3).flatten(-3)   # [..., block, 32]
    return ((n.float() - 8.0) * scales.float().unsqueeze(-1)).flatten(-2)


def _values(codes, scales):
    n = _unpack(codes).flatten(-2).unflatten(-1, (-1, 32))
    return ((n.float() - 8.0) * scales.float().unsqueeze(-1)).flatten(-2)


def _buckets(n, reach, both):
    """The bucket of every distance t - p from -reach to reach, int32."""
    d = torch.arange(-reach, reach + 1, dtype=torch.float64)
    side = n // 2 if both else n
    e = side // 2
    away = d.abs() if both else (-d).clamp(min=0)
    far = e + torch.floor(torch.log(away.clamp(min=1) / e) / math.log(reach / e) * (side - e) + 1e-9).clamp(max=side - e - 1)
    b = torch.where(away < e, away, far)
    return (b + side * (d > 0) if both else b).to(torch.int32)


def _cache(g, pages, kv_heads, page, dim):
    """A cache of rows as projections give them."""
    shape = (pages, kv_heads, page)
    cache = {"k_codes": torch.zeros(shape + (dim // 2,), dtype=torch.uint8, device="cuda"),
             "k_scales": torch.zeros(shape + (dim // 32,), dtype=torch.float16, device="cuda"),
             "v_codes": torch.zeros(shape + (dim // 2,), dtype=torch.uint8, device="cuda"),
             "v_scales": torch.zeros(shape + (dim // 32,), dtype=torch.float16, device="cuda")}
    for at in range(0, pages * page * kv_heads, 1 << 19):    # some rows at a time
        for part, pack in (("k", _pack_keys), ("v", _pack_values)):
            codes, scales = cache[part + "_codes"].view(-1, dim // 2), cache[part + "_scales"].view(-1, dim // 32)
            n, d = _quantize(_heads(g, len(codes[at:at + (1 << 19)]), 1, dim)[:, 0])
            codes[at:at + (1 << 19)], scales[at:at + (1 << 19)] = pack(n), d
    return cache


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h, dim, page = case["kv_heads"], case["dim"], case["page"]
    seqs, prefix = _sequences(case)
    common = [prefix[i // case["seqs"]] // page if prefix else 0 for i in range(len(seqs))]     # pages that are the group's
    count = [-(-n // page) for n, _ in seqs]
    total = sum(c - p for c, p in zip(count, common)) + sum(prefix) // page
    s = {"case": case, "cache": _cache(g, total, h, page, dim)}
    where = torch.randperm(total, generator=g, device="cuda").cpu().to(torch.int32)
    pages = torch.full((len(seqs), max(count)), -1, dtype=torch.int32)
    at = 0
    for i, (c, p) in enumerate(zip(count, common)):
        if prefix and i % case["seqs"] == 0:
            first = where[at:at + p]
            at += p
        if p:
            pages[i, :p] = first
        pages[i, p:c] = where[at:at + c - p]
        at += c - p
    s["pages"] = pages.cuda()
    s["q_start"] = torch.tensor(np.cumsum([0] + [new for _, new in seqs]), dtype=torch.int32).cuda()
    s["kv_len"] = torch.tensor([n for n, _ in seqs], dtype=torch.int32).cuda()
    if prefix:
        s["group_start"] = torch.arange(0, len(seqs) + 1, case["seqs"], dtype=torch.int32).cuda()
        s["shared_len"] = torch.tensor(prefix, dtype=torch.int32).cuda()
    s["q"] = _heads(g, sum(new for _, new in seqs), case["heads"], dim)
    s["y"] = torch.empty_like(s["q"])
    if case["op"] == "biased":
        s["table"] = 2.0 * torch.randn((case["buckets"], case["heads"]), generator=g, device="cuda")
        s["buckets"] = _buckets(case["buckets"], case["reach"], not case["causal"]).cuda()
    if own:
        from magnitude_amd import KvCache

        c = s["cache"]
        s["kv"] = KvCache(c["k_codes"], c["k_scales"], c["v_codes"], c["v_scales"])
        if case["op"] == "biased":      # the model's table, laid out once
            s["bias"] = _ctx().bias_by_distance(s["table"], s["buckets"])
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def _sums(scores, seen, v):
    """(largest score, sum of weights, sum of weighted values) over the tokens that are seen, [..., rows, tokens] x [..., tokens, dim]"""
    top = torch.where(seen, scores, -math.inf).amax(-1, keepdim=True).clamp(min=-3e38)
    w = torch.where(seen, torch.exp(scores - top), 0.0)
    return top, w.sum(-1, keepdim=True), torch.matmul(w.flatten(2, 3), v).view(w.shape[:4] + v.shape[-1:])


def _padded(s, n):
    """Queries as [sequences, kv heads, query heads of one, n rows, dim], scaled; rows of a sequence one after the other, then any others"""
    case, q, start = s["case"], s["q"], s["q_start"].long()
    i = torch.arange(n, device=q.device)
    rows = q[(start[:-1, None] + i).clamp(max=len(q) - 1)] * case["dim"] ** -0.5
    return rows.view(len(start) - 1, n, case["kv_heads"], -1, case["dim"]).permute(0, 2, 3, 1, 4)


def _scores(q, k):
    return torch.matmul(q.flatten(2, 3), k.transpose(-1, -2).contiguous()).view(q.shape[:4] + (-1,))


def _tokens(s, pages, back, part):
    """What pages [sequences, pages] hold, as [sequences, kv heads, tokens, dim]"""
    x = back(s["cache"][part + "_codes"][pages], s["cache"][part + "_scales"][pages])
    return x.transpose(1, 2).flatten(2, 3)


def _rows(s, y):
    """[sequences, kv heads, heads of one, rows, dim] -> the rows that there are, [tokens, heads, dim]"""
    start, n = s["q_start"].long(), y.shape[3]
    y = y.permute(0, 3, 1, 2, 4).flatten(2, 3).flatten(0, 1)
    row = torch.arange(len(s["q"]), device=y.device)
    seq = torch.searchsorted(start[1:], row, right=True)
    return y[seq * n + row - start[seq]]


def _shared_plain(s):
    case, n, page = s["case"], s["case"]["new"], s["case"]["page"]
    seqs, groups = case["seqs"], case["groups"]
    q = _padded(s, n)
    # the prefix, once a group: rows of all its sequences
    shared = s["shared_len"].long()
    most = -(-case["prefix_hi"] // page)
    first = s["pages"][::seqs, :most].clamp(min=0).long()
    all_rows = q.unflatten(0, (groups, seqs)).permute(0, 2, 3, 1, 4, 5).flatten(3, 4)      # [group, kv head, head, sequence x row, dim]
    t = torch.arange(most * page, device=q.device)
    seen = (t < shared[:, None])[:, None, None, None]
    a = _sums(_scores(all_rows, _tokens(s, first, _keys, "k")), seen, _tokens(s, first, _values, "v"))
    a = [x.unflatten(3, (seqs, n)).permute(0, 3, 1, 2, 4, 5).flatten(0, 1) for x in a]
    # a sequence's own tokens behind it (whole pages)
    start, length = s["q_start"].long(), s["kv_len"].long()
    shared = shared.repeat_interleave(seqs)
    deep = -(-(case["past_hi"] + n) // page)
    i = shared[:, None] // page + torch.arange(deep, device=q.device)
    mine = s["pages"].gather(1, i.clamp(max=s["pages"].shape[1] - 1)).clamp(min=0).long()
    t = shared[:, None] + torch.arange(deep * page, device=q.device)
    p = (length - (start[1:] - start[:-1]))[:, None] + torch.arange(n, device=q.device)
    seen = (t[:, None] <= p[:, :, None])[:, None, None]
    b = _sums(_scores(q, _tokens(s, mine, _keys, "k")), seen, _tokens(s, mine, _values, "v"))
    top = torch.maximum(a[0], b[0])
    f, g = torch.exp(a[0] - top), torch.exp(b[0] - top)
    return _rows(s, (a[2] * f + b[2] * g) / (a[1] * f + b[1] * g))


def _plain(s):
    case, n = s["case"], s["case"]["new"]
    q, at = _padded(s, n), s["pages"].clamp(min=0).long()
    scores = _scores(q, _tokens(s, at, _keys, "k"))
    start, length = s["q_start"].long(), s["kv_len"].long()
    t = torch.arange(scores.shape[-1], device=q.device)
    seen = (t < length[:, None])[:, None]
    if case["op"] == "biased":
        p = (length - (start[1:] - start[:-1]))[:, None] + torch.arange(n, device=q.device)
        away = t - p[:, :, None]
        if case["causal"]:
            seen = seen & (away <= 0)
        bias = s["table"][s["buckets"].long()].T[:, away.clamp(-case["reach"], case["reach"]) + case["reach"]]     # [head, sequence, row, token]
        scores = scores + bias.unflatten(0, (case["kv_heads"], -1)).permute(2, 0, 1, 3, 4)
    _, total, y = _sums(scores, seen[:, None, None], _tokens(s, at, _values, "v"))
    return _rows(s, torch.where(total > 0, y / total, 0.0))


def run(s):
    case = s["case"]
    if own:
        args = s["kv"], s["q"], s["q_start"], s["kv_len"], s["pages"]
        if case["op"] == "shared":
            return _ctx().attention_shared(*args, s["group_start"], s["shared_len"], max_q=case["new"], max_group=case["seqs"], out=s["y"], sync=False)
        if case["op"] == "cross":
            return _ctx().cross_attention(*args, max_q=case["new"], out=s["y"], sync=False)
        return _ctx().attention_biased(*args, s["bias"], causal=case["causal"], max_q=case["new"], out=s["y"], sync=False)
    return _shared_plain(s) if case["op"] == "shared" else _plain(s)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _bucket(n, reach, both, d):
    """Of one distance, in whole numbers: the bucket e + j where (d / e)^(side - e) reaches (reach / e)^j."""
    side, more = (n // 2, n // 2 if d > 0 else 0) if both else (n, 0)
    e, d = side // 2, abs(d) if both else max(0, -d)
    if d < e:
        return more + d
    j = 0
    while j + 1 < side - e and d ** (side - e) * e ** (j + 1) >= reach ** (j + 1) * e ** (side - e):
        j += 1
    return more + e + j


def exact(case, seed):
    s = prepare(case, seed)
    dim, h = case["dim"], case["kv_heads"]
    group = case["heads"] // h
    y = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    of = torch.arange(dim, device="cuda")
    word, turn, blk = of // 8 % 4 * (dim // 32) + of // 32, of % 8, of // 32     # of a key's value
    if case["op"] == "biased":
        reach = case["reach"]
        of_distance = torch.tensor([_bucket(case["buckets"], reach, not case["causal"], d) for d in range(-reach, reach + 1)], device="cuda")

    def codes(i, low, high, head):
        t = torch.arange(low, high, device="cuda")
        page, at = s["pages"][i].long()[t // case["page"]], t % case["page"]
        kc = s["cache"]["k_codes"][page, head, at].contiguous().view(torch.int32).long()
        k = ((kc[:, word] >> (4 * turn)) & 15).double() - 8
        k *= s["cache"]["k_scales"][page, head, at].double()[:, blk]
        vc = s["cache"]["v_codes"][page, head, at].long()[:, of // 2]
        v = ((vc >> (4 * (of % 2))) & 15).double() - 8
        v *= s["cache"]["v_scales"][page, head, at].double()[:, blk]
        return k, v

    seqs, prefix = _sequences(case)
    starts = np.cumsum([0] + [new for _, new in seqs])
    for head in range(h):
        common = None
        for i, (length, new) in enumerate(seqs):
            low = prefix[i // case["seqs"]] if prefix else 0
            if low and i % case["seqs"] == 0:
                common = codes(i, 0, low, head)
            k, v = codes(i, low, length, head)
            if low:
                k, v = torch.cat((common[0], k)), torch.cat((common[1], v))
            t, p = torch.arange(length, device="cuda"), torch.arange(length - new, length, device="cuda")
            hidden = (t[None] > p[:, None]) & bool(case["op"] == "shared" or case.get("causal", False))
            for j in range(head * group, (head + 1) * group):
                a = s["q"][starts[i]:starts[i + 1], j].double() @ k.T / math.sqrt(dim)
                if case["op"] == "biased":
                    away = (t[None] - p[:, None]).clamp(-reach, reach)
                    a += s["table"][:, j].double()[of_distance[away + reach]]
                y[starts[i]:starts[i + 1], j] = torch.softmax(a.masked_fill(hidden, -math.inf), dim=-1) @ v
    return y
