"""What stands between a transformer block's q/k/v projections and its output projection, as cases that can be measured.

Three operators, each in its plain form (elementary torch operations) and through the library:

* ``rope``   - rotary positions of `tokens` rows of heads: neighbouring pairs or halves of the head, all of it or its first
               part, plain, stretched, with factors a frequency, or YaRN.
* ``append`` - the same tokens' keys and values into a paged cache held in 4 bits, the keys rotated on the way, with the
               queries' rotation beside them; then what the cache holds at those places, as values.
* ``attend`` - attention over such a cache: every sequence's newest tokens against all of it, or its last `window` tokens.

The cache is four tensors.  A page holds `page` tokens of every key/value head; a head's row is blocks of 32 values, each
a scale d (fp16) and 32 codes n of four bits that stand for d * (n - 8).  Values' codes lie in order, two a byte, the first
in the low half.  Keys' codes lie in words of eight: word w of a row of B blocks holds values 8 * (w // B) .. + 7 of
block w % B.  A block's scale is its value of largest magnitude (the first of them) over -8; n = min(15, trunc(x / d + 8.5)).
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

def _rope(name, tokens, heads, dim, dims, mode, scaling, first, strided):
    """`first`: the first token's position; `strided`: the heads lie inside the rows of a joined q/k/v product."""
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "dim": dim, "dims": dims, "mode": mode,
            "scaling": scaling, "first": first, "strided": strided}


def _append(name, tokens, heads, kv_heads, dim, dims, mode, scaling, first, page):
    return {"name": name, "op": "append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dims": dims,
            "mode": mode, "scaling": scaling, "first": first, "page": page}


def _attend(name, seqs, new, past_lo, past_hi, heads, kv_heads, dim, page, window=0, ragged=False):
    """`seqs` sequences with `past_lo` to `past_hi` tokens in the cache before the `new` newest ones (ragged: one to `new`)."""
    return {"name": name, "op": "attend", "seqs": seqs, "new": new, "past_lo": past_lo, "past_hi": past_hi, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "ragged": ragged}


def listed():
    return [
        # one decoded token's queries of an 8B-class model
        _rope("rope-token", 1, 32, 128, 128, "pairs", "none", 5000, False),
        # a long document's batch far behind its start: half of each head rotated, frequencies stretched, rows of a joined product
        _rope("rope-prompt-far", 2048, 40, 128, 64, "halves", "yarn", 1000003, True),
        # one decoded token: the smallest call, where latency is all there is
        _append("append-token", 1, 32, 8, 128, 128, "pairs", "none", 700, 16),
        # a serving step of 48 sequences, one token each
        _append("append-batch", 48, 32, 8, 128, 128, "halves", "factors", 9000, 64),
        # a whole prompt
        _append("append-prompt", 4096, 32, 8, 128, 128, "pairs", "none", 0, 64),
        # a decoded token of a short chat
        _attend("attend-token-short", 1, 1, 499, 499, 32, 8, 128, 16),
        # a decoded token behind a very long document
        _attend("attend-token-long", 1, 1, 131071, 131071, 32, 8, 128, 64),
        # a serving step of 48 sequences of all lengths
        _attend("attend-batch", 48, 1, 100, 8191, 32, 8, 128, 64),
        # speculative decoding: up to eight draft tokens of four sequences verified at once
        _attend("attend-verify", 4, 8, 1500, 6000, 32, 8, 128, 32, ragged=True),
        # a prompt batch of the engine (512 tokens) at the start of a sequence
        _attend("attend-prompt", 1, 512, 0, 0, 32, 8, 128, 64),
        # the last, ragged chunk of a long prompt in a small model whose layers look back 1024 tokens
        _attend("attend-prompt-window", 1, 187, 5000, 5000, 14, 2, 64, 128, window=1024),
        # a whole prompt at once
        _attend("attend-prompt-long", 1, 4096, 0, 0, 32, 8, 128, 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = {k: max(w[k], most.get(c["op"], {}).get(k, 0)) for k in w}
    while True:
        op = rng.choice(["rope", "append", "append", "attend", "attend", "attend"])
        dim = rng.choice([64, 96, 128, 128, 256])
        kv_heads, group = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
        dims = rng.choice([dim, dim, dim // 2, dim // 4])
        mode, scaling = rng.choice(["pairs", "halves"]), rng.choice(["none", "none", "stretch", "factors", "yarn"])
        if op == "rope":
            case = _rope("", _log(rng, 1, 4096), rng.randint(1, 64), rng.choice([dim, 80]), min(dims, 80), mode, scaling, _log(rng, 1, 1000000), rng.random() < 0.3)
        elif op == "append":
            case = _append("", _log(rng, 1, 4096), kv_heads * group, kv_heads, dim, dims, mode, scaling, _log(rng, 1, 200000), rng.choice([16, 32, 64, 128, 256]))
        else:
            kind = rng.choice(["token", "token", "draft", "prompt"])
            new = 1 if kind == "token" else rng.randint(2, 16) if kind == "draft" else _log(rng, 17, 4096)
            lo, hi = sorted((_log(rng, 1, 65536) - 1, _log(rng, 1, 65536) - 1))
            window = _log(rng, 128, 4096) if rng.random() < 0.25 else 0
            case = _attend("", _log(rng, 1, 64) if kind != "prompt" else rng.randint(1, 4), new, lo, hi, kv_heads * group, kv_heads, dim,
                           rng.choice([16, 32, 64, 128, 256]), window, rng.random() < 0.4)
            deep = hi + new
            # what the plain form lays out: padded keys and values, and scores
            if case["seqs"] * deep * kv_heads * dim > 4.2e8 or case["seqs"] * deep * new * kv_heads * group > 5.4e8:
                continue
        del case["name"]
        w = work(case)
        if all(w[k] <= most[op][k] for k in w):
            return case


def _spread(i, lo, hi):
    """The i-th of a sequence of numbers between lo and hi that fills the range evenly."""
    return lo + int(((i * 0.6180339887498949) % 1.0) * (hi - lo + 1)) if i else hi


def _sequences(case):
    """(tokens in the cache with the new ones, new ones) of every sequence"""
    got = []
    for i in range(case["seqs"]):
        new = _spread(i, 1, case["new"]) if case["ragged"] else case["new"]
        got.append((_spread(i, case["past_lo"], case["past_hi"]) + new, new))
    return got


def work(case):
    """Inputs and results once each: fp32 rows; 4 bits a value and 2 bytes a block of 32 in the cache."""
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 8.0 * n * case["dim"] + 4.0 * case["tokens"] + 4.0 * case["dims"], "flops": 3.0 * n * case["dims"]}
    if case["op"] == "append":
        t, kv = case["tokens"], 2 * case["kv_heads"] * case["dim"]
        # rows in, rotated queries out, codes and scales written, read again and written as values
        return {"bytes": 8.0 * t * case["heads"] * case["dim"] + t * kv * (4 + 2 * 18 / 32 + 4) + 12.0 * t + 4.0 * case["dims"],
                "flops": t * (3.0 * case["heads"] * case["dims"] + 3.0 * case["kv_heads"] * case["dims"] + 4.0 * kv)}
    rows = pairs = kept = 0
    for length, new in _sequences(case):
        rows += new
        w = case["window"] or length
        first = length - new   # position of the first new token
        # a token at position p sees min(p + 1, w) tokens
        full = max(0, min(new, w - 1 - first))   # new tokens that see everything before them
        pairs += full * (first + 1) + full * (full - 1) // 2 + (new - full) * w
        kept += length - max(0, first - w + 1)
    return {"bytes": kept * 2 * case["kv_heads"] * case["dim"] * 18 / 32 + 8.0 * rows * case["heads"] * case["dim"],
            "flops": 4.0 * pairs * case["heads"] * case["dim"]}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _frequencies(dims, scaling):
    """(radians a position for every pair, in 64 bits; what cosines and sines are multiplied by)"""
    i = torch.arange(dims // 2, dtype=torch.float64)
    f = 10000.0 ** (-2.0 * i / dims)
    if scaling == "none":
        return f, 1.0
    if scaling == "stretch":
        return f / 4.0, 1.0
    if scaling == "factors":   # long wavelengths eight times as long, short ones as they are, a ramp between
        return f / (1.0 + 7.0 * torch.clamp((i / (dims // 2) - 0.3) / 0.4, 0.0, 1.0)), 1.0
    # YaRN: pairs that turn more than 32 times over the 32768 tokens of training stay, those of less than one are stretched by 32
    low = max(0.0, math.floor(dims * math.log(32768 / (32.0 * 2 * math.pi)) / (2 * math.log(10000.0))))
    high = min(dims - 1.0, math.ceil(dims * math.log(32768 / (1.0 * 2 * math.pi)) / (2 * math.log(10000.0))))
    keep = 1.0 - torch.clamp((i - low) / max(0.001, high - low), 0.0, 1.0)
    return f / 32.0 * (1.0 - keep) + f * keep, float(np.float32(1.0 + 0.1 * math.log(32.0)))


def _heads(g, tokens, heads, dim, strided=False):
    """Rows of heads as projections give them: N(0, 1), one channel in sixteen four times as large.  Strided: the first
    columns of wider rows."""
    x = torch.randn((tokens, heads * (2 if strided else 1), dim), generator=g, device="cuda")
    x[..., torch.randperm(dim, generator=g, device="cuda")[: dim // 16]] *= 4.0
    return x[:, :heads]


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


def _cache(pages, kv_heads, page, dim):
    shape = (pages, kv_heads, page)
    return {"k_codes": torch.zeros(shape + (dim // 2,), dtype=torch.uint8, device="cuda"),
            "k_scales": torch.zeros(shape + (dim // 32,), dtype=torch.float16, device="cuda"),
            "v_codes": torch.zeros(shape + (dim // 2,), dtype=torch.uint8, device="cuda"),
            "v_scales": torch.zeros(shape + (dim // 32,), dtype=torch.float16, device="cuda")}


def _handle(cache):
    """The library's view of those four tensors."""
    from magnitude_amd import KvCache

    return KvCache(cache["k_codes"], cache["k_scales"], cache["v_codes"], cache["v_scales"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] in ("rope", "append"):
        freqs, s["magnitude"] = _frequencies(case["dims"], case["scaling"])
        s["freqs"] = freqs.cuda()
        t = case["tokens"]
        s["pos"] = (case["first"] + torch.arange(t, device="cuda")).to(torch.int32)
        s["q"] = _heads(g, t, case["heads"], case["dim"], case.get("strided", False))
        s["q_out"] = torch.empty((t, case["heads"], case["dim"]), device="cuda")
    if case["op"] == "append":
        h, dim, page = case["kv_heads"], case["dim"], case["page"]
        s["k"], s["v"] = _heads(g, t, h, dim), _heads(g, t, h, dim)
        if t <= 64:   # a token each of many sequences: anywhere in their pages
            s["pos"] = torch.randint(0, case["first"] + 1, (t,), generator=g, device="cuda").to(torch.int32)
            places = torch.randperm(2 * t, generator=g, device="cuda")[:t] * page + torch.randint(0, page, (t,), generator=g, device="cuda")
            s["cache"] = _cache(2 * t, h, page, dim)
        else:         # a run of tokens, its pages in any order
            n = -(-t // page)
            where = torch.randperm(n, generator=g, device="cuda")
            i = torch.arange(t, device="cuda")
            places = where[i // page] * page + i % page
            s["cache"] = _cache(n, h, page, dim)
        s["slots"] = places.to(torch.int64)
        s["k_out"], s["v_out"] = (torch.empty((t, h, dim), device="cuda") for _ in "kv")
    if case["op"] == "attend":
        h, dim, page = case["kv_heads"], case["dim"], case["page"]
        seqs = _sequences(case)
        count = [-(-length // page) for length, _ in seqs]
        s["cache"] = _cache(sum(count), h, page, dim)
        where = torch.randperm(sum(count), generator=g, device="cuda")
        for at in range(0, sum(count) * page * h, 1 << 19):    # some rows at a time
            for part, pack in (("k", _pack_keys), ("v", _pack_values)):
                codes, scales = s["cache"][part + "_codes"].view(-1, dim // 2), s["cache"][part + "_scales"].view(-1, dim // 32)
                n, d = _quantize(_heads(g, len(codes[at:at + (1 << 19)]), 1, dim)[:, 0])
                codes[at:at + (1 << 19)], scales[at:at + (1 << 19)] = pack(n), d
        pages = torch.full((case["seqs"], max(count)), -1, dtype=torch.int32)
        ends = np.cumsum([0] + count)
        for i, n in enumerate(count):
            pages[i, :n] = where[ends[i]:ends[i + 1]].cpu().to(torch.int32)
        s["pages"] = pages.cuda()
        s["q_start"] = torch.tensor(np.cumsum([0] + [new for _, new in seqs]), dtype=torch.int32).cuda()
        s["kv_len"] = torch.tensor([length for length, _ in seqs], dtype=torch.int32).cuda()
        rows = sum(new for _, new in seqs)
        s["q"] = _heads(g, rows, case["heads"], dim)
        s["y"] = torch.empty_like(s["q"])
    if own and "cache" in s:
        s["kv"] = _handle(s["cache"])
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def _rotate(x, pos, freqs, mode, magnitude, exactly):
    """Rows of heads, rotated.  Angles in 64 bits: the fraction of a turn is what is left of a position of a million.
    `exactly`: the products too, rounded once, for values that go on to be rounded to codes."""
    dims = 2 * len(freqs)
    angle = pos.double()[:, None] * freqs
    c, s = (torch.cos(angle) * magnitude)[:, None], (torch.sin(angle) * magnitude)[:, None]
    part = x[..., :dims]
    if exactly:
        part = part.double()
    else:
        c, s = c.float(), s.float()
    a, b = (part[..., 0::2], part[..., 1::2]) if mode == "pairs" else (part[..., : dims // 2], part[..., dims // 2:])
    u, v = a * c - b * s, a * s + b * c
    turned = torch.stack((u, v), dim=-1).flatten(-2) if mode == "pairs" else torch.cat((u, v), dim=-1)
    return torch.cat((turned.float(), x[..., dims:]), dim=-1)


def _append_plain(s):
    case, cache = s["case"], s["cache"]
    k = _rotate(s["k"], s["pos"], s["freqs"], case["mode"], s["magnitude"], True)
    page, at = s["slots"] // case["page"], s["slots"] % case["page"]
    out = {"q": _rotate(s["q"], s["pos"], s["freqs"], case["mode"], s["magnitude"], False)}
    for part, x, pack, back in (("k", k, _pack_keys, _keys), ("v", s["v"], _pack_values, _values)):
        n, d = _quantize(x)
        cache[part + "_codes"][page, :, at] = pack(n)
        cache[part + "_scales"][page, :, at] = d
        out[part] = back(cache[part + "_codes"][page, :, at], cache[part + "_scales"][page, :, at])
    return out


def _attend_plain(s):
    case, cache, q = s["case"], s["cache"], s["q"]
    seqs, new, h, dim, group = case["seqs"], case["new"], case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    at = s["pages"].clamp(min=0).long()

    def rows(part, back):   # [seqs, kv_heads, tokens, dim]
        x = back(cache[part + "_codes"][at], cache[part + "_scales"][at])
        return x.transpose(1, 2).flatten(2, 3)

    k, v = rows("k", _keys), rows("v", _values)
    start, length = s["q_start"].long(), s["kv_len"].long()
    count = start[1:] - start[:-1]
    i = torch.arange(new, device=q.device)
    padded = q[(start[:-1, None] + i).clamp(max=len(q) - 1)] * dim ** -0.5
    padded = padded.view(seqs, new, h, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, h, group * new, dim)
    scores = torch.matmul(padded, k.transpose(-1, -2).contiguous()).view(seqs, h, group, new, -1)
    t = torch.arange(scores.shape[-1], device=q.device)
    p = (length[:, None] - count[:, None] + i)[:, :, None]                    # position of every new token
    seen = t <= p
    if case["window"]:
        seen &= t > p - case["window"]
    seen = seen[:, None, None]
    top = torch.where(seen, scores, -math.inf).amax(-1, keepdim=True).clamp(min=-3e38)
    w = torch.where(seen, torch.exp(scores - top), 0.0)
    del scores
    total = w.sum(-1, keepdim=True)
    y = torch.matmul(w.view(seqs, h, group * new, -1), v).view(seqs, h, group, new, dim)
    y = torch.where(total > 0, y / total, 0.0).permute(0, 3, 1, 2, 4).reshape(seqs * new, h * group, dim)
    row = torch.arange(len(q), device=q.device)
    seq = torch.searchsorted(start[1:], row, right=True)
    return y[seq * new + row - start[seq]]


def run(s):
    case = s["case"]
    if own:
        ctx = _ctx()
        if case["op"] == "attend":
            return ctx.attention(s["kv"], s["q"], s["q_start"], s["kv_len"], s["pages"], max_q=case["new"],
                                 window=case["window"], out=s["y"], sync=False)
        if case["op"] == "rope":
            return ctx.rope(s["q"], s["pos"], s["freqs"], mode=case["mode"], magnitude=s["magnitude"], out=s["q_out"], sync=False)
        ctx.kv_append(s["kv"], s["k"], s["v"], s["slots"], pos=s["pos"], freqs=s["freqs"], mode=case["mode"],
                      magnitude=s["magnitude"], q=s["q"], q_out=s["q_out"], sync=False)
        k, v = ctx.kv_read(s["kv"], s["slots"], k_out=s["k_out"], v_out=s["v_out"], sync=False)
        return {"q": s["q_out"], "k": k, "v": v}
    if case["op"] == "attend":
        return _attend_plain(s)
    if case["op"] == "rope":
        return _rotate(s["q"], s["pos"], s["freqs"], case["mode"], s["magnitude"], False)
    return _append_plain(s)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _turned(x, pos, freqs, mode, magnitude):
    """x[token, head, dim] in double as complex numbers times magnitude * e^(i angle)"""
    half = len(freqs)
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if mode == "pairs" else (slice(0, half), slice(half, 2 * half))
    z = torch.complex(x[..., one], x[..., two]) * torch.polar(torch.full_like(freqs, magnitude), pos.double()[:, None] * freqs)[:, None]
    y = x.clone()
    y[..., one], y[..., two] = z.real, z.imag
    return y


def _stands_for(x):
    """What a cache gives back for rows of values (numpy, fp32 in, double out)"""
    b = x.reshape(-1, 32)
    top = b[np.arange(len(b)), np.abs(b).argmax(1)]
    d = top / np.float32(-8)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        n = np.minimum(np.floor(b * (np.float32(1) / d)[:, None] + np.float32(8.5)), 15)
    d = d.astype(np.float16).astype(np.float64)[:, None]
    return np.where(d == 0, 0.0, d * (n - 8)).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _turned(s["q"].double(), s["pos"], s["freqs"], case["mode"], s["magnitude"])
    if case["op"] == "append":
        k = _turned(s["k"].double(), s["pos"], s["freqs"], case["mode"], s["magnitude"]).float()
        return {"q": _turned(s["q"].double(), s["pos"], s["freqs"], case["mode"], s["magnitude"]),
                "k": _stands_for(k.cpu().numpy()), "v": _stands_for(s["v"].cpu().numpy())}
    dim, h = case["dim"], case["kv_heads"]
    group = case["heads"] // h
    y = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    word = torch.arange(dim, device="cuda") // 8 % 4 * (dim // 32) + torch.arange(dim, device="cuda") // 32   # of a key's value
    turn, blk = torch.arange(dim, device="cuda") % 8, torch.arange(dim, device="cuda") // 32
    row = 0
    for i, (length, new) in enumerate(_sequences(case)):
        t = torch.arange(length, device="cuda")
        page, at = s["pages"][i].long()[t // case["page"]], t % case["page"]
        low = max(0, length - new - case["window"] + 1) if case["window"] else 0
        page, at, t = page[low:], at[low:], t[low:]
        p = torch.arange(length - new, length, device="cuda")
        seen = t[None] <= p[:, None]
        if case["window"]:
            seen &= p[:, None] - t[None] < case["window"]
        for head in range(h):
            kc = s["cache"]["k_codes"][page, head, at].contiguous().view(torch.int32).long()
            k = ((kc[:, word] >> (4 * turn)) & 15).double() - 8
            k *= s["cache"]["k_scales"][page, head, at].double()[:, blk]
            vc = s["cache"]["v_codes"][page, head, at].long()[:, torch.arange(dim, device="cuda") // 2]
            v = ((vc >> (4 * (torch.arange(dim, device="cuda") % 2))) & 15).double() - 8
            v *= s["cache"]["v_scales"][page, head, at].double()[:, blk]
            for j in range(head * group, (head + 1) * group):
                a = s["q"][row:row + new, j].double() @ k.T / math.sqrt(dim)
                a.masked_fill_(~seen, -math.inf)
                y[row:row + new, j] = torch.softmax(a, dim=-1) @ v
        row += new
    return y
