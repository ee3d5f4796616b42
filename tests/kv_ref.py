"""Plain numpy statements, in 64 bits, of rotary positions, the paged 4-bit cache and attention over it."""
import numpy as np


def rotate(x, pos, freqs, mode, magnitude=1.0):
    """x [tokens, heads, dim] -> float64"""
    y = np.array(x, dtype=np.float64)
    half = len(freqs)
    a = np.asarray(pos, dtype=np.float64)[:, None] * np.asarray(freqs, dtype=np.float64)
    c, s = (magnitude * np.cos(a))[:, None], (magnitude * np.sin(a))[:, None]
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if mode == "pairs" else (slice(0, half), slice(half, 2 * half))
    u, v = y[..., one].copy(), y[..., two].copy()
    y[..., one], y[..., two] = u * c - v * s, u * s + v * c
    return y


def quantize(x):
    """fp32 rows [..., dim] -> (codes [..., dim / 32, 32], fp16 scales [..., dim / 32])"""
    b = np.asarray(x, dtype=np.float32).reshape(x.shape[:-1] + (-1, 32))
    with np.errstate(all="ignore"):
        whole = np.isfinite(b).all(-1)
        top = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1)      # argmax: the first of equals
        d = top / np.float32(-8)
        h = d.astype(np.float16)[..., 0]
        n = np.clip(np.trunc(b * (np.float32(1) / d) + np.float32(8.5)), 0, 15)
    whole &= np.isfinite(h)
    n = np.where((whole & (h != 0))[..., None], n, 8).astype(np.uint8)
    return n, np.where(whole, h, np.float16(np.nan))


def pack_keys(n):
    blocks = n.shape[-2]
    words = np.zeros(n.shape[:-2] + (4 * blocks,), dtype=np.uint32)
    for b in range(blocks):
        for e in range(4):
            for j in range(8):
                words[..., e * blocks + b] |= n[..., b, 8 * e + j].astype(np.uint32) << (4 * j)
    return np.ascontiguousarray(words).view(np.uint8)


def pack_values(n):
    n = n.reshape(n.shape[:-2] + (-1, 2))
    return n[..., 0] | (n[..., 1] << 4)


def unpack_keys(codes):
    """bytes [..., dim / 2] -> codes [..., dim]"""
    words = np.ascontiguousarray(codes).view(np.uint32)
    blocks = words.shape[-1] // 4
    n = np.zeros(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=np.uint8)
    for b in range(blocks):
        for e in range(4):
            for j in range(8):
                n[..., 32 * b + 8 * e + j] = (words[..., e * blocks + b] >> (4 * j)) & 15
    return n


def unpack_values(codes):
    return np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[:-1] + (2 * codes.shape[-1],))


def decode(n, scales):
    """codes [..., dim], fp16 scales [..., dim / 32] -> float64"""
    with np.errstate(all="ignore"):
        return (n.astype(np.float64) - 8) * np.repeat(scales.astype(np.float64), 32, axis=-1)


def attention(cache, q, q_start, kv_len, pages, scale, window=0, dtype=np.float64):
    """cache: (k_codes, k_scales, v_codes, v_scales) as numpy arrays.  Returns (y, (weight, steep, spread)): y [tokens, heads, dim] with NaN in
    rows of no sequence, and for error bounds sum_t p_t |v_t| and, of a row, the largest of a token's sums over d of
    scale * |q_d| * 8 * (the scale of the key's block), which the products with its codes stay under, and sum_t |v_t|.  In
    another `dtype` the same statement with every number of that type."""
    k_codes, k_scales, v_codes, v_scales = cache
    page = k_codes.shape[2]
    heads_kv, dim = k_codes.shape[1], 2 * k_codes.shape[3]
    q, scale = np.asarray(q, dtype=dtype), dtype(scale)
    group = q.shape[1] // heads_kv
    y = np.full(q.shape, np.nan, dtype=dtype)
    weight, steep, spread = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape)
    for s in range(len(kv_len)):
        t = np.arange(int(kv_len[s]))
        where = np.asarray(pages)[s][t // page]
        good = (where >= 0) & (where < k_codes.shape[0])
        t, where = t[good], where[good]
        at = t % page
        k = decode(unpack_keys(k_codes[where, :, at]), k_scales[where, :, at]).astype(dtype)
        v = decode(unpack_values(v_codes[where, :, at]), v_scales[where, :, at]).astype(dtype)
        most = 8 * np.repeat(np.abs(k_scales[where, :, at].astype(np.float64)), 32, axis=-1)
        for r in range(q_start[s], q_start[s + 1]):
            p = int(kv_len[s]) - (q_start[s + 1] - r)
            seen = t <= p
            if window:
                seen &= t > p - window
            for h in range(q.shape[1]):
                y[r, h] = 0
                if not seen.any():
                    continue
                ks, vs = k[seen, h // group], v[seen, h // group]
                with np.errstate(all="ignore"):
                    a = ks @ q[r, h] * scale
                    w = np.exp(a - a.max())
                    w /= w.sum()
                    y[r, h] = (w[:, None] * vs).sum(0)
                    weight[r, h] = (w[:, None] * np.abs(vs)).sum(0)
                    spread[r, h] = np.abs(vs).sum(0)
                    steep[r, h] = (most[seen, h // group] @ np.abs(q[r, h])).max() * abs(scale)
    return y, (weight, steep, spread)


def allowed(sizes, dim, tokens):
    """How far an fp32 result may be from the exact one.  A score is `dim` products of q, kept in 22 bits (a fp16
    pair: off by 2^-22 of itself, or of the row's largest over 2^15), with codes of -8 to 7.  Their fp32 sums round at most
    dim + 16 times: delta <= steep * (2^-21 + (dim + 16) * 2^-24).  A weight is
    then off by a factor of exp(2 delta) at most, by its own rounding to 22 bits, the exponential's (2 ulp) and the running sums'
    (a rounding every 16 tokens, and one a rescaling: fewer than tokens / 8 + 64).  A weight that is under 2^-26 of the row's largest
    is a multiple of 2^-37 of that, a value under 2^-25 of the largest near it a multiple of 2^-36 of that: what a dimension in which
    the heavy tokens have zeros is off by."""
    weight, steep, spread = sizes
    delta = steep * (2.0 ** -21 + (dim + 16) * 2.0 ** -24)
    return weight * (np.expm1(2 * delta)[..., None] + (tokens / 8 + 64) * 2.0 ** -24 + 2.0 ** -21) + 2.0 ** -36 * spread.max(-1, keepdims=True) + 1e-37
