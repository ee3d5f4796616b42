"""Plain numpy statement, in 64 bits, of attention over the paged 4-bit cache in its other forms: rows that see everything, a
bias of the distance, both."""
import numpy as np

import kv_ref


def attention(cache, q, q_start, kv_len, pages, scale, sees_all=False, bias=None, dtype=np.float64):
    """As kv_ref.attention, for rows that see the tokens before them or all, with bias [heads, 2 * reach + 1] of t - p added to the scores.
    Returns (y, (weight, steep, spread, lift)): NaN in rows of no sequence, zeros in those that see nothing; lift is a head's largest bias."""
    k_codes, k_scales, v_codes, v_scales = cache
    page, heads_kv, dim = k_codes.shape[2], k_codes.shape[1], 2 * k_codes.shape[3]
    q, scale = np.asarray(q, dtype=dtype), dtype(scale)
    group = q.shape[1] // heads_kv
    y = np.full(q.shape, np.nan, dtype=dtype)
    weight, steep, spread = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape)
    lift = np.zeros(q.shape[:2])
    if bias is not None:
        finite = np.where(np.isfinite(bias), np.abs(bias), 0)
        lift[:] = finite.max(-1)
        reach = bias.shape[1] // 2
    for s in range(len(kv_len)):
        t = np.arange(int(kv_len[s]))
        where = np.asarray(pages)[s][t // page]
        good = (where >= 0) & (where < k_codes.shape[0])
        t, where = t[good], where[good]
        at = t % page
        k = kv_ref.decode(kv_ref.unpack_keys(k_codes[where, :, at]), k_scales[where, :, at]).astype(dtype)
        v = kv_ref.decode(kv_ref.unpack_values(v_codes[where, :, at]), v_scales[where, :, at]).astype(dtype)
        most = 8 * np.repeat(np.abs(k_scales[where, :, at].astype(np.float64)), 32, axis=-1)
        r = np.arange(q_start[s], q_start[s + 1])
        p = int(kv_len[s]) - (q_start[s + 1] - r)
        for h in range(q.shape[1]):
            with np.errstate(all="ignore"):
                a = q[r, h] @ k[:, h // group].T * scale
                if bias is not None:
                    a = a + bias[h].astype(dtype)[np.clip(t[None] - p[:, None], -reach, reach) + reach]
                if not sees_all:
                    a = np.where(t[None] <= p[:, None], a, -np.inf)
                seen = a != -np.inf
                top = np.where(seen, a, -np.inf).max(-1, initial=-np.inf, keepdims=True)
                w = np.where(seen, np.exp(a - np.where(np.isinf(top) & (top < 0), 0, top)), 0)
                total = w.sum(-1, keepdims=True)
                w = np.where(total != 0, w / total, 0).astype(dtype)
                y[r, h] = w @ v[:, h // group]
                weight[r, h] = w @ np.abs(v[:, h // group])
                spread[r, h] = seen.astype(np.float64) @ np.abs(v[:, h // group])
                if t.size:
                    steep[r, h] = np.where(seen, np.abs(q[r, h]) @ most[:, h // group].T, 0).max(-1) * abs(scale)
    return y, (weight, steep, spread, lift)


def allowed(sizes, dim, tokens):
    """kv_ref.allowed, and what a bias adds: its product with log2(e) is rounded twice (the constant, the product), its sum with the score or with what is
    taken off the score (the row's largest, which is a score and a bias too, and 13 + 2.5 in powers of two) once, of at most both: delta <=
    |bias| * 2 * 2^-24 + (2 * |bias| + |score| + 11) * 2^-24 more, and the score stays under `steep`."""
    weight, steep, spread, lift = sizes
    more = np.where(lift > 0, 4 * lift + steep + 11, 0) * 2.0 ** -24
    return kv_ref.allowed((weight, steep, spread), dim, tokens) + weight * np.expm1(2 * more)[..., None] * 1.01


def bucket(n, reach, both, d):
    """Of a distance t - p, in whole numbers: the bucket e + j where (d / e)^(side - e) reaches (reach / e)^j."""
    side, more = (n // 2, n // 2 if d > 0 else 0) if both else (n, 0)
    e, d = side // 2, abs(d) if both else max(0, -d)
    if d < e:
        return more + d
    j = 0
    while j + 1 < side - e and d ** (side - e) * e ** (j + 1) >= reach ** (j + 1) * e ** (side - e):
        j += 1
    return more + e + j
