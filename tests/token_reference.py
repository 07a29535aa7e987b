"""The token model's operators in numpy, in 64 bits, straight from their definitions: what the device is compared with."""
import math

import numpy as np


def philox4x32(counter, key, rounds=10):
    """The four words of Philox4x32 for arrays of counters (4 words) and one key (2 words)."""
    c = [np.asarray(x, np.uint64) for x in counter]
    k = [int(x) for x in key]
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return [x.astype(np.uint32) for x in c]


def kept(shape, p, seed, site, step):
    n = int(np.prod(shape))
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    same = lambda v: np.full(block.shape, v & 0xFFFFFFFF, np.uint64)
    words = philox4x32((block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), same(step), same(site)),
                       (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    return (np.stack(words, axis=1).reshape(-1)[:n].astype(np.uint64) >= np.uint64(math.floor(p * 2.0 ** 32))).reshape(shape)


def embedding_gradient(dout, ids, scale, vocab):
    """The gradient, and per element the sum of the magnitudes that went into it and their number (for rounding bounds);
    sums in the longest type there is."""
    total = np.zeros((vocab, dout.shape[1]), np.longdouble)
    size, count = np.zeros_like(total), np.zeros((vocab, 1))
    for i, r in enumerate(ids):
        if 0 <= r < vocab:
            total[r] += dout[i]
            size[r] += np.abs(dout[i])
            count[r] += 1
    return total * np.longdouble(scale), size * abs(scale), count


def attention(q, k, v, scale, g=None):
    """One head of one sequence: n queries at the end of m keys.  Returns o, lse and, with the gradient g of o, (dq, dk, dv).
    A query without keys: zeros and -inf.  Only visible keys take part, whatever the others hold."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n, m, d = len(q), len(k), q.shape[1]
    o, lse = np.zeros((n, v.shape[1])), np.full(n, -np.inf)
    dq, dk, dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    for i in range(n):
        seen = min(m, m - n + i + 1)
        if seen <= 0:
            continue
        s = k[:seen] @ q[i] * scale
        top = s.max()
        e = np.exp(s - top)
        p = e / e.sum()
        lse[i] = top + math.log(e.sum())
        o[i] = p @ v[:seen]
        if g is not None:
            gi = np.asarray(g[i], np.float64)
            dp = v[:seen] @ gi
            ds = p * (dp - p @ dp) * scale
            dq[i] = ds @ k[:seen]
            dk[:seen] += np.outer(ds, q[i])
            dv[:seen] += np.outer(p, gi)
    return (o, lse) if g is None else (o, lse, dq, dk, dv)


def attention_bounds(q, k, v, scale, u, g):
    """How far o, lse, dq, dk, dv of one head may be off in arithmetic of unit roundoff u, whatever the order of the sums,
    counted term by term to first order in u (the factor 1.1 of the comparison covers the rest):
      a score: d products and their sum, the scaling (d + 4 roundings of |scale| sum |q||k|);
      a weight exp(s - top) / sum: the errors of two scores, an exponential good to 4 u, a sum of m terms, a division;
      backward's weight exp(s - lse): a score's error, lse's own and its rounding, 4 u;  and so on along the formulas."""
    q, k, v, g = (np.asarray(x, np.float64) for x in (q, k, v, g))
    n, m, d = len(q), len(k), q.shape[1]
    seen = np.arange(m)[None, :] <= np.arange(n)[:, None] + (m - n)
    s = np.where(seen, q @ k.T * scale, -np.inf)
    some = seen.any(axis=1)
    top = np.where(some, s.max(axis=1, initial=-np.inf), 0)
    e = np.exp(s - top[:, None])
    total = np.where(some, e.sum(axis=1), 1)
    p = e / total[:, None]
    lse = top + np.log(total)
    ds_score = np.where(seen, (d + 4) * u * (np.abs(q) @ np.abs(k).T) * abs(scale), 0)
    row = ds_score.max(axis=1, initial=0)[:, None] + u * (np.abs(s, where=seen, out=np.zeros_like(s)) + np.abs(top)[:, None])
    weight = 2 * row + (m + 8) * u
    o_size = p @ np.abs(v)
    e_o = (p * weight) @ np.abs(v) + (m + 4) * u * o_size
    e_lse = row.max(axis=1, initial=0) + (m + 8) * u + 4 * u * np.abs(lse)
    o = p @ v
    again = row + e_lse[:, None] + (4 * np.abs(lse)[:, None] + 8) * u     # backward's weights, relative
    dp, dp_size = g @ v.T, np.abs(g) @ np.abs(v).T
    dot = (g * o).sum(axis=1)[:, None]
    e_dot = ((d + 2) * u * (np.abs(g) * np.abs(o)).sum(axis=1) + (np.abs(g) * e_o).sum(axis=1))[:, None]
    e_ds = p * (np.abs(dp - dot) * (again + 4 * u) + (d + 2) * u * dp_size + e_dot + 2 * u * (np.abs(dp) + np.abs(dot)))
    ds = p * np.abs(dp - dot)
    e_dq = abs(scale) * ((e_ds + (m + 4) * u * ds) @ np.abs(k))
    e_dk = abs(scale) * ((e_ds + (n + 4) * u * ds).T @ np.abs(q))
    e_dv = (p * (again + (n + 4) * u)).T @ np.abs(g)
    return e_o, np.where(some, e_lse, 0), e_dq, e_dk, e_dv
