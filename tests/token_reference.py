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
