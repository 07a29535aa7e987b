"""How exact causal attention is: errors in norm, and batches in whose sequences rows differ widely in size - what a row does not
see, and what it sees with a weight of next to nothing, leaves its results alone.  The short batches run on units of 16 rows, the
long ones of floats are computed from halves; both are held to the same bounds."""
import ctypes

import numpy as np
import pytest

from parallelreverseautodiff_amd import _lib
from parallelreverseautodiff_amd.exceptions import check
from test_causal_attention_gpu import Batch, close, dev, unfilled
from token_reference import attention

pytestmark = pytest.mark.gpu


def bounds(q, k, v, scale, u, g):
    """As token_reference.attention_bounds, with the error of each score taken for itself: err_ij of the score of query i and key
    j moves the weight p_ij by p_ij (err_ij + sum_l p_il err_il) to first order - the second term is the sum of the weights - and
    lse_i by sum_l p_il err_il, so that a score of great size whose weight is nothing loosens no bound."""
    q, k, v, g = (np.asarray(x, np.float64) for x in (q, k, v, g))
    n, m, d = len(q), len(k), q.shape[1]
    seen = np.arange(m)[None, :] <= np.arange(n)[:, None] + (m - n)
    with np.errstate(over="ignore", invalid="ignore"):     # (products with what is not seen)
        s, size = np.where(seen, q @ k.T * scale, -np.inf), np.where(seen, np.abs(q) @ np.abs(k).T, 0)
    top = s.max(axis=1)
    e = np.exp(s - top[:, None])
    p = e / e.sum(axis=1)[:, None]
    lse = top + np.log(e.sum(axis=1))
    err = (d + 4) * u * size * abs(scale)
    err += u * (np.abs(s, where=seen, out=np.zeros_like(s)) + np.abs(top)[:, None])
    mean = (p * err).sum(axis=1)[:, None]
    e_o = (p * (err + mean + (m + 8) * u)) @ np.abs(v) + (m + 4) * u * (p @ np.abs(v))
    e_lse = mean[:, 0] + (m + 8) * u + 4 * u * np.abs(lse)
    o = p @ v
    again = err + e_lse[:, None] + (4 * np.abs(lse)[:, None] + 8) * u
    with np.errstate(over="ignore", invalid="ignore"):
        dp, dp_size = np.where(seen, g @ v.T, 0), np.where(seen, np.abs(g) @ np.abs(v).T, 0)
    dot = (g * o).sum(axis=1)[:, None]
    e_dot = ((d + 2) * u * (np.abs(g) * np.abs(o)).sum(axis=1) + (np.abs(g) * e_o).sum(axis=1))[:, None]
    e_ds = p * (np.abs(dp - dot) * (again + 4 * u) + (d + 2) * u * dp_size + e_dot + 2 * u * (np.abs(dp) + np.abs(dot)))
    ds = p * np.abs(dp - dot)
    return (e_o, e_lse, abs(scale) * ((e_ds + (m + 4) * u * ds) @ np.abs(k)), abs(scale) * ((e_ds + (n + 4) * u * ds).T @ np.abs(q)),
            (p * (again + (n + 4) * u)).T @ np.abs(g))


HALVES = 0


class Spread(Batch):
    """A batch whose few heads are repeated `by` times on the device, or (HALVES) as often as makes it large enough for the
    halves: rows * heads * mean length of 2^23."""

    def repeat(self, by):
        if by == HALVES:
            by = -(-2 ** 23 * len(self.lengths) // (self.rows ** 2 * self.heads))
        self.few = self.heads, self.kv_heads, self.q, self.k, self.v, self.g
        self.by = by
        self.heads, self.kv_heads = by * self.heads, by * self.kv_heads
        self.q, self.k, self.v, self.g = (np.tile(x, (1, by)) for x in (self.q, self.k, self.v, self.g))
        self.cols = (0, self.q.shape[1], self.q.shape[1] + self.k.shape[1])
        self.full = [self.q.shape[1] + 2 * self.k.shape[1]] * 3
        self.tail = (self.heads, self.kv_heads) + self.tail[2:]
        self.upload()
        return self

    def run(self):
        """(o, lse, dq, dk, dv) of the few heads, after a look at whether all copies of them are the same."""
        o, l = self.forward()
        out = [o.download(), l.download(), *self.backward(o, l)]
        self.heads, self.kv_heads, self.q, self.k, self.v, self.g = self.few
        for i, x in enumerate(out):
            few = x[:x.shape[0] // self.by] if i == 1 else x[:, :x.shape[1] // self.by]
            assert np.array_equal(x, np.tile(few, (self.by, 1) if i == 1 else (1, self.by)), equal_nan=True)
            out[i] = few
        return out

    def definition(self):
        o, lse = np.zeros(self.q.shape), np.zeros((self.heads, self.rows))
        dq, dk, dv = np.zeros(self.q.shape), np.zeros(self.k.shape), np.zeros(self.v.shape)
        errors = [np.zeros_like(x) for x in (o, lse, dq, dk, dv)]
        u = float(np.finfo(self.dtype).eps) / 2
        for rows, h, qc, kc in self.each():
            args = self.q[rows, qc], self.k[rows, kc], self.v[rows, kc], self.scale
            o[rows, qc], lse[h, rows], dq[rows, qc], a, b = attention(*args, self.g[rows, qc])
            dk[rows, kc] += a
            dv[rows, kc] += b
            # a shared head's gradient is a sum over its group: one more rounding per head, in the bound's own terms
            e = bounds(*args, u * (1 + self.heads // self.kv_heads / (rows.stop - rows.start + 8)), self.g[rows, qc])
            errors[0][rows, qc], errors[1][h, rows], errors[2][rows, qc] = e[0], e[1], e[2]
            errors[3][rows, kc] += e[3]
            errors[4][rows, kc] += e[4]
        return (o, lse, dq, dk, dv), errors


NAMES = "o", "lse", "dq", "dk", "dv"


def compare(batch, names=NAMES, without=()):
    """The named results within their bounds in all rows of the sequences but `without`."""
    got = batch.run()
    with np.errstate(over="ignore", invalid="ignore"):      # (the rows that see a large value)
        want, error = batch.definition()
    rows = np.setdiff1d(np.arange(batch.starts[0], batch.starts[-1]), np.asarray(without, int))
    for name, x, r, e in zip(NAMES, got, want, error):
        if name in names:
            at = np.s_[:, rows] if name == "lse" else rows
            close(x[at], r[at], e[at], name)


KINDS = pytest.mark.parametrize("dtype,by", [(np.float64, 1), (np.float32, 1), (np.float32, HALVES)], ids=["f64", "f32", "f32-halves"])
SHAPES = pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 64), (4, 2, 40), (3, 1, 128)], ids=str)
LENGTHS = [190, 64, 100]


@KINDS
@pytest.mark.parametrize("lengths", [LENGTHS, [64] * 8, [400]], ids=str)
def test_errors_in_norm(gpu, dtype, by, lengths):
    """Normal data, the norm of a result's error over the result's: 16 unit roundoffs u.  A score is a chain of 64 products whose
    partial sums grow to 1.1: additions off by u / sqrt(3) of them in the mean, 1.1 * 0.7 * sqrt(64 / 3) = 4 u together; lse, of
    size 5, is rounded, taken in other units and rounded again, 2 * 5 / sqrt(3) = 6 u; their difference moves a weight by
    sqrt(4 ** 2 + 6 ** 2) = 7 u, a difference dP - D is off by as much, and a gradient by both, 10 u, before its sum over the
    rows evens out a part of that."""
    batch = Spread(dtype, lengths, 2, 2, 64, "fused").repeat(by)
    got, (want, _) = batch.run(), batch.definition()
    inside = slice(int(batch.starts[0]), int(batch.starts[-1]))
    for name, x, r in zip(NAMES, got, want):
        at = np.s_[:, inside] if name == "lse" else inside
        off = np.linalg.norm(x[at] - r[at]) / np.linalg.norm(r[at])
        assert off <= 8 * float(np.finfo(dtype).eps), (name, off)


@KINDS
@SHAPES
@pytest.mark.parametrize("down", [16, 24, 60])
def test_large_gradients_that_have_no_weight(gpu, dtype, by, heads, kv_heads, d, down):
    """The gradients of a sequence's tokens from 64 to 127 are 2^down times the others; to keys in front of them these tokens give
    weights of less than e^-90.  (The gradient of K is held as well: what those tokens add to it vanishes with their weight.)"""
    batch = Spread(dtype, [190, 64, 130], heads, kv_heads, d, "fused")
    large, front = np.zeros(batch.rows, bool), np.zeros(batch.rows, bool)
    for s in (batch.starts[0], batch.starts[2]):
        front[s:s + 64] = True
        large[s + 64:s + 128] = True
    large &= np.arange(batch.rows) < batch.starts[-1]
    batch.g[large] *= dtype(2.0 ** down)
    for i in range(kv_heads):
        batch.k[front, i * d] = -40
    for i in range(heads):
        batch.q[large, i * d] = 120 / (40 * batch.scale)
    compare(batch.repeat(by), ("dv", "dk"))


@KINDS
@SHAPES
@pytest.mark.parametrize("down", [16, 24, 100])
def test_large_gradients_that_do_not_reach_a_key(gpu, dtype, by, heads, kv_heads, d, down):
    """The gradients of a sequence's first 64 tokens are 2^down times the others: keys behind them are not seen by them."""
    batch = Spread(dtype, LENGTHS, heads, kv_heads, d, "fused")
    for s in batch.starts[:-1]:
        batch.g[s:s + 64] *= dtype(2.0 ** down)
    compare(batch.repeat(by), ("dq", "dk", "dv"))


# ---- tiles of different size, of which the large one has next to no weight -----------------------------------------------
@KINDS
@SHAPES
@pytest.mark.parametrize("down", [16, 24, 60])
def test_large_values_that_have_no_weight(gpu, dtype, by, heads, kv_heads, d, down):
    """The values of a sequence's first 64 tokens are 2^down times the others, and later queries give them weights of less than
    e^-90: 2^-130 of the sum, which is less than a rounding of what the others give."""
    batch = Spread(dtype, LENGTHS, heads, kv_heads, d, "fused")
    first = np.zeros(batch.rows, bool)
    for s in batch.starts[:-1]:
        first[s:s + 64] = True
    batch.v[first] *= dtype(2.0 ** down)
    for i in range(kv_heads):
        batch.k[first, i * d] = -40
    for i in range(heads):
        batch.q[~first, i * d] = 120 / (40 * batch.scale)
    compare(batch.repeat(by), ("o", "lse"))


# ---- one row of a tile much larger than the others ------------------------------------------------------------------------
LARGER = pytest.mark.parametrize("up", [14, 20, 40, 100, "lowest"])


def value_of(up, dtype):
    return np.finfo(dtype).min if up == "lowest" else dtype(2.0 ** up)


@KINDS
@SHAPES
@LARGER
@pytest.mark.parametrize("where", ["k", "v"])
def test_a_large_row_that_is_not_seen(gpu, dtype, by, heads, kv_heads, d, where, up):
    """The last token of each sequence, which no other sees, has a K or V that is 2^up times the others or the type's lowest value
    throughout."""
    batch = Spread(dtype, LENGTHS, heads, kv_heads, d, "fused")
    last = batch.starts[1:] - 1
    x = getattr(batch, where)
    if up == "lowest":
        x[last] = np.finfo(dtype).min
    else:
        x[last] *= value_of(up, dtype)
    compare(batch.repeat(by), ("o", "lse"), without=last)


@KINDS
@SHAPES
@pytest.mark.parametrize("up", [20, 40, 80])
def test_large_values_within_a_tile_that_have_no_weight(gpu, dtype, by, heads, kv_heads, d, up):
    """Every fifth token has values 2^up times the others, and all queries give those weights of less than e^-90 (2^-130)."""
    batch = Spread(dtype, LENGTHS, heads, kv_heads, d, "fused")
    large = np.arange(batch.rows) % 5 == 3
    for s in batch.starts[:-1]:
        large[s:s + 4] = False
    batch.v[large] *= dtype(2.0 ** min(up, 30))
    for i in range(kv_heads):
        batch.k[large, i * d] = -40
    for i in range(heads):
        batch.q[:, i * d] = 120 / (40 * batch.scale)
    batch.v[~large] *= dtype(2.0 ** (min(up, 30) - up))
    compare(batch.repeat(by), ("o", "lse"))


@KINDS
@SHAPES
@LARGER
@pytest.mark.parametrize("where", ["k", "v"])
def test_gradients_beside_a_large_row_that_is_not_seen(gpu, dtype, by, heads, kv_heads, d, where, up):
    """The same; the last token's own gradient is zero, so that it adds nothing to those of the keys that it sees."""
    batch = Spread(dtype, LENGTHS, heads, kv_heads, d, "fused")
    last = batch.starts[1:] - 1
    x = getattr(batch, where)
    if up == "lowest":
        x[last] = np.finfo(dtype).min
    else:
        x[last] *= value_of(up, dtype)
    batch.g[last] = 0
    batch.q[last] = 0       # (a score of 2^up, whose lse has an error of 2^up / 2^24, would give a weight of any size)
    compare(batch.repeat(by), ("dq", "dk", "dv"), without=last)


@KINDS
@SHAPES
@pytest.mark.parametrize("up", [14, 20, 40, 100])
@pytest.mark.parametrize("where", ["q", "g"])
def test_a_large_query_in_front(gpu, dtype, by, heads, kv_heads, d, where, up):
    """The second token of each sequence has a Q (of small keys) or a gradient 2^up times the others: keys behind it get nothing
    from it, the others' gradients of Q nothing either."""
    batch = Spread(dtype, LENGTHS, heads, kv_heads, d, "fused")
    getattr(batch, where)[batch.starts[:-1] + 1] *= dtype(2.0 ** up)
    if where == "q":
        batch.k *= dtype(2.0 ** -up)
    compare(batch.repeat(by), ("dq", "dk", "dv"))


# ---- scores far beyond what a weight resolves ------------------------------------------------------------------------------
@KINDS
@SHAPES
@pytest.mark.parametrize("size", [10, 22, 26, 31, 40, 60])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size(gpu, dtype, by, heads, kv_heads, d, size, sign):
    """One column of Q and K makes all scores, each a multiple of 2^size and without any rounding; the values grow and shrink by
    2^20 from one tile of 64 tokens to the next.  A query's largest score is 2^size above the others, at its own token or at the
    first: its weight is one and all others are nothing, so O is that token's value and lse that score.
    How far they may be off, in unit roundoffs u = 2^-24 of single precision.  In two halves x = hi + lo + r: hi has 11 bits, so
    |lo| <= 2^-11 |x|, and lo 11 more, |r| <= 2^-23 |x| = 2 u |x|.  O is a weight times a value without the product of the two lo, at
    most 2^-22 = 4 u, each off by 2 u, a sum of three products (1 u) over the sum of the weights (1 u): 10 u of the row's largest.
    The score is scale log2 e (2 u) times Q (1 u), split (2 u), times K (a half: exact), summed (1 u), times ln 2 (2 u): 8 u.  The
    other kernels have fewer roundings."""
    batch = Spread(dtype, [300, 64, 100], heads, kv_heads, d, "fused")
    batch.scale = 0.5
    batch.tail = batch.tail[:3] + (0.5,)
    batch.q[:], batch.k[:] = 0, 0
    want_at = np.arange(batch.rows)
    for a, b in zip(batch.starts[:-1], batch.starts[1:]):
        place = np.arange(b - a)
        batch.k[a:b, ::d] = sign * dtype(2.0) * (place[:, None] + 1)
        batch.v[a:b] *= (2.0 ** (20 * (place // 64 % 2)))[:, None].astype(dtype)
        if sign < 0:
            want_at[a:b] = a
    batch.q[:, ::d] = dtype(2.0 ** size)
    got = batch.repeat(by).run()
    inside = np.arange(batch.starts[0], batch.starts[-1])
    u, group = float(np.finfo(dtype).eps) / 2, heads // kv_heads
    for h in range(heads):
        kv = h // group
        v = batch.v[want_at[inside], kv * d:kv * d + d].astype(np.float64)
        o = got[0][inside, h * d:h * d + d].astype(np.float64)
        assert (np.abs(o - v) <= 10 * u * np.abs(v).max(axis=1, keepdims=True)).all(), (h, np.abs(o - v).max())
        score = batch.k[want_at[inside], kv * d].astype(np.float64) * 2.0 ** size * 0.5
        assert (np.abs(got[1][h, inside] - score) <= 8 * u * np.abs(score)).all(), h


# ---- which kernels a batch takes --------------------------------------------------------------------------------------------
def device_memory_left():
    free, total = ctypes.c_size_t(), ctypes.c_size_t()
    assert ctypes.CDLL("libamdhip64.so").hipMemGetInfo(ctypes.byref(free), ctypes.byref(total)) == 0
    return free.value


def test_thousands_of_short_sequences_of_many_heads(gpu):
    """Sequences of one to three tokens: kernels that give each a tile of 64 rows a head would work on 30 times the rows, in a
    workspace of 18 GB forward and 36 backward for operands of 74 MB."""
    batch = Spread(np.float32, [1, 2, 3] * 2000, 1, 1, 8, "fused")
    before = device_memory_left()
    compare(batch.repeat(192))
    assert before - device_memory_left() < 2 ** 31


def test_very_many_heads_of_one_column(gpu):
    """Head dimensions are padded to 32 where a batch is computed from halves: 8192 heads of one column would take 10 GB of
    workspace for operands of 67 MB."""
    batch = Spread(np.float32, [1500, 548], 2, 2, 1, "fused")
    before = device_memory_left()
    compare(batch.repeat(4096))
    assert before - device_memory_left() < 2 ** 31


@KINDS
@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("where", ["q", "k", "v", "g"])
def test_rows_without_a_finite_value(gpu, dtype, by, where, value):
    """Token 20 of the first sequence holds nothing finite: who does not see it keeps every bit."""
    clean, dirty = (Spread(dtype, LENGTHS, 2, 1, 64, "fused") for _ in range(2))
    at, end, last = int(clean.starts[0]) + 20, int(clean.starts[1]), int(clean.starts[-1])
    getattr(dirty, where)[at] = value
    a, b = clean.repeat(by).run(), dirty.repeat(by).run()
    before, others, behind = np.arange(clean.starts[0], at), np.arange(end, last), np.arange(at + 1, end)
    keep = {"o": np.r_[before, others], "lse": np.r_[before, others], "dq": np.r_[before, others], "dk": others, "dv": others}
    if where in "qg":       # one row that is not to be had, and the keys that it sees
        keep.update(o=np.r_[before, behind, others], lse=np.r_[before, behind, others], dq=np.r_[before, behind, others],
                    dk=np.r_[behind, others], dv=np.r_[behind, others])
    if where == "g":
        keep.update(o=np.r_[before, at, behind, others], lse=np.r_[before, at, behind, others])
    for name, x, y in zip(NAMES, a, b):
        rows = np.s_[:, keep[name]] if name == "lse" else keep[name]
        assert np.array_equal(x[rows], y[rows]), name
    assert where == "g" or np.isnan(b[0][at]).all()
