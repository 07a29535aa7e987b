"""Causal attention over packed sequences with grouped heads, forward and backward, and the newest tokens against a cache,
on the device against their definition in 64 bits."""
import ctypes

import numpy as np
import pytest

from conftest import assert_parity
from parallelreverseautodiff_amd import _lib, seeded
from parallelreverseautodiff_amd.exceptions import check
from parallelreverseautodiff_amd.matrix import DeviceBuffer, IndexVector
from token_reference import attention, attention_bounds

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dtype", [np.float64, np.float32], ids=["f64", "f32"])


def dev(a):
    b = DeviceBuffer.alloc(a.dtype, *a.shape)
    b.upload(a)
    return b


def unfilled(dtype, rows, cols):
    return dev(np.full((rows, cols), np.nan, dtype))


class Batch:
    """Packed sequences with rows in front and behind that belong to none; the three operands as columns of one matrix
    ("fused") or as matrices of their own with columns around them, which makes every address odd ("apart")."""

    def __init__(self, dtype, lengths, heads, kv_heads, d, layout, seed=31, front=2, behind=3):
        self.dtype, self.lengths, self.heads, self.kv_heads, self.d = np.dtype(dtype), lengths, heads, kv_heads, d
        self.starts = front + np.concatenate([[0], np.cumsum(lengths)])
        self.rows = int(self.starts[-1]) + behind
        self.scale = 1.1 / np.sqrt(d)
        wide, narrow = heads * d, kv_heads * d
        normal = lambda t, cols: seeded.normal(seed, t, (self.rows, cols), 1.0, dtype)
        self.q, self.k, self.v, self.g = normal(1, wide), normal(2, narrow), normal(3, narrow), normal(4, wide)
        if layout == "fused":
            self.cols = (0, wide, wide + narrow)
            self.full = [wide + 2 * narrow] * 3
        else:
            self.cols = (1, 3, 2)
            self.full = [wide + 1, narrow + 4, narrow + 3]
        self.layout = layout
        self.offsets = IndexVector.from_values(self.starts)
        self.tail = (heads, kv_heads, d, self.scale)
        self.upload()

    def upload(self):
        if self.layout == "fused":
            one = dev(np.concatenate([self.q, self.k, self.v], axis=1))
            self.b = [one] * 3
        else:
            self.b = []
            for x, col, full in zip((self.q, self.k, self.v), self.cols, self.full):
                m = np.full((self.rows, full), np.nan, self.dtype)      # (columns of nobody hold NaN)
                m[:, col:col + x.shape[1]] = x
                self.b.append(dev(m))

    def operands(self):
        return [x for b, c in zip(self.b, self.cols) for x in (b.handle, c)]

    def forward(self, lse=True):
        o = unfilled(self.dtype, self.rows, self.heads * self.d)
        l = unfilled(self.dtype, self.heads, self.rows) if lse else None
        check(_lib.load().prad_causal_attention_fwd(*self.operands(), o.handle, l.handle if lse else None, self.offsets.handle, *self.tail))
        return o, l

    def backward(self, o, l):
        """(dq, dk, dv) as numpy, and that no other cell was written."""
        g = dev(self.g)
        if self.layout == "fused":
            d = [unfilled(self.dtype, self.rows, self.full[0])] * 3
        else:
            d = [unfilled(self.dtype, self.rows, full) for full in self.full]
        grads = [x for b, c in zip(d, self.cols) for x in (b.handle, c)]
        check(_lib.load().prad_causal_attention_bwd(*self.operands(), o.handle, l.handle, g.handle, *grads, self.offsets.handle, *self.tail))
        whole = [b.download() for b in d]
        out, first, last = [], self.starts[0], self.starts[-1]
        for m, col, x in zip(whole, self.cols, (self.q, self.k, self.v)):
            part = m[:, col:col + x.shape[1]]
            assert np.isnan(part[:first]).all() and np.isnan(part[last:]).all(), "rows outside the sequences were written"
            out.append(part)
            if self.layout == "apart":
                rest = np.delete(m, np.s_[col:col + x.shape[1]], axis=1)
                assert np.isnan(rest).all(), "other columns were written"
        return out

    def each(self):
        """(sequence rows, query head columns, key head columns) of every head of every sequence."""
        group, d = self.heads // self.kv_heads, self.d
        for s, n in enumerate(self.lengths):
            if n == 0:
                continue
            rows = slice(int(self.starts[s]), int(self.starts[s]) + n)
            for h in range(self.heads):
                yield rows, h, slice(h * d, h * d + d), slice(h // group * d, h // group * d + d)

    def reference(self):
        o, lse = np.zeros(self.q.shape), np.zeros((self.heads, self.rows))
        dq, dk, dv = np.zeros(self.q.shape), np.zeros(self.k.shape), np.zeros(self.v.shape)
        errors = [np.zeros_like(x) for x in (o, lse, dq, dk, dv)]
        # a shared head's gradient is a sum over its group: one more rounding per head, in the bound's own terms
        u = float(np.finfo(self.dtype).eps) / 2
        for rows, h, qc, kc in self.each():
            args = self.q[rows, qc], self.k[rows, kc], self.v[rows, kc], self.scale
            o[rows, qc], lse[h, rows], dq[rows, qc], a, b = attention(*args, self.g[rows, qc])
            dk[rows, kc] += a
            dv[rows, kc] += b
            e = attention_bounds(*args, u * (1 + self.heads // self.kv_heads / (rows.stop - rows.start + 8)), self.g[rows, qc])
            errors[0][rows, qc], errors[1][h, rows], errors[2][rows, qc] = e[0], e[1], e[2]
            errors[3][rows, kc] += e[3]
            errors[4][rows, kc] += e[4]
        return (o, lse, dq, dk, dv), errors


def close(got, want, bound, what):
    # a weight below the smallest normal number becomes zero, which moves a result by that number times what the weight would have
    # multiplied: up to some hundred terms of a size of some thousand here
    worst = np.abs(got.astype(np.float64) - want) - 1.1 * bound - float(np.finfo(got.dtype).tiny) * 2.0 ** 20
    assert not np.isnan(got).any(), what + ": not written, or NaN"
    assert worst.max() <= 0, "%s: %.3g over its bound at %s" % (what, worst.max(), np.unravel_index(worst.argmax(), worst.shape))


def close_in_norm(got, want, dtype, what):
    """The norm of the error against the norm of the result, 32 unit roundoffs.  The maximum over the elements of a gradient
    cannot be held to the bar of a single product: an element of dS is P (dP - D), a difference of two sums of d products whose
    rounding alone, (d + 2) u sum |g||v|, reaches 130 * 6e-8 * 80 = 6e-4 at d = 128 where the result is of order 1; `close`
    holds each element to its own bound.  Over all elements these errors have either sign: a chain of d rounded additions
    wanders by sqrt(d / 3) u of its size, a score of size 1 built from partial sums of at most sqrt(d) scale = 1.1 by 7 u at
    d = 128, a weight is off by two of them, and a gradient by a weight and a difference: under 32 u together."""
    off = np.linalg.norm(got.astype(np.float64) - want) / max(np.linalg.norm(want), np.finfo(np.float64).tiny)
    assert off <= 16 * float(np.finfo(dtype).eps), "%s: off by %.3g in norm" % (what, off)


def compare(batch, parity=True):
    """Every element within its rounding bound and, unless the scores are so large that a score's own rounding moves a weight by
    more than that, within the bar of the other operations."""
    inner = slice(int(batch.starts[0]), int(batch.starts[-1]))
    o, l = batch.forward()
    got_o, got_l = o.download(), l.download()
    for part in (got_o[:inner.start], got_o[inner.stop:], got_l[:, :inner.start], got_l[:, inner.stop:]):
        assert np.isnan(part).all(), "rows outside the sequences were written"
    got = batch.backward(o, l)
    (ro, rl, *rg), (eo, el, *eg) = batch.reference()
    if inner.start == inner.stop:
        return
    close(got_o[inner], ro[inner], eo[inner], "o")
    close(got_l[:, inner], rl[:, inner], el[:, inner], "lse")
    for x, r, e, name in zip(got, rg, eg, ("dq", "dk", "dv")):
        close(x[inner], r[inner], e[inner], name)
        if parity and r[inner].any():
            close_in_norm(x[inner], r[inner], batch.dtype, name)
    if parity:
        assert_parity(got_o[inner], ro[inner], batch.dtype, "o")
    alone, _ = batch.forward(lse=False)
    assert np.array_equal(alone.download(), got_o, equal_nan=True)


# lengths on both sides of a tile (16, 32, 64), single tokens, empty sequences, none at all; head dimensions on both sides of the
# padded ones (32, 64, 128); groups of 1, 2, 3, 5 and 8; operands in one matrix or at odd addresses
CASES = [([1], 1, 1, 1, "fused"), ([5], 2, 1, 3, "apart"), ([0, 0], 2, 2, 8, "fused"), ([0, 3, 0, 1, 2, 0], 2, 2, 16, "fused"), ([49, 1, 17, 33], 3, 3, 32, "fused"),
         ([16, 15, 17], 4, 2, 33, "apart"), ([64, 63, 65, 1], 2, 1, 40, "fused"), ([31, 32, 33], 6, 2, 64, "fused"), ([130, 2], 5, 1, 64, "apart"),
         ([20, 100], 3, 1, 65, "apart"), ([70, 0, 129], 4, 4, 80, "fused"), ([129], 8, 1, 128, "fused"), ([90, 45], 2, 2, 127, "apart"), ([200], 6, 3, 96, "apart"),
         ([260, 90], 4, 2, 128, "apart"),
         # longer ones
         ([300, 0, 129, 64, 1, 77, 40], 4, 2, 64, "fused"), ([520], 3, 1, 40, "apart"), ([63, 65, 130, 255, 100], 2, 2, 32, "fused"), ([257, 256, 31], 4, 1, 128, "fused"),
         ([600, 32], 5, 1, 80, "apart"), ([1] * 530, 2, 1, 64, "fused"), ([1300], 1, 1, 16, "fused"), ([130, 400], 6, 2, 127, "apart")]


# Batches whose rows * heads * mean length passes 2^23: those of floats are computed from halves.
LARGE = [([300, 0, 129, 64, 1, 77, 40], 160, 80, 64, "fused"), ([520], 33, 11, 40, "apart"), ([63, 65, 130, 255, 100], 112, 112, 32, "fused"), ([257, 256, 31], 84, 21, 128, "fused"),
         ([600, 32], 45, 9, 80, "apart"), ([1] * 20 + [900], 208, 104, 16, "fused"), ([1300], 13, 13, 16, "fused"), ([130, 400], 60, 20, 127, "apart"), ([1, 700, 2], 64, 1, 8, "fused")]


@DTYPES
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention_against_its_definition(gpu, dtype, case):
    compare(Batch(dtype, *case))


@pytest.mark.parametrize("case", LARGE, ids=[str((len(c[0]), *c[1:])) for c in LARGE])
def test_attention_of_large_batches_against_its_definition(gpu, case):
    batch = Batch(np.float32, *case)
    assert batch.rows * batch.heads * (batch.rows // len(batch.lengths)) >= 2 ** 23
    compare(batch)


# (long: in the sense of LARGE)
LONG = pytest.mark.parametrize("long", [False, True], ids=["short", "long"])


def times(long, heads, kv_heads, by=32):
    return (heads * by, kv_heads * by) if long else (heads, kv_heads)


@DTYPES
@LONG
def test_scores_far_apart_and_far_from_zero(gpu, dtype, long):
    """Scores of several hundreds: the running maximum moves, most weights vanish."""
    batch = Batch(dtype, [550, 40] if long else [150, 40], *times(long, 2, 1), 64, "fused")
    batch.q *= 12
    batch.k *= 12
    batch.upload()
    compare(batch, parity=False)


@DTYPES
@LONG
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_a_scale_that_is_not_positive(gpu, dtype, long, scale):
    batch = Batch(dtype, [540] if long else [70], *times(long, 2, 1), 32, "fused")
    batch.scale = scale
    batch.tail = batch.tail[:3] + (scale,)
    compare(batch)


@DTYPES
@LONG
def test_rows_of_very_different_size(gpu, dtype, long):
    """Tokens whose values differ by thousands, tiles of zeros among them, everything far below one: every element stays within
    its bound (which grows with the largest values a row mixes)."""
    batch = Batch(dtype, [560, 30] if long else [190, 30], *times(long, 2, 1), 64, "fused")
    size = 2.0 ** (np.arange(batch.rows) // 37 % 5 * 3.0 - 12)
    for x in (batch.v, batch.g):
        x *= (size * 2.0 ** -20)[:, None].astype(dtype)
    batch.v[70:140] = 0
    batch.k *= size[::-1, None].astype(dtype)
    batch.q[100:170] = 0
    batch.upload()
    compare(batch, parity=False)


@DTYPES
@LONG
def test_equal_calls_give_equal_bits(gpu, dtype, long):
    batch = Batch(dtype, [900, 77, 1, 130] if long else [300, 77, 1, 130], *times(long, 6, 2, 8), 64, "fused")
    first = batch.forward()
    grads = batch.backward(*first)
    for _ in range(2):
        again = batch.forward()
        assert all(np.array_equal(a.download(), b.download(), equal_nan=True) for a, b in zip(first, again))
        assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(grads, batch.backward(*again)))


@DTYPES
@LONG
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("where", ["q", "k", "v", "g"])
def test_values_that_are_not_finite_reach_only_who_sees_them(gpu, dtype, where, value, long):
    """Token 20 of the second sequence holds one: earlier tokens and other sequences keep every bit of O and of the gradients
    that do not depend on it; whoever sees it gets NaN."""
    lengths = [33, 450, 140] if long else [33, 50, 40]
    clean, dirty = (Batch(dtype, lengths, *times(long, 2, 1, 36), 40, "fused") for _ in range(2))
    at = int(clean.starts[1]) + 20
    getattr(dirty, where)[at, 7] = value        # (head 0)
    dirty.upload()
    co, cl = clean.forward()
    do, dl = dirty.forward()
    cg, dg = clean.backward(co, cl), dirty.backward(do, dl)
    a, b = co.download(), do.download()
    first, last, second_end = int(clean.starts[0]), int(clean.starts[-1]), int(clean.starts[2])
    head0, head1, both = slice(0, 40), slice(40, 80), slice(0, 80)
    # rows of O that see it: of head 0 the row itself (q), of both heads that share its k and v this row and the later ones
    hit = np.zeros(a.shape, bool)
    if where == "q":
        hit[at, head0] = True
    elif where in "kv":
        hit[at:second_end, both] = True
    inside = np.zeros(a.shape, bool)
    inside[first:last] = True
    assert np.array_equal(a[inside & ~hit], b[inside & ~hit]) and np.isnan(b[hit]).all()
    # gradients: sequences one and three keep their bits, nothing outside the second is NaN
    for x, y in zip(cg, dg):
        for rows in (slice(first, int(clean.starts[1])), slice(second_end, last)):
            assert np.array_equal(x[rows], y[rows])
    dq, dk, dv = dg
    if where in "qg":       # one query row: its own dq, and the keys it sees
        assert np.isnan(dq[at, head0]).all() and np.array_equal(dq[at, head1], cg[0][at, head1])
        rest = np.r_[int(clean.starts[1]):at, at + 1:second_end]
        assert np.array_equal(dq[rest], cg[0][rest])
        later = slice(at + 1, second_end)
        for x, y in ((dk, cg[1]), (dv, cg[2])):
            assert np.array_equal(x[later], y[later]) and np.isnan(x[int(clean.starts[1]):at + 1, head0]).all()
    else:                   # a key: the queries from it on
        before = slice(int(clean.starts[1]), at)
        assert np.array_equal(dq[before], cg[0][before]) and np.isnan(dq[at:second_end, both]).all()
        assert np.isnan(dk[int(clean.starts[1]):second_end, head0]).all()
    for x, y, own in zip(cg, dg, (both, head0, head0)):        # other heads: nothing
        others = np.delete(np.arange(x.shape[1]), np.r_[own])
        assert np.array_equal(x[first:last, others], y[first:last, others])


@LONG
def test_rows_of_nobody_are_not_read_for_a_result(gpu, long):
    clean, dirty = (Batch(np.float32, [470, 20] if long else [70, 20], *times(long, 4, 2, 12), 64, "fused", front=70, behind=70) for _ in range(2))
    first, last = int(clean.starts[0]), int(clean.starts[-1])
    for x in (dirty.q, dirty.k, dirty.v, dirty.g):
        x[:first] = np.nan
        x[last:] = np.inf
    dirty.upload()
    a, b = clean.forward(), dirty.forward()
    assert np.array_equal(a[0].download()[first:last], b[0].download()[first:last])
    assert all(np.array_equal(x[first:last], y[first:last]) for x, y in zip(clean.backward(*a), dirty.backward(*b)))


@DTYPES
@LONG
def test_a_recorded_training_pass_reads_the_offsets_of_each_launch(gpu, dtype, long):
    lib, by = _lib.load(), 5 if long else 1
    batch = Batch(dtype, [60 * by, 60 * by, 30 * by], *times(long, 4, 2, 12), 64, "fused", front=0, behind=0)
    o, l = unfilled(dtype, batch.rows, batch.heads * 64), unfilled(dtype, batch.heads, batch.rows)
    g, d = dev(batch.g), unfilled(dtype, batch.rows, batch.full[0])
    grads = [x for c in batch.cols for x in (d.handle, c)]

    def enqueue():
        check(lib.prad_causal_attention_fwd(*batch.operands(), o.handle, l.handle, batch.offsets.handle, *batch.tail))
        check(lib.prad_causal_attention_bwd(*batch.operands(), o.handle, l.handle, g.handle, *grads, batch.offsets.handle, *batch.tail))

    enqueue()
    check(lib.prad_graph_begin())
    try:
        enqueue()
    finally:
        gr = ctypes.c_void_p()
        check(lib.prad_graph_end(ctypes.byref(gr)))
    for lengths in ([150, 0, 0], [1, 148, 1], [50, 50, 50], [0, 75, 75]):
        batch.offsets.upload(by * np.concatenate([[0], np.cumsum(lengths)]))
        check(lib.prad_graph_launch(gr))
        got = o.download(), l.download(), d.download()
        o.zero(), l.zero(), d.zero()
        enqueue()
        assert all(np.array_equal(a, b.download()) for a, b in zip(got, (o, l, d)))
    check(lib.prad_graph_destroy(gr))


@LONG
def test_offsets_that_describe_no_rows_do_no_harm(gpu, long):
    """Offsets past the rows, negative or falling: cut off to rows of the buffers, nothing outside is touched."""
    lib = _lib.load()
    batch = Batch(np.float32, [40, 540] if long else [40, 40], *times(long, 2, 1), 32, "fused", front=0, behind=0)
    room = DeviceBuffer.alloc(np.float32, batch.rows + 64, batch.heads * 32)
    room.upload(np.full((room.rows, room.cols), 7, np.float32))
    o = room.view_rows(32, batch.rows)
    for values in ([0, 40, 1000], [-5, 40, 80], [40, 0, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1, -1]):
        batch.offsets.upload(values)
        check(lib.prad_causal_attention_fwd(*batch.operands(), o.handle, None, batch.offsets.handle, *batch.tail))
        whole = room.download()
        assert np.all(whole[:32] == 7) and np.all(whole[32 + batch.rows:] == 7)


def test_attention_refusals(gpu):
    lib = _lib.load()
    f = lambda r, c, t=np.float32: DeviceBuffer.alloc(t, r, c)
    x, o, lse, off = f(10, 64), f(10, 32), f(2, 10), IndexVector.from_values([0, 10])
    fwd = lambda q=x, qc=0, k=x, kc=32, v=x, vc=48, o=o, lse=lse, off=off, h=2, kvh=1, d=16, sc=0.25: \
        lib.prad_causal_attention_fwd(q.handle, qc, k.handle, kc, v.handle, vc, o.handle, lse.handle if lse else None, off.handle, h, kvh, d, sc)
    assert fwd() == _lib.PRAD_OK and fwd(lse=None) == _lib.PRAD_OK
    for change, status in (({"qc": 33}, _lib.PRAD_ERR_SHAPE), ({"vc": 49}, _lib.PRAD_ERR_SHAPE), ({"kc": -1}, _lib.PRAD_ERR_SHAPE), ({"vc": 2 ** 62}, _lib.PRAD_ERR_SHAPE),
                           ({"k": f(9, 64)}, _lib.PRAD_ERR_SHAPE), ({"o": f(10, 48)}, _lib.PRAD_ERR_SHAPE), ({"o": f(9, 32)}, _lib.PRAD_ERR_SHAPE),
                           ({"lse": f(10, 2)}, _lib.PRAD_ERR_ARG), ({"off": IndexVector.alloc(1)}, _lib.PRAD_ERR_SHAPE), ({"h": 3}, _lib.PRAD_ERR_SHAPE),
                           ({"h": 2, "kvh": 3}, _lib.PRAD_ERR_ARG), ({"h": 0}, _lib.PRAD_ERR_ARG), ({"d": 129}, _lib.PRAD_ERR_ARG), ({"d": 0}, _lib.PRAD_ERR_ARG),
                           ({"h": 2 ** 62, "kvh": 2 ** 62}, _lib.PRAD_ERR_ARG), ({"sc": float("inf")}, _lib.PRAD_ERR_ARG), ({"v": f(10, 64, np.float64)}, _lib.PRAD_ERR_DTYPE),
                           ({"off": x}, _lib.PRAD_ERR_BAD_HANDLE), ({"q": off}, _lib.PRAD_ERR_BAD_HANDLE)):
        assert fwd(**change) == status, change
    # more rows than the kernels count (borrowed views of the same few rows: refused before anything is read)
    tall = lambda b, rows: DeviceBuffer.wrap(np.float32, rows, b.cols, b.ptr, parent=b)
    n = 2 ** 30 - 384
    assert fwd(q=tall(x, n), k=tall(x, n), v=tall(x, n), o=tall(o, n), lse=None) == _lib.PRAD_ERR_ARG
    wide = f(20, 32)
    assert fwd(q=wide.view_rows(0, 10), o=wide.view_rows(5, 10), k=x, v=x) == _lib.PRAD_ERR_ARG     # an output over an input
    dx, g = f(10, 64), f(10, 32)
    bwd = lambda dq=dx, dqc=0, dk=dx, dkc=32, dv=dx, dvc=48, g=g, o=o: lib.prad_causal_attention_bwd(
        x.handle, 0, x.handle, 32, x.handle, 48, o.handle, lse.handle, g.handle, dq.handle, dqc, dk.handle, dkc, dv.handle, dvc, off.handle, 2, 1, 16, 0.25)
    assert bwd() == _lib.PRAD_OK
    for change, status in (({"dkc": 31}, _lib.PRAD_ERR_ARG), ({"dvc": 40}, _lib.PRAD_ERR_ARG), ({"dvc": 49}, _lib.PRAD_ERR_SHAPE), ({"dq": x}, _lib.PRAD_ERR_ARG),
                           ({"dk": g, "dkc": 0}, _lib.PRAD_ERR_ARG), ({"g": f(10, 31)}, _lib.PRAD_ERR_ARG), ({"dv": f(11, 64)}, _lib.PRAD_ERR_SHAPE),
                           ({"dv": f(10, 64, np.float64)}, _lib.PRAD_ERR_DTYPE)):
        assert bwd(**change) == status, change


# ---- the newest tokens against the cache ----------------------------------------------------------------------------------
def cached(dtype, new, ranges, rows, heads, kv_heads, d, seed=41, edit=None, odd=False):
    """Runs the call; returns (what the device gave, the queries, keys, values, scale)."""
    q = seeded.normal(seed, 1, (sum(new) + 4, heads * d), 1.0, dtype)       # two rows of nobody on either side
    k, v = (seeded.normal(seed, t, (rows, kv_heads * d), 1.0, dtype) for t in (2, 3))
    if edit is not None:
        edit(q, k, v)
    scale = 0.9 / np.sqrt(d)
    if odd:
        wide = [np.full((x.shape[0], x.shape[1] + 3), np.nan, dtype) for x in (q, k, v)]
        for w, x in zip(wide, (q, k, v)):
            w[:, 1:1 + x.shape[1]] = x
        b, col = [dev(w) for w in wide], 1
    else:
        b, col = [dev(x) for x in (q, k, v)], 0
    o = unfilled(dtype, *q.shape)
    off = IndexVector.from_values(2 + np.concatenate([[0], np.cumsum(new)]))
    begin, end = (IndexVector.from_values([r[i] for r in ranges]) for i in (0, 1))
    call = lambda: check(_lib.load().prad_cached_attention(b[0].handle, col, b[1].handle, col, b[2].handle, col, o.handle, off.handle, begin.handle, end.handle,
                                                           heads, kv_heads, d, scale))
    call()
    got = o.download()
    o.upload(np.full(q.shape, np.nan, dtype))
    call()
    assert np.array_equal(o.download(), got, equal_nan=True)
    return got, q, k, v, scale


def against_definition(dtype, new, ranges, rows, heads, kv_heads, d, odd=False):
    got, q, k, v, scale = cached(dtype, new, ranges, rows, heads, kv_heads, d, odd=odd)
    u, group, at = float(np.finfo(dtype).eps) / 2, heads // kv_heads, 2
    want, bound = np.zeros(q.shape), np.zeros(q.shape)
    for n, (b, e) in zip(new, ranges):
        rows_q = slice(at, at + n)
        at += n
        for h in range(heads):
            qc, kc = slice(h * d, h * d + d), slice(h // group * d, h // group * d + d)
            keys = slice(b, max(b, e))
            want[rows_q, qc], _ = attention(q[rows_q, qc], k[keys, kc], v[keys, kc], scale)
            if e > b:
                bound[rows_q, qc] = attention_bounds(q[rows_q, qc], k[keys, kc], v[keys, kc], scale, 2 * u, np.zeros((n, d)))[0]
    assert np.isnan(got[:2]).all() and np.isnan(got[at:]).all(), "rows outside the sequences were written"
    if at > 2:
        close(got[2:at], want[2:at], bound[2:at], "o")      # (2 u: joining parts rescales each sum once more)
        assert_parity(got[2:at], want[2:at], dtype, "o")


# single tokens with caches of every kind (empty, one key, around a tile of 16, long), chunks of new tokens, more new tokens than
# keys, no new token, ranges that overlap or share rows, groups of more than the 16 rows of a tile
CACHED = [([1], [(0, 1)], 1, 1, 1, 4), ([1], [(3, 3)], 9, 2, 1, 32), ([1, 1, 1], [(0, 16), (20, 35), (40, 57)], 64, 4, 2, 64), ([1], [(7, 2007)], 2048, 8, 2, 128),
          ([1, 1], [(0, 300), (0, 300)], 512, 3, 1, 33), ([5, 1, 0, 9], [(0, 40), (30, 80), (80, 90), (95, 104)], 120, 4, 1, 80), ([4], [(10, 12)], 30, 2, 2, 16),
          ([1], [(0, 70)], 70, 20, 1, 64), ([33], [(0, 100)], 128, 6, 2, 40), ([1] * 40, [(10 * i, 10 * i + i) for i in range(40)], 400, 2, 1, 64),
          ([1], [(100, 4100)], 4200, 16, 1, 128), ([200], [(0, 350)], 400, 2, 1, 64),
          # caches of more than 512 rows, whose keys are cut into parts: some sequences with parts and some without, an empty one,
          # several tiles of rows, fewer keys than queries, more than 64 sequences, none or few keys in the last part, as many
          # parts as there may be
          ([1, 1, 1], [(0, 700), (700, 700), (650, 2000)], 2048, 2, 1, 33), ([9, 40], [(5, 900), (300, 1700)], 1800, 6, 2, 40), ([700], [(0, 600)], 640, 2, 2, 16),
          ([1] * 70, [(20 * i, 20 * i + i * 37 % 900) for i in range(70)], 2400, 2, 1, 64), ([2, 0, 3], [(0, 5000), (10, 5000), (4990, 5000)], 5000, 20, 1, 128),
          ([1], [(0, 513)], 513, 1, 1, 1), ([1, 1], [(0, 9000), (0, 640)], 9001, 4, 4, 8)]


@DTYPES
@pytest.mark.parametrize("case", CACHED, ids=[str(i) for i in range(len(CACHED))])
@pytest.mark.parametrize("odd", [False, True], ids=["even", "odd"])
def test_cached_attention_against_its_definition(gpu, dtype, case, odd):
    against_definition(dtype, *case, odd=odd)


def test_thousands_of_sequences(gpu):
    """Sequences are found by a search of three rounds; short and empty ones in between, packed and against a cache."""
    compare(Batch(np.float64, [1, 0, 2] * 1400, 2, 1, 4, "fused"))
    against_definition(np.float32, [1, 0, 2] * 1400, [(i % 500, i % 500 + i % 13) for i in range(4200)], 512, 2, 1, 4)


def test_more_units_than_a_launch_has_workgroups(gpu):
    """With 40000 heads of one column a launch has 26 workgroups to a head and the sequences 30 tiles: some take two.  All heads
    hold the same, so all results do."""
    lib, heads, lengths = _lib.load(), 40000, [433, 16]
    rows, starts = sum(lengths), [0, 433, 449]
    x = [seeded.normal(77, i, (rows, 1), 1.0, np.float64) for i in range(4)]
    q, k, v, g = (dev(np.repeat(y, heads, axis=1)) for y in x)
    o, l, dq, dk, dv = (unfilled(np.float64, *s) for s in ((rows, heads), (heads, rows), (rows, heads), (rows, heads), (rows, heads)))
    off = IndexVector.from_values(starts)
    check(lib.prad_causal_attention_fwd(q.handle, 0, k.handle, 0, v.handle, 0, o.handle, l.handle, off.handle, heads, heads, 1, 1.0))
    check(lib.prad_causal_attention_bwd(q.handle, 0, k.handle, 0, v.handle, 0, o.handle, l.handle, g.handle, dq.handle, 0, dk.handle, 0, dv.handle, 0,
                                        off.handle, heads, heads, 1, 1.0))
    got = [b.download() for b in (o, dq, dk, dv)]
    assert all((y == y[:, :1]).all() for y in got)
    u = float(np.finfo(np.float64).eps) / 2
    for first, last in zip(starts[:-1], starts[1:]):
        args = [y[first:last] for y in x[:3]]
        ro, _, *rg = attention(*args, 1.0, x[3][first:last])
        eo, _, *eg = attention_bounds(*args, 1.0, 2 * u, x[3][first:last])
        for y, r, e in zip(got, [ro] + rg, [eo] + eg):
            close(y[first:last, :1], r, e, "a head")


def test_calls_of_several_threads_at_once(gpu):
    """Each with operands of its own, sharing the library's one workspace: what each gets is what it gets alone."""
    import threading
    large, short = (lambda i: Batch(np.float32, [500, 200 + i], 64, 32, 16, "fused", seed=i)), (lambda i: Batch(np.float64, [40 + i, 90], 2, 1, 32, "fused", seed=i))
    batches = [make(i) for i in range(4) for make in (large, short)]
    alone = [(b.forward(), None) for b in batches]
    alone = [(o.download(), b.backward(o, l)) for b, ((o, l), _) in zip(batches, alone)]
    wrong = []

    def run(b, want):
        for _ in range(3):
            o, l = b.forward()
            got = o.download(), b.backward(o, l)
            if not (np.array_equal(got[0], want[0], equal_nan=True) and all(np.array_equal(x, y, equal_nan=True) for x, y in zip(got[1], want[1]))):
                wrong.append(b.lengths)

    threads = [threading.Thread(target=run, args=(b, w)) for b, w in zip(batches, alone)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert wrong == []


def test_rows_behind_two_to_the_31_elements(gpu):
    """A cache of 8.6 GB, keys and values in its last rows; its rows as a table."""
    lib, cols, rows, n = _lib.load(), 1024, 2 ** 21 + 700, 650
    whole = DeviceBuffer.alloc(np.float32, rows, cols)
    end = seeded.normal(78, 1, (n, cols), 1.0, np.float32)
    whole.view_rows(rows - n, n).upload(end)
    x = seeded.normal(78, 2, (2, 128), 1.0, np.float32)
    q, o, off = dev(x), unfilled(np.float32, 2, 128), IndexVector.from_values([0, 1, 2])
    begin, last = IndexVector.from_values([rows - n, rows - 40]), IndexVector.from_values([rows - 3, rows])
    check(lib.prad_cached_attention(q.handle, 0, whole.handle, 64, whole.handle, 640, o.handle, off.handle, begin.handle, last.handle, 2, 1, 64, 0.125))
    got, u = o.download(), float(np.finfo(np.float32).eps) / 2
    for i, keys in enumerate((slice(0, n - 3), slice(n - 40, n))):
        for h in (slice(0, 64), slice(64, 128)):
            args = x[i:i + 1, h], end[keys, 64:128], end[keys, 640:704], 0.125
            close(got[i:i + 1, h], attention(*args)[0], attention_bounds(*args, 2 * u, np.zeros((1, 64)))[0], "o")
    ids, out = IndexVector.from_values([rows - 1, rows - n, rows]), unfilled(np.float32, 3, cols)
    check(lib.prad_embedding_fwd(whole.handle, ids.handle, 1.0, out.handle))
    assert np.array_equal(out.download(), np.stack([end[-1], end[0], np.zeros(cols, np.float32)]))


def test_a_workspace_that_grows_behind_a_recording(gpu):
    """A recorded call keeps the workspace of its recording when a larger eager call takes another."""
    lib, gr = _lib.load(), ctypes.c_void_p()
    small, large = (Batch(np.float32, lengths, 64, 32, d, "fused", front=0, behind=0) for lengths, d in (([300, 200], 16), ([1200, 800], 64)))
    # (the larger takes 230 MB: more than the tests above, less than the 288 MiB that another file's test grows to)
    o, l = small.forward()
    g, d = dev(small.g), unfilled(np.float32, small.rows, small.full[0])
    grads = [x for c in small.cols for x in (d.handle, c)]
    step = lambda: check(lib.prad_causal_attention_bwd(*small.operands(), o.handle, l.handle, g.handle, *grads, small.offsets.handle, *small.tail))
    step()
    want = d.download()
    check(lib.prad_graph_begin())
    try:
        step()
    finally:
        check(lib.prad_graph_end(ctypes.byref(gr)))
    first = large.backward(*large.forward())
    for _ in range(3):
        d.zero()
        check(lib.prad_graph_launch(gr))
        assert np.array_equal(d.download(), want)
        assert all(np.array_equal(x, y) for x, y in zip(large.backward(*large.forward()), first))
    check(lib.prad_graph_destroy(gr))


@DTYPES
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_cached_values_that_are_not_finite_reach_only_who_sees_them(gpu, dtype, which, value):
    args = ([3, 1, 1], [(0, 50), (60, 90), (100, 160)], 200, 2, 1, 64)
    clean = cached(dtype, *args)[0]

    def edit(q, k, v):
        x = k if which == "k" else v
        x[48, 5] = value            # the next to last key of the first sequence: its first new token does not see it
        x[50:60] = value            # between the ranges
        x[90:100] = value
        x[160:] = value

    dirty = cached(dtype, *args, edit=edit)[0]
    assert np.array_equal(dirty[2], clean[2]) and np.isnan(dirty[3:5]).all()
    assert np.array_equal(dirty[5:7], clean[5:7])


def test_cached_attention_equals_the_prompt_row_by_row(gpu):
    """Tokens fed one at a time against the growing cache give the rows of the whole prompt."""
    lib, n, heads, kv_heads, d = _lib.load(), 70, 4, 2, 64
    batch = Batch(np.float64, [n], heads, kv_heads, d, "fused", front=0, behind=0)
    want = batch.forward(lse=False)[0].download()
    q, k, v = dev(batch.q), dev(batch.k), dev(batch.v)
    o, off = unfilled(np.float64, 1, heads * d), IndexVector.from_values([0, 1])
    begin, end = IndexVector.from_values([0]), IndexVector.from_values([0])
    for i in range(n):
        end.add(1)
        one = q.view_rows(i, 1)
        check(lib.prad_cached_attention(one.handle, 0, k.handle, 0, v.handle, 0, o.handle, off.handle, begin.handle, end.handle, *batch.tail))
        assert_parity(o.download()[0], want[i], np.float64, "row %d" % i)


def test_a_recorded_step_follows_the_cache_as_it_grows(gpu):
    lib, heads, kv_heads, d, room = _lib.load(), 8, 2, 64, 600
    q = seeded.normal(51, 1, (2, heads * d), 1.0, np.float32)
    k, v = (seeded.normal(51, t, (2 * room, kv_heads * d), 1.0, np.float32) for t in (2, 3))
    bq, bk, bv, o = dev(q), dev(k), dev(v), unfilled(np.float32, 2, heads * d)
    off, begin, end = IndexVector.from_values([0, 1, 2]), IndexVector.from_values([0, room]), IndexVector.from_values([0, room])
    call = lambda: check(lib.prad_cached_attention(bq.handle, 0, bk.handle, 0, bv.handle, 0, o.handle, off.handle, begin.handle, end.handle, heads, kv_heads, d, 0.125))
    call()
    check(lib.prad_graph_begin())
    try:
        check(lib.prad_index_add(end.handle, 150))
        call()
    finally:
        gr = ctypes.c_void_p()
        check(lib.prad_graph_end(ctypes.byref(gr)))
    for turn in range(1, 5):
        check(lib.prad_graph_launch(gr))
        got = o.download()
        assert end.download().tolist() == [150 * turn, room + 150 * turn]
        o.zero()
        call()
        assert np.array_equal(got, o.download())
        h = 3
        want, _ = attention(q[1:2, h * d:h * d + d], k[room:room + 150 * turn, :d], v[room:room + 150 * turn, :d], 0.125)
        assert_parity(got[1, h * d:h * d + d], want[0], np.float32)
    check(lib.prad_graph_destroy(gr))


def test_cached_attention_refusals(gpu):
    lib = _lib.load()
    f = lambda r, c, t=np.float32: DeviceBuffer.alloc(t, r, c)
    q, k, v, o, off, one = f(3, 32), f(20, 16), f(20, 16), f(3, 32), IndexVector.from_values([0, 1, 3]), IndexVector.alloc(2)
    call = lambda q=q, k=k, v=v, o=o, off=off, b=one, e=one, d=16: lib.prad_cached_attention(
        q.handle, 0, k.handle, 0, v.handle, 0, o.handle, off.handle, b.handle, e.handle, 2, 1, d, 0.25)
    assert call() == _lib.PRAD_OK
    tall = lambda b, rows: DeviceBuffer.wrap(np.float32, rows, b.cols, b.ptr, parent=b)     # (refused before anything is read)
    assert call(q=tall(q, 2 ** 30 - 384), o=tall(o, 2 ** 30 - 384)) == _lib.PRAD_ERR_ARG
    assert call(k=tall(k, 2 ** 31), v=tall(v, 2 ** 31)) == _lib.PRAD_ERR_ARG
    for change, status in (({"v": f(21, 16)}, _lib.PRAD_ERR_SHAPE), ({"b": IndexVector.alloc(3)}, _lib.PRAD_ERR_SHAPE), ({"e": IndexVector.alloc(1)}, _lib.PRAD_ERR_SHAPE),
                           ({"e": q}, _lib.PRAD_ERR_BAD_HANDLE), ({"o": f(3, 16)}, _lib.PRAD_ERR_SHAPE), ({"o": q}, _lib.PRAD_ERR_ARG), ({"k": f(20, 8)}, _lib.PRAD_ERR_SHAPE),
                           ({"d": 200}, _lib.PRAD_ERR_ARG), ({"q": f(3, 32, np.float64)}, _lib.PRAD_ERR_DTYPE)):
        assert call(**change) == status, change


def test_key_ranges_that_describe_no_rows_do_no_harm(gpu):
    lib, k, v = _lib.load(), dev(seeded.normal(52, 1, (20, 16), 1.0, np.float32)), dev(seeded.normal(52, 2, (20, 16), 1.0, np.float32))
    q, o, off = dev(seeded.normal(52, 3, (1, 16), 1.0, np.float32)), unfilled(np.float32, 1, 16), IndexVector.from_values([0, 1])
    b, e = IndexVector.alloc(1), IndexVector.alloc(1)
    for begin, end in ((0, 1000), (-7, 20), (2 ** 31 - 1, 5), (10, 5), (-2 ** 31, 2 ** 31 - 1)):
        b.upload([begin])
        e.upload([end])
        check(lib.prad_cached_attention(q.handle, 0, k.handle, 0, v.handle, 0, o.handle, off.handle, b.handle, e.handle, 1, 1, 16, 0.25))
        got = o.download()
        assert np.isfinite(got).all()
        if begin >= end:
            assert np.all(got == 0)


@pytest.mark.parametrize("rows,heads,kv_heads,d", [(63, 1100, 1100, 2), (50, 1700, 1700, 4), (40, 6000, 6000, 1)])
def test_one_sequence_within_a_tile_of_very_many_heads(gpu, rows, heads, kv_heads, d):
    """Fewer than 64 rows of one sequence, but so many heads that the batch is computed from halves: a single tile of rows, and
    the gradients of K and V have their schedule all the same.  Heads hold one of eight values."""
    lib, few = _lib.load(), 8
    small = Batch(np.float32, [rows], few, few, d, "fused", seed=83, front=0, behind=0)
    spread = lambda x: np.tile(x, (1, -(-heads // few)))[:, :heads * d]
    q, k, v, g = (dev(spread(x)) for x in (small.q, small.k, small.v, small.g))
    o, l, dq, dk, dv = (unfilled(np.float32, *s) for s in ((rows, heads * d), (heads, rows)) + ((rows, heads * d),) * 3)
    tail = (small.offsets.handle, heads, kv_heads, d, small.scale)
    check(lib.prad_causal_attention_fwd(q.handle, 0, k.handle, 0, v.handle, 0, o.handle, l.handle, *tail))
    check(lib.prad_causal_attention_bwd(q.handle, 0, k.handle, 0, v.handle, 0, o.handle, l.handle, g.handle, dq.handle, 0, dk.handle, 0, dv.handle, 0, *tail))
    (ro, rl, *rg), (eo, el, *eg) = small.reference()
    for b, r, e, name in zip((o, dq, dk, dv), (ro, *rg), (eo, *eg), ("o", "dq", "dk", "dv")):
        got = b.download()
        assert np.array_equal(got, spread(got[:, :few * d])), name
        close(got[:, :few * d], r, e, name)
    close(l.download()[:few], rl, el, "lse")
