"""Index vectors, embedding lookup with its gradient, and dropout on the device against their definitions in 64 bits."""
import ctypes

import numpy as np
import pytest

from parallelreverseautodiff_amd import _lib, seeded
from parallelreverseautodiff_amd.exceptions import ArgumentException, InvalidOperationException, check
from parallelreverseautodiff_amd.matrix import DeviceBuffer, IndexVector
from token_reference import embedding_gradient, kept

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dtype", [np.float64, np.float32], ids=["f64", "f32"])


def dev(a):
    b = DeviceBuffer.alloc(a.dtype, *a.shape)
    b.upload(a)
    return b


_held = []


def handle_of(b):
    """The handle of a buffer made on the spot, which has to outlive the call."""
    _held.append(b)
    return b.handle


def unfilled(dtype, rows, cols):
    """A buffer full of NaN: what a call leaves unwritten shows."""
    return dev(np.full((rows, cols), np.nan, dtype))


def shifted(a):
    """The same values at an address that is a multiple of the element size only."""
    whole = DeviceBuffer.alloc(a.dtype, 1, a.size + 1)
    view = DeviceBuffer.wrap(a.dtype, a.shape[0], a.shape[1], whole.ptr + a.dtype.itemsize, parent=whole)
    view.upload(a)
    return view


# ---- index vectors ------------------------------------------------------------------------------------------------------
def test_index_vector_round_trip_and_addition(gpu):
    v = IndexVector.alloc(3)
    assert v.download().tolist() == [0, 0, 0]
    v.upload([7, -1, 2 ** 31 - 1])
    n = ctypes.c_int64()
    check(_lib.load().prad_index_length(v.handle, ctypes.byref(n)))
    assert n.value == 3
    v.add(2)
    assert v.download().tolist() == [9, 1, -2 ** 31 + 1]    # modulo 2^32
    v.add(-2)
    w = IndexVector.wrap(_lib.load().prad_index_device_ptr(v.handle) + 4, 2, parent=v)
    assert w.download().tolist() == [-1, 2 ** 31 - 1]
    big = IndexVector.from_values(np.arange(100001))
    big.add(5)
    assert np.array_equal(big.download(), np.arange(5, 100006))


def test_index_vector_refusals(gpu):
    lib = _lib.load()
    h = ctypes.c_void_p()
    for n in (0, -1, 2 ** 62):
        assert lib.prad_index_alloc(n, ctypes.byref(h)) == _lib.PRAD_ERR_ARG and not h.value
    assert lib.prad_index_wrap(1, None, ctypes.byref(h)) == _lib.PRAD_ERR_ARG
    v = IndexVector.alloc(4)
    assert lib.prad_index_wrap(1, ctypes.c_void_p(lib.prad_index_device_ptr(v.handle) + 2), ctypes.byref(h)) == _lib.PRAD_ERR_ARG
    with pytest.raises(ArgumentException):
        v.upload([1, 2, 3])
    b = DeviceBuffer.alloc(np.float32, 2, 2)
    assert lib.prad_index_add(b.handle, 1) == _lib.PRAD_ERR_BAD_HANDLE      # a matrix is no index vector
    assert lib.prad_buf_zero(v.handle) == _lib.PRAD_ERR_BAD_HANDLE          # nor the other way round
    assert lib.prad_index_free(None) == _lib.PRAD_OK
    check(lib.prad_graph_begin())
    try:
        assert lib.prad_index_alloc(4, ctypes.byref(h)) == _lib.PRAD_ERR_RECORDING
        x = np.zeros(4, np.int32)
        assert lib.prad_index_upload(v.handle, x.ctypes.data, 4) == _lib.PRAD_ERR_RECORDING
        check(lib.prad_index_add(v.handle, 1))
    finally:
        gr = ctypes.c_void_p()
        check(lib.prad_graph_end(ctypes.byref(gr)))
    check(lib.prad_graph_launch(gr))
    check(lib.prad_graph_launch(gr))
    assert v.download().tolist() == [2, 2, 2, 2]
    check(lib.prad_graph_destroy(gr))


# ---- embedding ----------------------------------------------------------------------------------------------------------
def token_ids(seed, tokens, vocab, kind):
    u = seeded.u01(seed, 1, tokens)
    if kind == "text":       # a few tokens very often
        ids = np.minimum(np.exp(u * np.log(vocab + 1)).astype(np.int64) - 1, vocab - 1)
    elif kind == "one":
        ids = np.full(tokens, vocab - 1)
    elif kind == "none":
        ids = np.where(u < 0.5, -1, vocab)
    else:
        ids = np.minimum((u * vocab).astype(np.int64), vocab - 1)
    if kind == "text" and tokens > 3:
        ids[1], ids[2], ids[tokens - 1] = -1, vocab, -2 ** 31     # outside the table on both sides
    return ids.astype(np.int32)


# (tokens, vocabulary, width, ids): one token, one row; odd widths; counts on both sides of the one-launch form (512), of a
# chunk of the sums (32), of a wavefront; more rows than one workgroup orders; one token alone; no token at all
EMBEDDINGS = [(1, 1, 1, "any"), (1, 10, 96, "any"), (49, 1000, 96, "text"), (256, 31, 4, "any"), (257, 31, 4, "any"), (257, 5, 130, "text"), (300, 2000, 7, "any"),
              (1024, 1, 260, "one"), (3000, 50, 33, "one"), (700, 1500, 64, "none"), (5000, 700, 66, "text"), (2049, 520, 256, "any"), (4096, 40000, 8, "text"),
              (6000, 270000, 4, "any"), (512, 70, 33, "text"), (512, 900, 64, "one"), (513, 70, 33, "text"), (400, 40, 8, "any")]


@DTYPES
@pytest.mark.parametrize("cfg", EMBEDDINGS, ids=str)
def test_embedding_lookup_and_gradient(gpu, dtype, cfg):
    tokens, vocab, width, kind = cfg
    lib, eps = _lib.load(), float(np.finfo(dtype).eps)
    ids = token_ids(11, tokens, vocab, kind)
    table = seeded.normal(11, 2, (vocab, width), 1.0, dtype)
    dout = seeded.normal(11, 3, (tokens, width), 1.0, dtype)
    scale = 1.7
    inside = (ids >= 0) & (ids < vocab)
    bids, out, d_table = IndexVector.from_values(ids), unfilled(dtype, tokens, width), unfilled(dtype, vocab, width)
    bt, bd = dev(table), dev(dout)
    check(lib.prad_embedding_fwd(bt.handle, bids.handle, scale, out.handle))
    want = np.where(inside[:, None], table[np.where(inside, ids, 0)].astype(np.float64) * scale, 0)
    got = out.download().astype(np.float64)
    assert np.all(np.abs(got - want) <= 1.01 * eps * np.abs(want))      # the factor and the product are rounded once each
    check(lib.prad_embedding_bwd(bd.handle, bids.handle, scale, d_table.handle, 0))
    ref, size, count = embedding_gradient(dout, ids, scale, vocab)
    got = d_table.download()
    # sums of `count` terms in double, one factor, one rounding to the element type
    bound = (count + 2) * 2.0 ** -53 * size + 0.5 * eps * np.abs(ref) + 1e-300
    assert np.all(np.abs(got.astype(np.longdouble) - ref) <= 1.01 * bound)
    again = unfilled(dtype, vocab, width)
    check(lib.prad_embedding_bwd(bd.handle, bids.handle, scale, again.handle, 0))
    assert np.array_equal(again.download(), got)                        # equal calls, equal bits
    held = seeded.normal(11, 4, (vocab, width), 1.0, dtype)
    acc = dev(held)
    check(lib.prad_embedding_bwd(bd.handle, bids.handle, scale, acc.handle, 1))
    assert np.array_equal(acc.download(), np.where(count > 0, held + got, held))


@DTYPES
@pytest.mark.parametrize("tokens", [100, 1000])
def test_embedding_at_addresses_that_are_no_multiple_of_sixteen(gpu, dtype, tokens):
    lib, vocab, width = _lib.load(), 77, 32
    ids = token_ids(12, tokens, vocab, "text")
    table, dout = seeded.normal(12, 2, (vocab, width), 1.0, dtype), seeded.normal(12, 3, (tokens, width), 1.0, dtype)
    bids, plain, odd = IndexVector.from_values(ids), [unfilled(dtype, tokens, width), unfilled(dtype, vocab, width)], \
        [shifted(np.full((tokens, width), np.nan, dtype)), shifted(np.full((vocab, width), np.nan, dtype))]
    for make, (out, d_table) in ((dev, plain), (shifted, odd)):
        bt, bd = make(table), make(dout)
        check(lib.prad_embedding_fwd(bt.handle, bids.handle, 1.0, out.handle))
        check(lib.prad_embedding_bwd(bd.handle, bids.handle, 1.0, d_table.handle, 0))
        gpu.Synchronize()
    for a, b in zip(plain, odd):
        assert np.array_equal(a.download(), b.download())


def test_embedding_refusals(gpu):
    lib = _lib.load()
    f32 = lambda r, c: DeviceBuffer.alloc(np.float32, r, c)
    table, out, ids = f32(10, 8), f32(5, 8), IndexVector.alloc(5)
    call = lambda t, i, s, o: (lib.prad_embedding_fwd(t, i, s, o), lib.prad_embedding_bwd(o, i, s, t, 0))
    assert call(table.handle, ids.handle, 1.0, handle_of(f32(5, 7))) == (_lib.PRAD_ERR_SHAPE,) * 2
    assert call(table.handle, ids.handle, 1.0, handle_of(f32(6, 8))) == (_lib.PRAD_ERR_SHAPE,) * 2
    assert call(table.handle, ids.handle, float("nan"), out.handle) == (_lib.PRAD_ERR_ARG,) * 2
    assert call(table.handle, ids.handle, 1.0, handle_of(DeviceBuffer.alloc(np.float64, 5, 8))) == (_lib.PRAD_ERR_DTYPE,) * 2
    assert call(table.handle, table.handle, 1.0, out.handle) == (_lib.PRAD_ERR_BAD_HANDLE,) * 2
    assert call(None, ids.handle, 1.0, out.handle) == (_lib.PRAD_ERR_BAD_HANDLE,) * 2
    assert call(table.handle, ids.handle, 1.0, handle_of(table.view_rows(2, 5))) == (_lib.PRAD_ERR_ARG,) * 2
    assert call(handle_of(DeviceBuffer.alloc(np.float32, 10, 8, depth=2)), ids.handle, 1.0, out.handle) == (_lib.PRAD_ERR_SHAPE,) * 2


@pytest.mark.parametrize("tokens", [400, 900])
def test_a_recorded_embedding_reads_the_ids_of_each_launch(gpu, tokens):
    lib, dtype, vocab, width = _lib.load(), np.float32, 50, 16
    table, dout = seeded.normal(13, 1, (vocab, width), 1.0, dtype), seeded.normal(13, 2, (tokens, width), 1.0, dtype)
    bt, bd, ids = dev(table), dev(dout), IndexVector.alloc(tokens)
    out, d_table = unfilled(dtype, tokens, width), unfilled(dtype, vocab, width)

    def enqueue(o, d):
        check(lib.prad_embedding_fwd(bt.handle, ids.handle, 2.0, o.handle))
        check(lib.prad_embedding_bwd(bd.handle, ids.handle, 2.0, d.handle, 0))

    enqueue(out, d_table)
    check(lib.prad_graph_begin())
    try:
        enqueue(out, d_table)
    finally:
        gr = ctypes.c_void_p()
        check(lib.prad_graph_end(ctypes.byref(gr)))
    for turn in range(4):
        ids.upload(token_ids(20 + turn, tokens, vocab, "text"))
        check(lib.prad_graph_launch(gr))
        got = out.download(), d_table.download()
        eager = unfilled(dtype, tokens, width), unfilled(dtype, vocab, width)
        enqueue(*eager)
        assert np.array_equal(got[0], eager[0].download()) and np.array_equal(got[1], eager[1].download())
    check(lib.prad_graph_destroy(gr))


# ---- dropout ------------------------------------------------------------------------------------------------------------
@DTYPES
@pytest.mark.parametrize("shape", [(1, 1), (1, 3), (49, 96), (7, 31), (513, 130), (1, 4), (300, 1000)], ids=str)
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.9999])
def test_dropout_forward_and_backward(gpu, dtype, shape, p):
    lib, eps = _lib.load(), float(np.finfo(dtype).eps)
    x, res, dy = (seeded.normal(14, t, shape, 1.0, dtype) for t in (1, 2, 3))
    seed, site, step = -0x123456789ABCDEF, 5, IndexVector.from_values([77, 1])
    keep = kept(shape, p, seed, site, 77)
    scaled = lambda a: np.where(keep, a.astype(np.float64) / (1.0 - p), 0)
    for make in (dev, shifted):
        bx, br, bdy, y, z, dx = make(x), make(res), make(dy), unfilled(dtype, *shape), unfilled(dtype, *shape), unfilled(dtype, *shape)
        check(lib.prad_dropout_fwd(bx.handle, None, y.handle, p, seed, site, step.handle))
        check(lib.prad_dropout_fwd(bx.handle, br.handle, z.handle, p, seed, site, step.handle))
        check(lib.prad_dropout_bwd(bdy.handle, dx.handle, p, seed, site, step.handle))
        # the factor 1 / (1 - p) (a subtraction and a division in double, then one rounding) and the product: two roundings of
        # the element type, two more of the double's
        per = 1.01 * eps + 2.0 ** -52
        assert np.all(np.abs(y.download() - scaled(x)) <= per * np.abs(scaled(x)))
        assert np.all(np.abs(dx.download() - scaled(dy)) <= per * np.abs(scaled(dy)))
        want = scaled(x) + res
        assert np.all(np.abs(z.download() - want) <= 1.01 * (per * np.abs(scaled(x)) + eps * np.abs(want)))
        if p == 0.0:
            assert np.array_equal(y.download(), x)


@DTYPES
def test_dropout_in_place_and_without_a_step(gpu, dtype):
    lib, shape = _lib.load(), (33, 41)
    x, res = seeded.normal(15, 1, shape, 1.0, dtype), seeded.normal(15, 2, shape, 1.0, dtype)
    out = unfilled(dtype, *shape)
    bx, br = dev(x), dev(res)
    check(lib.prad_dropout_fwd(bx.handle, br.handle, out.handle, 0.3, 9, 2, None))
    want = out.download()
    zero = IndexVector.from_values([0])
    check(lib.prad_dropout_fwd(bx.handle, br.handle, out.handle, 0.3, 9, 2, zero.handle))
    assert np.array_equal(out.download(), want)
    into_x, into_res = dev(x), dev(res)
    check(lib.prad_dropout_fwd(into_x.handle, br.handle, into_x.handle, 0.3, 9, 2, None))
    check(lib.prad_dropout_fwd(bx.handle, into_res.handle, into_res.handle, 0.3, 9, 2, None))
    assert np.array_equal(into_x.download(), want) and np.array_equal(into_res.download(), want)


def test_what_is_dropped_does_not_show(gpu):
    lib, shape, p = _lib.load(), (64, 65), 0.5
    keep = kept(shape, p, 3, 0, 0)
    x = seeded.normal(16, 1, shape, 1.0, np.float32)
    x[~keep] = np.array([np.nan, np.inf, -np.inf])[np.arange((~keep).sum()) % 3]
    bx, y = dev(x), unfilled(np.float32, *shape)
    check(lib.prad_dropout_fwd(bx.handle, None, y.handle, p, 3, 0, None))
    got = y.download()
    assert np.all(got[~keep] == 0) and np.array_equal(got[keep], x[keep] * np.float32(2))


def test_dropout_refusals(gpu):
    lib = _lib.load()
    b = lambda r=4, c=6, t=np.float32: DeviceBuffer.alloc(t, r, c)
    x, y, long = b(), b(), b(9)
    fwd = lambda x, r, y, p=0.1, step=None: lib.prad_dropout_fwd(x, r, y, p, 1, 0, step)
    for p in (1.0, -0.1, 1.5, float("nan")):
        assert fwd(x.handle, None, y.handle, p) == _lib.PRAD_ERR_ARG and lib.prad_dropout_bwd(x.handle, y.handle, p, 1, 0, None) == _lib.PRAD_ERR_ARG
    assert fwd(x.handle, None, handle_of(b(4, 5))) == _lib.PRAD_ERR_ARG
    assert fwd(x.handle, handle_of(b(5, 6)), y.handle) == _lib.PRAD_ERR_ARG
    assert fwd(x.handle, None, handle_of(b(4, 6, np.float64))) == _lib.PRAD_ERR_DTYPE
    assert fwd(handle_of(long.view_rows(0, 4)), None, handle_of(long.view_rows(2, 4))) == _lib.PRAD_ERR_ARG
    assert fwd(x.handle, None, y.handle, 0.1, x.handle) == _lib.PRAD_ERR_BAD_HANDLE
    assert fwd(None, None, y.handle) == _lib.PRAD_ERR_BAD_HANDLE


def test_a_recorded_dropout_draws_another_mask_at_every_launch(gpu):
    lib, shape, p = _lib.load(), (100, 37), 0.25
    x, dy = (seeded.normal(17, t, shape, 1.0, np.float64) for t in (1, 2))
    step = IndexVector.from_values([5])
    bx, bdy, y, dx = dev(x), dev(dy), unfilled(np.float64, *shape), unfilled(np.float64, *shape)
    check(lib.prad_graph_begin())
    try:
        check(lib.prad_dropout_fwd(bx.handle, None, y.handle, p, 1, 0, step.handle))
        check(lib.prad_dropout_bwd(bdy.handle, dx.handle, p, 1, 0, step.handle))
        check(lib.prad_index_add(step.handle, 1))
    finally:
        gr = ctypes.c_void_p()
        check(lib.prad_graph_end(ctypes.byref(gr)))
    for turn in range(4):
        check(lib.prad_graph_launch(gr))
        keep = kept(shape, p, 1, 0, 5 + turn)
        assert np.array_equal(y.download() != 0, keep) and np.array_equal(dx.download() != 0, keep)
    assert step.download().tolist() == [9]
    check(lib.prad_graph_destroy(gr))


def test_another_thread_is_refused_while_one_records(gpu):
    import threading
    lib = _lib.load()
    v, x, y = IndexVector.alloc(4), DeviceBuffer.alloc(np.float32, 4, 4), DeviceBuffer.alloc(np.float32, 4, 4)
    seen = []
    check(lib.prad_graph_begin())
    try:
        t = threading.Thread(target=lambda: seen.extend([lib.prad_index_add(v.handle, 1), lib.prad_dropout_fwd(x.handle, None, y.handle, 0.1, 1, 0, None),
                                                         lib.prad_embedding_fwd(x.handle, v.handle, 1.0, y.handle)]))
        t.start()
        t.join()
        check(lib.prad_index_add(v.handle, 1))
    finally:
        gr = ctypes.c_void_p()
        check(lib.prad_graph_end(ctypes.byref(gr)))
    assert seen == [_lib.PRAD_ERR_RECORDING] * 3
    check(lib.prad_graph_destroy(gr))
    with pytest.raises(InvalidOperationException):
        check(_lib.PRAD_ERR_RECORDING)


@pytest.mark.parametrize("tokens", [1, 5, 512, 600])
def test_gradient_of_a_table_of_very_many_rows(gpu, tokens):
    """More than 2^26 rows, whatever the number of tokens."""
    lib, vocab = _lib.load(), 2 ** 26 + 1000
    ids = np.array([vocab - 1, 0, vocab - 1, -1, 2 ** 26 - 1] * (tokens // 5 + 1), np.int64)[:tokens]
    dout = seeded.normal(19, 1, (tokens, 1), 1.0, np.float32)
    bd, bi, d_table = dev(dout), IndexVector.from_values(ids), DeviceBuffer.alloc_output(np.float32, vocab, 1)
    check(lib.prad_embedding_bwd(bd.handle, bi.handle, 0.5, d_table.handle, 0))
    flat = DeviceBuffer.wrap(np.float32, 1, vocab, d_table.ptr, parent=d_table)      # (one row: a download goes row by row)
    got = flat.download()[0]
    want = np.zeros(vocab, np.float32)
    for r in set(ids[ids >= 0].tolist()):       # (sums in double, rounded once)
        want[r] = np.float32(dout[ids == r, 0].astype(np.float64).sum() * 0.5)
    assert np.allclose(got, want, rtol=2.0 ** -23, atol=0)
    check(lib.prad_embedding_bwd(bd.handle, bi.handle, 0.5, d_table.handle, 1))
    assert np.allclose(flat.download()[0], 2 * want, rtol=2.0 ** -22, atol=0)


@DTYPES
def test_a_scale_that_the_element_type_does_not_hold(gpu, dtype):
    """1e39 is a number in double and infinite in float."""
    lib, wanted = _lib.load(), _lib.PRAD_OK if dtype == np.float64 else _lib.PRAD_ERR_ARG
    table, out, ids = DeviceBuffer.alloc(dtype, 10, 8), DeviceBuffer.alloc(dtype, 5, 8), IndexVector.alloc(5)
    assert lib.prad_embedding_fwd(table.handle, ids.handle, 1e39, out.handle) == wanted
    assert lib.prad_embedding_bwd(out.handle, ids.handle, 1e39, table.handle, 0) == wanted
    x, o, lse, dx = (DeviceBuffer.alloc(dtype, r, c) for r, c in ((5, 24), (5, 8), (2, 5), (5, 24)))
    off, begin, end = IndexVector.from_values([0, 5]), IndexVector.alloc(1), IndexVector.from_values([5])
    qkv = x.handle, 0, x.handle, 8, x.handle, 16
    for scale, status in ((1e39, wanted), (-1e39, wanted), (1e300, wanted), (1e38, _lib.PRAD_OK), (float("inf"), _lib.PRAD_ERR_ARG)):
        assert lib.prad_causal_attention_fwd(*qkv, o.handle, lse.handle, off.handle, 2, 2, 4, scale) == status
        assert lib.prad_causal_attention_bwd(*qkv, o.handle, lse.handle, o.handle, dx.handle, 0, dx.handle, 8, dx.handle, 16, off.handle, 2, 2, 4, scale) == status
        assert lib.prad_cached_attention(*qkv, o.handle, off.handle, begin.handle, end.handle, 2, 2, 4, scale) == status
