"""The operators of a token model together, as a training step and a generation loop use them: through the operation classes
against the same model written down in numpy in 64 bits, and recorded as a launch sequence against the same calls made one by one."""
import ctypes

import numpy as np
import pytest

from parallelreverseautodiff_amd import _lib, seeded
from parallelreverseautodiff_amd.exceptions import ArgumentException, InvalidOperationException, check
from parallelreverseautodiff_amd.matrix import DeviceBuffer, IndexVector, Matrix
from parallelreverseautodiff_amd.operations import (CachedAttentionOperation, CategoricalCrossEntropyLossOperation, CausalAttentionOperation,
                                                    DropoutOperation, EmbeddingOperation, MatrixAddOperation, MatrixMultiplyOperation,
                                                    SoftmaxOperation, TanhOperation, accumulate_gradient, handle_array)
from token_reference import attention, kept

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dtype", [np.float64, np.float32], ids=["f64", "f32"])
VOCAB, HEADS, KV, D, HIDDEN = 29, 4, 2, 12, 40
WIDTH = HEADS * D
LENGTHS = [17, 0, 1, 34, 9]
P, SEED, SITE = 0.25, 77, 3
NAMES = ("table", "wq", "wk", "wv", "wo", "w1", "w2")
SHAPES = ((VOCAB, WIDTH), (WIDTH, WIDTH), (WIDTH, KV * D), (WIDTH, KV * D), (WIDTH, WIDTH), (WIDTH, HIDDEN), (HIDDEN, VOCAB))


def problem(dtype, seed=5):
    tokens = sum(LENGTHS)
    w = {n: seeded.normal(seed, i, s, s[0] ** -0.5 if n != "table" else 1.0, dtype) for i, (n, s) in enumerate(zip(NAMES, SHAPES))}
    ids = np.arange(tokens) * 7 % (VOCAB + 2) - 1            # (-1 and VOCAB stand for no token)
    target = np.zeros((tokens, VOCAB), dtype)
    target[np.arange(tokens), np.arange(tokens) * 11 % VOCAB] = 1
    return w, ids, np.concatenate([[0], np.cumsum(LENGTHS)]), target


def reference(w, ids, offsets, target, step):
    """The loss and the gradients of all weights."""
    w = {n: np.asarray(x, np.float64) for n, x in w.items()}
    tokens, there = len(ids), (ids >= 0) & (ids < VOCAB)
    x = np.where(there[:, None], w["table"][np.clip(ids, 0, VOCAB - 1)], 0.0)
    q, k, v = x @ w["wq"], x @ w["wk"], x @ w["wv"]
    mask = kept((tokens, WIDTH), P, SEED, SITE, step) / (1 - P)

    def heads(g=None):
        o, d = np.zeros_like(q), (np.zeros_like(q), np.zeros_like(k), np.zeros_like(v))
        for a, b in zip(offsets[:-1], offsets[1:]):
            for h in range(HEADS):
                c, s = slice(h * D, h * D + D), slice(h // (HEADS // KV) * D, h // (HEADS // KV) * D + D)
                got = attention(q[a:b, c], k[a:b, s], v[a:b, s], D ** -0.5, None if g is None else g[a:b, c])
                o[a:b, c] = got[0]
                if g is not None:
                    d[0][a:b, c] = got[2]
                    d[1][a:b, s] += got[3]
                    d[2][a:b, s] += got[4]
        return o, d

    o, _ = heads()
    h = (o @ w["wo"]) * mask + x
    y = np.tanh(h @ w["w1"])
    z = y @ w["w2"]
    e = np.exp(z - z.max(axis=1, keepdims=True))
    p = e / e.sum(axis=1, keepdims=True)
    loss = -(target * np.log(p + 1e-15)).sum() / tokens
    dz = (p - target) / tokens
    dy = (dz @ w["w2"].T) * (1 - y * y)
    dh = dy @ w["w1"].T
    do = (dh * mask) @ w["wo"].T
    _, (dq, dk, dv) = heads(do)
    dx = dh + dq @ w["wq"].T + dk @ w["wk"].T + dv @ w["wv"].T
    dtable = np.zeros_like(w["table"])
    np.add.at(dtable, ids[there], dx[there])
    return loss, {"table": dtable, "wq": x.T @ dq, "wk": x.T @ dk, "wv": x.T @ dv, "wo": o.T @ (dh * mask), "w1": h.T @ dy, "w2": y.T @ dz}


class Net:
    """The model of `reference` out of operations."""

    def __init__(self):
        self.embed, self.attend, self.drop = EmbeddingOperation(), CausalAttentionOperation(HEADS, KV), DropoutOperation(P, SEED, SITE)
        self.mm = {n: MatrixMultiplyOperation() for n in NAMES[1:]}
        self.tanh, self.softmax, self.loss = TanhOperation(), SoftmaxOperation(), CategoricalCrossEntropyLossOperation()

    def forward(self, w, ids, offsets, target, step):
        x = self.embed.Forward(w["table"], ids)
        q, k, v = (self.mm[n].Forward(x, w[n]) for n in ("wq", "wk", "wv"))
        o = self.mm["wo"].Forward(self.attend.Forward(q, k, v, offsets), w["wo"])
        y = self.tanh.Forward(self.mm["w1"].Forward(self.drop.Forward(o, x, step), w["w1"]))
        self.p = self.softmax.Forward(self.mm["w2"].Forward(y, w["w2"]))
        return self.loss.Forward(self.p, target)

    def backward(self):
        g = {}
        d = self.softmax.Backward(self.loss.Backward(self.p).Item1).Item1
        d, g["w2"] = self.mm["w2"].Backward(d).Results
        d, g["w1"] = self.mm["w1"].Backward(self.tanh.Backward(d).Item1).Results
        d, dx = self.drop.Backward(d).Results
        d, g["wo"] = self.mm["wo"].Backward(d).Results
        for n, d in zip(("wq", "wk", "wv"), self.attend.Backward(d).Results):
            d, g[n] = self.mm[n].Backward(d).Results
            accumulate_gradient(dx, d)
        g["table"] = self.embed.Backward(dx).Item1
        return g


def near(got, want, dtype, what):
    """Some twelve operations in series, forward and backward; a product over at most 48 values of a size is off by at most
    (48 + 8) u of it in norm, and nothing here cancels in norm: 12 * 56 u, with half as much again for the norms of products, is
    1000 u = 500 eps."""
    off = np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want)
    assert off <= 512 * float(np.finfo(dtype).eps), "%s: off by %.3g in norm" % (what, off)


@DTYPES
def test_a_training_step_out_of_operations(gpu, dtype):
    w, ids, offsets, target = problem(dtype)
    net, step = Net(), IndexVector.from_values([4])
    m = {n: Matrix.from_numpy(x) for n, x in w.items()}
    loss = net.forward(m, ids, offsets, Matrix.from_numpy(target), step)
    grads = net.backward()
    want_loss, want = reference(w, ids, offsets, target, 4)
    near(loss.to_numpy(), np.array([[want_loss]]), dtype, "loss")
    for n in NAMES:
        near(grads[n].to_numpy(), want[n], dtype, n)


def test_gradients_of_a_training_step_against_differences(gpu):
    """Central differences of the loss along one direction of all weights: off by about h^2 of the third derivative and
    eps / h of the loss, 1e-9 together at h = 1e-5."""
    w, ids, offsets, target = problem(np.float64)
    direction = {n: seeded.normal(9, i, w[n].shape, 0.1, np.float64) for i, n in enumerate(NAMES)}
    net, goal = Net(), Matrix.from_numpy(target)
    ids, offsets, step = IndexVector.from_values(ids), IndexVector.from_values(offsets), IndexVector.from_values([2])

    def at(h):
        return float(net.forward({n: Matrix.from_numpy(w[n] + h * direction[n]) for n in NAMES}, ids, offsets, goal, step).to_numpy()[0, 0])

    difference = (at(1e-5) - at(-1e-5)) / 2e-5
    at(0.0)
    slope = sum(float((g.to_numpy() * direction[n]).sum()) for n, g in net.backward().items())
    assert abs(slope) > 1e-3 and abs(difference - slope) <= 1e-7 * max(1.0, abs(slope))


def test_operations_keep_what_backward_needs_for_each_id(gpu):
    """Store and Restore: two samples forward, both backward, as a net with several steps does."""
    w, ids, offsets, _ = problem(np.float64)
    table, attend, embed = Matrix.from_numpy(w["table"]), CausalAttentionOperation(HEADS, HEADS), EmbeddingOperation(2.0)
    drop = DropoutOperation(0.5, 1, 2)
    want, grad = [], Matrix.from_numpy(seeded.normal(3, 3, (len(ids), WIDTH), 1.0, np.float64))
    for i in (0, 1):
        x = embed.Forward(table, np.roll(ids, i))
        attend.Forward(x, x, x, offsets)
        drop.Forward(x, None, [i])
        for op in (embed, attend, drop):
            op.Store(i)
        want.append([r.to_numpy() for op in (embed, attend, drop) for r in op.Backward(grad).Results])
    for i in (0, 1):
        for op in (embed, attend, drop):
            op.Restore(i)
        again = [r.to_numpy() for op in (embed, attend, drop) for r in op.Backward(grad).Results]
        assert len(again) == 5 and all(np.array_equal(a, b) for a, b in zip(again, want[i]))
    assert not np.array_equal(want[0][0], want[1][0]) and not np.array_equal(want[0][4], want[1][4])


def test_operations_refuse(gpu):
    w, ids, offsets, _ = problem(np.float64)
    x = EmbeddingOperation().Forward(Matrix.from_numpy(w["table"]), ids)
    with pytest.raises(ArgumentException):
        CausalAttentionOperation(5).Forward(x, x, x, offsets)
    with pytest.raises(ArgumentException):
        CausalAttentionOperation(0).Forward(x, x, x, offsets)
    for op in (CausalAttentionOperation(HEADS, 3), CausalAttentionOperation(HEADS, 2), CausalAttentionOperation(HEADS, HEADS, float("nan"))):
        with pytest.raises((ArgumentException, InvalidOperationException)):
            op.Forward(x, x, x, offsets)
    with pytest.raises((ArgumentException, InvalidOperationException)):
        DropoutOperation(1.0).Forward(x)
    with pytest.raises(ArgumentException):
        EmbeddingOperation().Forward(Matrix.from_numpy(w["table"]), [0.5])
    with pytest.raises(InvalidOperationException):
        CachedAttentionOperation(HEADS).Backward(x)


@DTYPES
def test_generating_token_by_token_gives_the_prompts_rows(gpu, dtype):
    """Two texts continued at the same time against one cache: what each step gives is the row of the whole text's attention.
    Both are within their own rounding of the definition: two of the bars above."""
    rows, lengths = 40, (23, 11)
    q, k, v = (Matrix.from_numpy(seeded.normal(8, i, (rows, n * D), 1.0, dtype)) for i, n in enumerate((HEADS, KV, KV)))
    whole = CausalAttentionOperation(HEADS, KV).Forward(q, k, v, [0, 23, 34]).to_numpy()
    step = CachedAttentionOperation(HEADS, KV)
    for t in range(11):
        now = Matrix.from_numpy(q.to_numpy()[[t, 23 + t]])
        got = step.Forward(now, k, v, [0, 1, 2], [0, 23], [t + 1, 23 + t + 1]).to_numpy()
        near(got, whole[[t, 23 + t]].astype(np.float64), dtype, "step %d" % t)
    assert not whole[34:].any()


class Recorded:
    """The same step on buffers that stay, with clipping and Adam, for recording."""

    def __init__(self, dtype, layout_tokens):
        self.dtype, n = dtype, layout_tokens
        w, ids, offsets, target = problem(dtype)
        make = lambda r, c: DeviceBuffer.alloc(dtype, r, c)
        self.w = {name: make(*s) for name, s in zip(NAMES, SHAPES)}
        for name in NAMES:
            self.w[name].upload(w[name])
        self.g, self.m, self.v = ({name: make(*s) for name, s in zip(NAMES, SHAPES)} for _ in range(3))
        self.ids, self.offsets, self.step = IndexVector.from_values(ids), IndexVector.from_values(offsets), IndexVector.alloc(1)
        self.target = make(n, VOCAB)
        self.target.upload(target)
        self.x, self.o, self.wo, self.h, self.dx, self.dwo, self.do = (make(n, WIDTH) for _ in range(7))
        self.y, self.dy, self.dh1 = (make(n, HIDDEN) for _ in range(3))
        self.q, self.dq = make(n, WIDTH), make(n, WIDTH)
        self.k, self.v_, self.dk, self.dv = (make(n, KV * D) for _ in range(4))
        self.z, self.p, self.dp, self.dz = (make(n, VOCAB) for _ in range(4))
        self.lse, self.loss = make(HEADS, n), make(1, 1)

    def enqueue(self, iteration):
        lib, h, w, g = _lib.load(), lambda b: b.handle, self.w, self.g
        heads = (HEADS, KV, D, D ** -0.5)
        check(lib.prad_embedding_fwd(h(w["table"]), h(self.ids), 1.0, h(self.x)))
        for name, to in (("wq", self.q), ("wk", self.k), ("wv", self.v_)):
            check(lib.prad_matmul_fwd(h(self.x), h(w[name]), h(to)))
        qkv = (h(self.q), 0, h(self.k), 0, h(self.v_), 0)
        check(lib.prad_causal_attention_fwd(*qkv, h(self.o), h(self.lse), h(self.offsets), *heads))
        check(lib.prad_matmul_fwd(h(self.o), h(w["wo"]), h(self.wo)))
        check(lib.prad_dropout_fwd(h(self.wo), h(self.x), h(self.h), P, SEED, SITE, h(self.step)))
        check(lib.prad_matmul_fwd_fused(h(self.h), h(w["w1"]), None, None, h(self.y), _lib.ACT_TANH, 0.0))
        check(lib.prad_matmul_fwd(h(self.y), h(w["w2"]), h(self.z)))
        check(lib.prad_softmax_cce(h(self.z), h(self.target), h(self.p), h(self.loss), h(self.dp), h(self.dz)))
        check(lib.prad_matmul_bwd(h(self.dz), h(self.y), h(w["w2"]), h(self.dy), h(g["w2"]), 0, 0))
        check(lib.prad_act_bwd(_lib.ACT_TANH, h(self.y), h(self.dy), h(self.dh1), 0.0))
        check(lib.prad_matmul_bwd(h(self.dh1), h(self.h), h(w["w1"]), h(self.dx), h(g["w1"]), 0, 0))
        check(lib.prad_dropout_bwd(h(self.dx), h(self.dwo), P, SEED, SITE, h(self.step)))
        check(lib.prad_matmul_bwd(h(self.dwo), h(self.o), h(w["wo"]), h(self.do), h(g["wo"]), 0, 0))
        check(lib.prad_causal_attention_bwd(*qkv, h(self.o), h(self.lse), h(self.do), h(self.dq), 0, h(self.dk), 0, h(self.dv), 0, h(self.offsets), *heads))
        for name, d in (("wq", self.dq), ("wk", self.dk), ("wv", self.dv)):
            check(lib.prad_matmul_bwd(h(d), h(self.x), h(w[name]), h(self.dx), h(g[name]), 1, 0))
        check(lib.prad_embedding_bwd(h(self.dx), h(self.ids), 1.0, h(g["table"]), 0))
        all_of = lambda d: handle_array([d[name] for name in NAMES])
        check(lib.prad_clip_multi(all_of(g), len(NAMES), 4.0, 1e-12))
        check(lib.prad_adam_multi(all_of(w), all_of(self.m), all_of(self.v), all_of(g), len(NAMES), 1e-3, 0.9, 0.999, 1e-8, float(iteration)))
        check(lib.prad_index_add(h(self.step), 1))

    def state(self):
        return [self.loss.download()] + [self.w[n].download() for n in NAMES]


@DTYPES
def test_a_recorded_training_step_equals_the_calls_one_by_one(gpu, dtype):
    """Replays with other tokens, other lengths and other masks at every launch."""
    tokens = sum(LENGTHS)
    one, two = Recorded(dtype, tokens), Recorded(dtype, tokens)
    lib, gr = _lib.load(), ctypes.c_void_p()
    for both in (one, two):
        both.enqueue(1)                     # (workspaces grow outside the recording)
    check(lib.prad_graph_begin())
    try:
        two.enqueue(2)
    finally:
        check(lib.prad_graph_end(ctypes.byref(gr)))
    losses = set()
    for i, lengths in enumerate(([17, 0, 1, 34, 9], [61, 0, 0, 0, 0], [5, 20, 20, 15, 1], [0, 0, 30, 0, 31])):
        for both in (one, two):
            both.ids.upload((np.arange(tokens) * (3 + 2 * i) + i) % VOCAB)
            both.offsets.upload(np.concatenate([[0], np.cumsum(lengths)]))
        one.enqueue(2 + i)
        check(lib.prad_graph_launch(gr))
        a, b = one.state(), two.state()
        assert all(np.array_equal(x, y) for x, y in zip(a, b)), "launch %d" % i
        assert all(np.isfinite(x).all() for x in a)
        losses.add(float(a[0][0, 0]))
    assert len(losses) == 4 and one.step.download()[0] == two.step.download()[0] == 5
    check(lib.prad_graph_destroy(gr))
