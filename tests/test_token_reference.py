"""The numpy statements the token model's device tests compare with, pinned by something other than themselves; and what
the host side refuses before it reaches the library."""
import numpy as np
import pytest

from parallelreverseautodiff_amd.exceptions import ArgumentException
from parallelreverseautodiff_amd.matrix import IndexVector
from token_reference import attention, embedding_gradient, kept, philox4x32


def test_generator_gives_the_published_answers():
    """Known answers of Philox4x32-10 (the authors' test vectors)."""
    ones = 0xFFFFFFFF
    for counter, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((ones,) * 4, (ones,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        got = philox4x32([np.array([x]) for x in counter], key)
        assert tuple(int(w[0]) for w in got) == want


def test_kept_share_and_independence_of_places():
    p, n = 0.3, 1 << 18
    masks = [kept((n,), p, seed, site, step) for seed, site, step in ((1, 0, 0), (2, 0, 0), (1, 1, 0), (1, 0, 1))]
    spread = np.sqrt(p * (1 - p) / n)
    for m in masks:
        assert abs(m.mean() - (1 - p)) < 6 * spread
    for other in masks[1:]:
        both = (masks[0] & other).mean()
        assert abs(both - (1 - p) ** 2) < 6 * np.sqrt((1 - p) ** 2 / n)
    assert kept((5, 7), 0.0, 9, 9, 9).all()


@pytest.mark.parametrize("n,m", [(5, 5), (3, 9), (1, 4), (6, 4)])
def test_attention_gradients_against_differences(n, m):
    rng = np.random.default_rng(3)
    q, k, v, g = rng.normal(size=(n, 4)), rng.normal(size=(m, 4)), rng.normal(size=(m, 4)), rng.normal(size=(n, 4))
    o, lse, *grads = attention(q, k, v, 0.6, g)
    if n > m:
        assert np.all(o[:n - m] == 0) and np.all(lse[:n - m] == -np.inf)
    h = 1e-5
    for which, grad in zip((q, k, v), grads):
        for at in np.ndindex(which.shape):
            old = which[at]
            which[at] = old + h
            up = np.sum(attention(q, k, v, 0.6)[0] * g)
            which[at] = old - h
            down = np.sum(attention(q, k, v, 0.6)[0] * g)
            which[at] = old
            assert abs((up - down) / (2 * h) - grad[at]) < 1e-8   # truncation h^2 and cancellation eps / h, both 1e-10


def test_embedding_gradient_against_differences():
    rng = np.random.default_rng(4)
    ids = np.array([2, 0, 2, -1, 5, 2])
    g = rng.normal(size=(6, 3))
    grad, size, count = embedding_gradient(g, ids, 1.5, 5)   # (id 5 lies outside)
    table = rng.normal(size=(5, 3))
    loss = lambda t: sum(float(1.5 * t[r] @ g[i]) for i, r in enumerate(ids) if 0 <= r < 5)
    for at in np.ndindex(table.shape):
        up, down = table.copy(), table.copy()
        up[at] += 0.5
        down[at] -= 0.5
        assert abs((loss(up) - loss(down)) - float(grad[at])) < 1e-12   # (linear: no truncation)
    assert count[:, 0].tolist() == [1, 0, 3, 0, 0]


@pytest.mark.parametrize("values", [[], [0.5], [2 ** 31], [-2 ** 31 - 1]])
def test_index_values_are_whole_numbers_of_32_bits(values):
    with pytest.raises(ArgumentException):
        IndexVector._as_int32(values)


def test_index_values_are_taken_as_they_are():
    got = IndexVector._as_int32(np.array([[3, -1], [2 ** 31 - 1, -2 ** 31]], np.int64))
    assert got.dtype == np.int32 and got.tolist() == [3, -1, 2 ** 31 - 1, -2 ** 31]
