"""The bound that the 4-bit attention is held to rejects outputs that lack pages or the tail of the weights."""
import math

import numpy as np
import pytest

from oracle import q4

D, BS = 128, 16


def case(rng, n, values):
    K = rng.standard_normal((n // BS, 1, BS, D)).astype(np.float16)
    pages = q4.fill_pages(K, values.reshape(n // BS, BS, 1, D).transpose(0, 2, 1, 3).astype(np.float16), 32)[:, None]
    return rng.standard_normal((1, 2, D)).astype(np.float16), pages, np.arange(n // BS)[None], [n]


def without(q, pages, table, lens, lost):
    """The output over all pages but the lost ones."""
    kept = np.setdiff1d(table[0], lost)
    return q4.attention(q, pages, kept[None], [len(kept) * BS], 0, 1 / math.sqrt(D), 32)[0]


@pytest.mark.parametrize("n", [8960, 40000])
def test_a_hundredth_of_the_pages_lost_is_seen(n):
    rng = np.random.default_rng(n)
    values = np.zeros((n, D))
    values[np.arange(n), np.arange(n) // BS * D // (n // BS)] = 1  # page i shows in channel 128 i / pages
    q, pages, table, lens = case(rng, n, values)
    want, tol = q4.attention_bound(q, pages, table, lens, 0, 1 / math.sqrt(D), 32)
    assert (np.abs(want.astype(np.float16) - want) <= tol).all() and not (np.abs(want) <= tol).all()
    few = n // BS // 100
    for at in (0, n // BS // 2, n // BS - few):
        assert (np.abs(without(q, pages, table, lens, np.arange(at, at + few)) - want).max() > 10 * tol.max()).all()
    lone = without(q, pages, table, lens, [3])
    assert (np.abs(lone - want) > tol).any()


def test_random_values_show_a_lost_quarter():
    rng = np.random.default_rng(1)
    n = 40000
    q, pages, table, lens = case(rng, n, rng.standard_normal((n, D)))
    want, tol = q4.attention_bound(q, pages, table, lens, 0, 1 / math.sqrt(D), 32)
    for lost in (np.arange(n // BS * 3 // 4, n // BS), np.arange(n // BS // 100)):
        assert (np.abs(without(q, pages, table, lens, lost) - want) / tol).max() > 1
    assert (np.abs(want) / tol).max() > 5


@pytest.mark.parametrize("below", [23.5, 25.2])
def test_a_lost_tail_is_seen(below):
    """One key with the weight and a value of zero; the others, 2^-below of it each with values of one, are the output. fp16 weights up to one
    drop what is below 2^-25 and round what is near 2^-24."""
    n = 40000
    K, V = np.zeros((n // BS, 1, BS, D), np.float16), np.ones((n // BS, 1, BS, D), np.float16)
    K[0, 0, 0, 0], V[0, 0, 0] = 4, 0
    q = np.zeros((1, 1, D), np.float16)
    q[0, 0, 0] = below * math.log(2) * math.sqrt(D) / 4
    pages = q4.fill_pages(K, V, 32)[:, None]
    want, tol = q4.attention_bound(q, pages, np.arange(n // BS)[None], [n], 0, 1 / math.sqrt(D), 32)
    w = np.exp(-float(q[0, 0, 0]) * 4 / math.sqrt(D))
    high = np.float16(w)
    held = float(high) + float(np.float16(w - float(high)))
    lost = (n - 1) * held / (1 + (n - 1) * w)
    assert (np.abs(lost - want) > tol).all()
    assert (np.abs(want.astype(np.float16) - want) <= tol).all()
