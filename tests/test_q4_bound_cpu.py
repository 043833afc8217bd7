"""The bound that the 4-bit attention is held to rejects outputs that lack the tail of the weights."""
import math

import numpy as np
import pytest

from oracle import q4

D, BS = 128, 16


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
