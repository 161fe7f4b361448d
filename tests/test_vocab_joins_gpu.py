"""The log sum of a row of many classes, all of whose logits are around 1000: joining the parts of a row adds no error of its own."""
import numpy as np
import pytest

import test_vocab_gpu as vocab
from langhelp import *

pytestmark = pytest.mark.gpu


def common_part():
    """A multiple of 1/64 below 1024 whose product with log2 e is rounded by nearly half a step of float32, and values of a few bits that add up to it."""
    steps = np.arange(62000, 65536)
    product = (steps / 64.0) * np.float64(np.float32(1.44269504088896341))
    off = np.abs(product - product.astype(np.float32).astype(np.float64))
    best = int(steps[np.argmax(off)])
    return best / 64.0, off.max(), [2.0 ** (bit - 6) for bit in range(16) if best >> bit & 1]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=NAMES.get)
@pytest.mark.parametrize("tied", [False, True], ids=["rows", "transposed"])
@pytest.mark.parametrize("rows,classes", [(16, 32768), (64, 9000), (300, 50000), (2000, 20000)])
def test_logits_around_a_thousand(rows, classes, tied, dtype):
    rng = np.random.default_rng(classes)
    most, off, parts = common_part()
    k = 64
    v = np.zeros((k, classes))
    v[:len(parts)] = np.array(parts)[:, None]
    v[-1] = -rng.integers(0, 8, classes) / 8.0                   # (every logit is a multiple of 1/64 below 1024: exact in float32, whatever the order of its sum)
    w = Operand(v, dtype, 1, k) if tied else Operand(v, dtype)
    x, targets = Operand(np.ones((rows, k)), dtype), rng.integers(0, classes, rows)
    z = v.sum(0)
    want = most + np.log(np.exp(z - most).sum())
    _, stats = vocab.forward(x, w, None, targets, dtype, 1)
    got = stats.read()[0, :rows]
    # once the rounding of a tile's largest value times log2 e; the result's own; sums of fewer than 300 one after the other, a dozen roundings of exponentials, their arguments and the logarithm
    bound = off * np.log(2.0) + 2.0 ** -24 * abs(want) + 2.0 ** -24 * 320
    assert np.abs(got - want).max() <= bound, (np.abs(got - want).max(), bound)
