"""The loss of a vocabulary of fewer classes than a 16-byte vector, as rows and as a transposed view, against the formulas in 64 bits."""
import pytest

import test_vocab_gpu as vocab
from langhelp import ALL, NAMES

pytestmark = pytest.mark.gpu
SIZES = [(20, 64, 3), (300, 72, 7), (1, 4096, 1), (257, 520, 5), (2000, 256, 2), (64, 128, 8)]


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("tied", [False, True], ids=["rows", "transposed"])
@pytest.mark.parametrize("rows,k,classes", SIZES)
def test_forward(rows, k, classes, tied, dtype):
    vocab.test_forward(rows, k, classes, tied, dtype)


@pytest.mark.parametrize("dtype", ALL, ids=NAMES.get)
@pytest.mark.parametrize("tied", [False, True], ids=["rows", "transposed"])
@pytest.mark.parametrize("reduction", [0, 1])
@pytest.mark.parametrize("rows,k,classes", SIZES)
def test_backward(rows, k, classes, reduction, tied, dtype):
    vocab.check_backward(rows, k, classes, tied, dtype, reduction, bias=classes % 2 == 1)
