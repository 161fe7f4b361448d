"""What the loss of a large vocabulary asks for as its workspace (no GPU needed)."""
import pytest

from recpulse_amd import capi

MIB = 1 << 20
HALF = [capi.F16, capi.BF16]
# few rows before many classes, where W is by far the largest thing in the call
FEW = [(1, 4096, 128256), (16, 4096, 131072), (64, 4096, 32768), (7, 8192, 256000), (64, 16384, 1000), (1, 100000, 3000)]


def workspace(rows, k, classes, backward, dtype):
    return capi.lib().rp_hip_linear_cross_entropy_workspace(rows, k, classes, backward, dtype)


def strided(rows, k, classes, backward, strides, dtype):
    return capi.lib().rp_hip_linear_cross_entropy_workspace_strided(rows, k, classes, backward, *strides, dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,k,classes", FEW)
def test_a_piece_is_bounded_whatever_is_widened(rows, k, classes, dtype):
    """64 MiB of logits and 16 of partial sums; up to 128 of W, or 256 columns of it, and as much of dW; x and dx; sums of shares."""
    piece = max(128 * MIB, 256 * k * 4)
    assert 0 < workspace(rows, k, classes, 0, dtype) <= (64 + 16 + 1) * MIB + piece + 4 * rows * k
    assert 0 < workspace(rows, k, classes, 1, dtype) <= (64 + 32 + 2) * MIB + 2 * piece + 8 * rows * k


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,k,classes", FEW)
def test_operands_with_unit_strides_take_less_than_their_logits(rows, k, classes, dtype):
    logits = 2 * rows * classes
    for strides in ((k, 1, classes, 1), (k, 1, 1, k), (k + 8, 1, classes + 8, 1)):
        assert 0 < strided(rows, k, classes, 0, strides, dtype) < logits + 4096
        # backward: their gradient in columns of whole tiles, the sums of its columns by 32 rows, and two lots of sums of shares, 32 MiB each
        assert 0 < strided(rows, k, classes, 1, strides, dtype) < (2 * rows + 32 * ((rows + 255) // 256)) * (classes + 256) + 65 * MIB


@pytest.mark.parametrize("dtype", range(4))
def test_no_way_to_lie_takes_more_than_the_question_without_strides_says(dtype):
    for rows, k, classes in FEW + [(1, 1, 1), (3, 5, 7), (8192, 4096, 32768), (1000, 520, 10007), (20, 64, 3)]:
        for backward in (0, 1):
            for strides in ((k, 1, classes, 1), (k, 1, 1, k), (2 * k, 2, classes, 1), (k, 1, 3 * classes, 3), (0, 1, classes, 1)):
                assert 0 < strided(rows, k, classes, backward, strides, dtype) <= workspace(rows, k, classes, backward, dtype)


@pytest.mark.parametrize("dtype", HALF)
def test_fewer_classes_than_a_vector_go_one_way_however_the_weight_lies(dtype):
    """The tiles' unaligned loads of the logits' gradient would begin before it: the kernels for any strides take these, and ask for the same memory either way."""
    for rows, k in ((20, 64), (300, 72), (1, 4096)):
        for classes in range(1, 8):
            for backward in (0, 1):
                assert strided(rows, k, classes, backward, (k, 1, 1, k), dtype) == strided(rows, k, classes, backward, (k, 1, classes, 1), dtype)


def test_refusals():
    lib = capi.lib()
    for args, why in (((0, 64, 100, 1, 64, 1, 100, 1, capi.BF16), "extent"), ((4, 64, 100, 1, 64, -1, 100, 1, capi.BF16), "negative stride"), ((4, 64, 100, 1, 64, 1, 100, 1, 9), "unsupported dtype")):
        assert lib.rp_hip_linear_cross_entropy_workspace_strided(*args) == -1
        message = lib.rp_hip_last_error().decode()
        assert "rp_hip_linear_cross_entropy_workspace_strided" in message and why in message
