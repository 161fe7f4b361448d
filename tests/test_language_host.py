"""Layer norm, gated layers, the loss of a large vocabulary and distillation refuse host tensors with a message (no GPU needed), and their modules keep their parameters."""
import numpy as np
import pytest

import recpulse_cuda as rp
from recpulse.module import GatedFeedForward, GatedLinear, LayerNorm, LinearCrossEntropy


def test_host_tensors_are_refused():
    x = rp.from_numpy(np.ones((4, 6), np.float32))
    for name, call in (("op_layer_norm", lambda: LayerNorm(6)(x)), ("op_gated_linear", lambda: GatedFeedForward(6, 8)(x)), ("op_linear_cross_entropy", lambda: LinearCrossEntropy(6, 9)(x, [0, 1, 2, 8])),
                       ("op_distillation_loss", lambda: x.op_distillation_loss([[0], [1], [2], [3]], rp.from_numpy(np.ones((4, 1), np.float32))))):
        with pytest.raises(RuntimeError, match=f"{name} on host tensors"):
            call()


def test_names_that_do_not_exist_are_refused():
    x = rp.from_numpy(np.ones((4, 6), np.float32))
    with pytest.raises(ValueError, match="gate must be"):
        GatedLinear(6, 8, gate="tanh")(x)
    with pytest.raises(ValueError, match="reduction must be"):
        LinearCrossEntropy(6, 9, reduction="max")(x, [0, 1, 2, 3])
    with pytest.raises(RuntimeError, match="one class for each"):
        x.op_distillation_loss([[0, 1]], rp.from_numpy(np.ones((4, 1), np.float32)))
    with pytest.raises(RuntimeError, match="one class for each"):      # as many as the teacher has, but not a row's
        x.op_distillation_loss([[0, 1, 2], [3], [0, 1], [2, 3]], rp.from_numpy(np.ones((4, 2), np.float32)))


def test_modules_keep_their_parameters():
    block = GatedFeedForward(6, 8)
    assert {name: t.shape for name, t in block.tracked.items()} == {"up.weight": (6, 16), "up.bias": (16,), "down.weight": (8, 6), "down.bias": (6,)}
    assert sorted(GatedFeedForward(6, 8, bias=False).tracked) == ["down.weight", "up.weight"]
    norm = LayerNorm(5)
    assert np.all(norm.weight.to_numpy() == 1) and np.all(norm.bias.to_numpy() == 0) and sorted(LayerNorm(5, bias=False).tracked) == ["weight"]
    assert {name: t.shape for name, t in LinearCrossEntropy(6, 9).tracked.items()} == {"weight": (6, 9), "bias": (9,)}
