"""The ops whose weight depends on the row refuse host tensors with a message (no GPU needed)."""
import numpy as np
import pytest

import recpulse_cuda as rp
from recpulse.module import AdapterLinear, ExpertLinear, MixtureOfExperts


def test_host_tensors_are_refused():
    x = rp.from_numpy(np.ones((4, 6), np.float32))
    with pytest.raises(RuntimeError, match="op_route on host tensors"):
        x.op_route(2)
    with pytest.raises(RuntimeError, match="routing lives on a GPU"):
        rp.group_rows([0, 1], 2, "cpu")
    with pytest.raises(RuntimeError, match="op_adapter_linear on host tensors"):
        AdapterLinear(6, 5, 2, 3)(x, [0], [4])
    with pytest.raises(RuntimeError, match="op_route on host tensors"):
        MixtureOfExperts(6, 8, 4, 2)(x)


def test_modules_keep_their_parameters():
    moe = MixtureOfExperts(6, 8, 4, 2)
    assert {name: t.shape for name, t in moe.tracked.items()} == {"router.weight": (6, 4), "up.weight": (4, 6, 8), "up.bias": (4, 8),
                                                                  "down.weight": (4, 8, 6), "down.bias": (4, 6)}
    assert sorted(MixtureOfExperts(6, 8, 4, 2, bias=False).tracked) == ["down.weight", "router.weight", "up.weight"]
    layer = AdapterLinear(6, 5, 2, 3)
    assert {name: t.shape for name, t in layer.tracked.items()} == {"weight": (6, 5), "bias": (5,), "a": (2, 6, 3), "b": (2, 3, 5)}
    assert sorted(layer.learnable()) == ["a", "b"] and sorted(AdapterLinear(6, 5, 2, 3, train_shared=True).learnable()) == ["a", "b", "bias", "weight"]
    assert np.all(layer.b.to_numpy() == 0) and ExpertLinear(2, 3, 4).weight.shape == (2, 3, 4)
