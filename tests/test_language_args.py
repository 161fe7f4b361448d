"""What layer norm, gated layers, the loss of a large vocabulary and distillation refuse, and say why (no GPU needed: a refused call touches no device)."""

from recpulse_amd import capi

P = 4096                                                        # stands for a device pointer; refused calls never look at it
BF16, F32 = capi.BF16, capi.F32


def refused(name, args, why):
    lib = capi.lib()
    assert getattr(lib, name)(*args) == -1
    message = lib.rp_hip_last_error().decode()
    assert name in message and why in message, message


def changed(args, **at):
    args = list(args)
    for where, value in at.items():
        args[int(where[1:])] = value
    return args


def test_layer_norm():
    ok = [P, None, P, P, P, 4, 64, 64, 64, 1e-5, BF16]
    name = "rp_hip_layer_norm_forward"
    for at in (0, 2):
        refused(name, changed(ok, **{f"_{at}": None}), "null operand")
    for at in (5, 6):
        refused(name, changed(ok, **{f"_{at}": 0}), "extent")
    refused(name, changed(ok, _7=63), "rows of y are 63 elements apart")
    refused(name, changed(ok, _8=-1), "negative stride")
    refused(name, changed(ok, _9=-1e-5), "eps")
    refused(name, changed(ok, _9=float("nan")), "eps")
    refused(name, changed(ok, _10=9), "unsupported dtype")
    ok = [P, P, P, P, P, P, P, P, 4, 64, 64, 64, 64, 0, 0, 0, BF16]
    name = "rp_hip_layer_norm_backward"
    for at in (3, 4, 6, 7):                                      # dy, x, stats, and the workspace where dw or db is asked for
        refused(name, changed(ok, **{f"_{at}": None}), "null operand")
    refused(name, changed(ok, _12=10), "rows of dx")
    refused(name, changed(ok, _16=-1), "unsupported dtype")
    refused("rp_hip_layer_norm_workspace", [0, 64, BF16], "extent")
    refused("rp_hip_layer_norm_workspace", [4, 64, 7], "unsupported dtype")
    assert capi.lib().rp_hip_layer_norm_workspace(4, 64, BF16) > 0
    assert capi.lib().rp_hip_layer_norm_backward(None, None, None, P, P, P, P, None, 4, 64, 64, 64, 64, 0, 0, 0, BF16) == 0      # nothing asked for


def test_gated_linear():
    ok = [P, None, P, P, None, 4, 32, 64, 0, 32, 1, 128, 1, 64, BF16]
    name = "rp_hip_gated_linear_forward"
    for at in (0, 2, 3):
        refused(name, changed(ok, **{f"_{at}": None}), "null operand")
    for at in (5, 6, 7):
        refused(name, changed(ok, **{f"_{at}": -2}), "extent")
    for gate in (-1, 5):
        refused(name, changed(ok, _8=gate), "unknown gate")
    refused(name, changed(ok, _11=-128), "negative stride")
    refused(name, changed(ok, _13=32), "rows of h")
    refused(name, changed(ok, _14=4), "unsupported dtype")
    ok = [P] * 8 + [4, 32, 64, 0, 64, 32, 1, 128, 1, 32, 128, 1, 0, 0, 0, BF16]
    name = "rp_hip_gated_linear_backward"
    for at in (3, 4, 5, 6, 7):                                   # dz, dh, z; x for dw, w for dx
        refused(name, changed(ok, **{f"_{at}": None}), "null operand")
    refused(name, changed(ok, _17=31), "rows of dx")
    for strides in ((128, 2), (127, 1), (1, 31), (2, 128)):
        refused(name, changed(ok, _18=strides[0], _19=strides[1]), "dw has unit stride")
    refused(name, changed(ok, _11=9), "unknown gate")


def test_linear_cross_entropy():
    ok = [P] * 7 + [4, 32, 100, 1, 32, 1, 100, 1, BF16]
    name = "rp_hip_linear_cross_entropy_forward"
    for at in (0, 1, 2, 3, 5, 6):
        refused(name, changed(ok, **{f"_{at}": None}), "null operand")
    for at in (7, 8, 9):
        refused(name, changed(ok, **{f"_{at}": 0}), "extent")
    refused(name, changed(ok, _10=3), "reduction")
    refused(name, changed(ok, _13=-1), "negative stride")
    refused(name, changed(ok, _15=5), "unsupported dtype")
    ok = [P] * 10 + [4, 32, 100, 1, 32, 1, 100, 1, 32, 100, 1, 0, 0, 0, BF16]
    name = "rp_hip_linear_cross_entropy_backward"
    for at in (3, 4, 6, 7, 9):
        refused(name, changed(ok, **{f"_{at}": None}), "null operand")
    refused(name, changed(ok, _18=20), "rows of dx")
    for strides in ((99, 1), (100, 2), (1, 31)):
        refused(name, changed(ok, _19=strides[0], _20=strides[1]), "dw has unit stride")
    refused("rp_hip_linear_cross_entropy_workspace", [4, 0, 100, 1, BF16], "extent")
    for dtype in range(4):
        for sizes in ((1, 1, 1), (4, 32, 100), (1 << 20, 64, 1 << 17)):
            forward, backward = (capi.lib().rp_hip_linear_cross_entropy_workspace(*sizes, b, dtype) for b in (0, 1))
            assert 0 < forward <= backward


def test_distillation():
    ok = [P] * 7 + [4, 100, 8, 100, 2.0, 1, BF16]
    name = "rp_hip_distillation_forward"
    for at in (0, 2, 3, 4, 5):
        refused(name, changed(ok, **{f"_{at}": None}), "null operand")
    for at in (7, 8, 9):
        refused(name, changed(ok, **{f"_{at}": 0}), "extent")
    refused(name, changed(ok, _9=1025), "at most 1024 entries")
    refused(name, changed(ok, _10=-1), "negative stride")
    for temperature in (0.0, -1.0, float("nan"), float("inf")):
        refused(name, changed(ok, _11=temperature), "temperature")
    refused(name, changed(ok, _12=-1), "reduction")
    refused(name, changed(ok, _13=11), "unsupported dtype")
    ok = [P] * 6 + [4, 100, 8, 100, 2.0, 1, F32]
    name = "rp_hip_distillation_backward"
    for at in (0, 1, 2, 3, 4):
        refused(name, changed(ok, **{f"_{at}": None}), "null operand")
    refused(name, changed(ok, _12=9), "unsupported dtype")
