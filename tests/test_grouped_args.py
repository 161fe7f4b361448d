"""Refusals of the routing, exchange, grouped and adapter entry points: reported with -1 and a message before any device work (no GPU needed)."""
import pytest

from recpulse_amd import capi

P = 4096          # an address that is never touched


def refused(name, args, word):
    lib = capi.lib()
    assert getattr(lib, name)(*args) == -1
    assert word in lib.rp_hip_last_error().decode(), lib.rp_hip_last_error()


def changed(args, at, value):
    return args[:at] + (value,) + args[at + 1:]


ROUTE = (P, P, P, P, P, P, 64, 10, 64, 4, 1, capi.BF16)
ROUTE_BACK = (P, P, P, P, P, 64, 10, 64, 4, 0, capi.BF16)
DISPATCH = (P, P, P, 10, 2, 64, 64, 64, capi.F32)
COMBINE = (P, P, None, P, 10, 2, 64, 64, 64, capi.F32)
COMBINE_BACK = (P, P, P, P, P, P, 10, 2, 64, 64, 64, 64, capi.F32)
GROUPED = (P, P, P, None, P, 4, 100, 64, 72, 64, 1, 64 * 72, 72, 1, 72, capi.F16)
GROUPED_BACK = (P, P, P, P, P, P, P, 4, 100, 64, 72, 72, 64, 1, 64 * 72, 72, 1, 64, 0, 0, 0, capi.F16)
ADAPTER = (P, P, P, P, None, P, P, None, P, P, 4, 2, 100, 64, 72, 8, 64, 1, 72, 1, 72, capi.F16)
ADAPTER_BACK = (P, P, P, P, P, P, P, P, P, P, None, P, P, 4, 2, 100, 64, 72, 8, 72, 64, 1, 72, 1, 64, 0, 0, 0, capi.F16)


@pytest.mark.parametrize("name, args, pointers", [
    ("rp_hip_route_forward", ROUTE, range(6)), ("rp_hip_route_backward", ROUTE_BACK, range(5)), ("rp_hip_group_rows", (P, P, P, P, 10, 4), range(4)),
    ("rp_hip_dispatch_rows", DISPATCH, range(3)), ("rp_hip_combine_forward", COMBINE, (0, 1, 3)), ("rp_hip_combine_backward", COMBINE_BACK, range(6)),
    ("rp_hip_grouped_linear_forward", GROUPED, (0, 1, 2, 4)), ("rp_hip_grouped_linear_backward", GROUPED_BACK, (3, 4, 5, 6)),
    ("rp_hip_adapter_linear_forward", ADAPTER, (0, 1, 2, 3, 5, 6, 8, 9)), ("rp_hip_adapter_linear_backward", ADAPTER_BACK, (3, 4, 5, 6, 7, 8, 9, 11, 12))])
def test_null_operands(name, args, pointers):
    for at in pointers:
        refused(name, changed(args, at, None), "null operand")


@pytest.mark.parametrize("name, args, extents, dtype", [
    ("rp_hip_route_forward", ROUTE, (7, 8, 9), 11), ("rp_hip_route_backward", ROUTE_BACK, (6, 7, 8), 10), ("rp_hip_group_rows", (P, P, P, P, 10, 4), (4, 5), None),
    ("rp_hip_dispatch_rows", DISPATCH, (3, 4, 5), 8), ("rp_hip_combine_forward", COMBINE, (4, 5, 6), 9), ("rp_hip_combine_backward", COMBINE_BACK, (6, 7, 8), 12),
    ("rp_hip_grouped_linear_forward", GROUPED, (5, 6, 7, 8), 15), ("rp_hip_grouped_linear_backward", GROUPED_BACK, (7, 8, 9, 10), 21),
    ("rp_hip_adapter_linear_forward", ADAPTER, (10, 11, 12, 13, 14, 15), 21), ("rp_hip_adapter_linear_backward", ADAPTER_BACK, (13, 14, 15, 16, 17, 18), 28)])
def test_extents_and_types(name, args, extents, dtype):
    for at in extents:
        for value in (0, -3):
            refused(name, changed(args, at, value), "non-positive extent")
    if dtype is not None:
        for value in (-1, 4, 99):
            refused(name, changed(args, dtype, value), "unsupported dtype")


def test_limits_of_routing():
    refused("rp_hip_route_forward", changed(changed(ROUTE, 8, 1025), 6, 2000), "at most 1024 experts")
    refused("rp_hip_route_forward", changed(ROUTE, 9, 17), "k at most 16")
    refused("rp_hip_route_forward", changed(changed(ROUTE, 8, 3), 9, 4), "no more than the experts")
    refused("rp_hip_route_forward", changed(ROUTE, 6, 63), "rows of 63 elements apart hold 64")
    refused("rp_hip_route_forward", changed(ROUTE, 7, 1 << 29), "slots")
    refused("rp_hip_group_rows", (P, P, P, P, 10, 1025), "at most 1024 groups")
    refused("rp_hip_group_rows", (P, P, P, P, (1 << 30) + 1, 4), "at most 1024 groups")


def test_strides():
    for at in (6, 7):
        refused("rp_hip_dispatch_rows", changed(DISPATCH, at, 63), "rows of 63 elements apart hold 64")
    for at in (7, 8):
        refused("rp_hip_combine_forward", changed(COMBINE, at, 10), "rows of 10 elements apart hold 64")
    for at in (9, 10, 11):
        refused("rp_hip_combine_backward", changed(COMBINE_BACK, at, 10), "rows of 10 elements apart hold 64")
    for at in range(9, 15):
        refused("rp_hip_grouped_linear_forward", changed(GROUPED, at, -1), "negative stride")
    for at in range(11, 18):
        refused("rp_hip_grouped_linear_backward", changed(GROUPED_BACK, at, -1), "negative stride")
    for at in range(16, 21):
        refused("rp_hip_adapter_linear_forward", changed(ADAPTER, at, -1), "negative stride")
    for at in range(19, 25):
        refused("rp_hip_adapter_linear_backward", changed(ADAPTER_BACK, at, -1), "negative stride")
    refused("rp_hip_grouped_linear_forward", changed(GROUPED, 14, 71), "rows of y are 71 elements apart and hold 72")
    refused("rp_hip_grouped_linear_backward", changed(GROUPED_BACK, 17, 63), "rows of dx are 63 elements apart and hold 64")
    refused("rp_hip_adapter_linear_forward", changed(ADAPTER, 20, 71), "rows of y are 71 elements apart and hold 72")
    refused("rp_hip_adapter_linear_backward", changed(ADAPTER_BACK, 24, 63), "rows of dx are 63 elements apart and hold 64")


def test_zero_rows_behind():
    args = (P, P, 4, 10, 64, 64, capi.BF16)
    for at in (0, 1):
        refused("rp_hip_zero_rows_behind", changed(args, at, None), "null operand")
    for at in (2, 3, 4):
        refused("rp_hip_zero_rows_behind", changed(args, at, 0), "non-positive extent")
    refused("rp_hip_zero_rows_behind", changed(args, 5, 63), "rows of 63 elements apart hold 64")
    refused("rp_hip_zero_rows_behind", changed(args, 6, 9), "unsupported dtype")
