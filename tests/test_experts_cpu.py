"""CPU checks of the expert-layer entry points: arguments are refused with a status and a
message before anything touches a device."""

import pytest


@pytest.fixture(scope="module")
def capi():
    from lightgbm_rs_b200 import build

    build.build()
    from lightgbm_rs_b200 import _lib

    return _lib


def test_arguments_are_refused_with_a_status(capi):
    L, bad, cap, length = (capi.lib(), capi.INVALID_ARGUMENT, capi.CAPABILITY_UNAVAILABLE,
                           capi.LENGTH_MISMATCH)
    p = 1 << 20  # never read: every call below is refused first
    route = L.lgbm_b200_experts_route
    assert route(p, 7, 4, 8, 8, 2, 1, p, p, p, p, p, p, 0, None) == bad      # dtype
    assert route(p, 0, 4, 8, 8, 9, 1, p, p, p, p, p, p, 0, None) == bad      # k > experts
    assert route(p, 0, 4, 8, 7, 2, 1, p, p, p, p, p, p, 0, None) == bad      # pitch < experts
    assert route(p, 0, -1, 8, 8, 2, 1, p, p, p, p, p, p, 0, None) == bad
    assert route(p, 0, 4, 513, 513, 2, 1, p, p, p, p, p, p, 0, None) == cap
    assert route(p, 0, 4, 64, 64, 17, 1, p, p, p, p, p, p, 0, None) == cap
    assert route(p, 0, 1 << 31, 8, 8, 2, 1, p, p, p, p, p, p, 0, None) == cap
    assert route(None, 0, 4, 8, 8, 2, 1, p, p, p, p, p, p, 0, None) == bad
    assert route(p, 0, 100000, 8, 8, 2, 1, p, p, p, p, p, None, 0, None) == length
    assert b"workspace" in L.lgbm_b200_last_error()
    assert L.lgbm_b200_experts_route_workspace(100000, 8, 2) > 0
    back = L.lgbm_b200_experts_route_backward
    assert back(None, p, p, p, 0, 4, 8, 8, 2, 1, p, None) == bad
    assert back(p, p, p, p, 0, 0, 8, 8, 2, 1, p, None) == capi.OK            # no tokens

    mm = L.lgbm_b200_experts_matmul
    assert mm(p, 4, 8, None, p, p, 0, 4, 2, 8, 8, p, None, 0, None) == bad   # f32
    assert mm(p, 4, 8, None, p, p, 1, 4, 0, 8, 8, p, None, 0, None) == bad   # no experts
    assert mm(p, 4, 8, None, p, p, 1, 4, 513, 8, 8, p, None, 0, None) == cap
    wide = (1 << 28) + 8
    assert mm(p, 4, wide, None, p, p, 1, 4, 2, wide, 8, p, None, 0, None) == cap
    assert mm(p, 4, 7, None, p, p, 1, 4, 2, 8, 8, p, None, 0, None) == length
    assert mm(p, 5, 8, None, p, p, 1, 4, 2, 8, 8, p, None, 0, None) == length
    assert mm(p, 400, 9, None, p, p, 1, 400, 2, 9, 8, p, None, 0, None) == length  # workspace
    assert mm(p, 4, 8, None, None, p, 1, 4, 2, 8, 8, p, None, 0, None) == bad
    assert mm(p, 0, 8, None, p, p, 1, 0, 2, 8, 8, p, None, 0, None) == capi.OK
    assert mm(p, 4, 8, None, p, p, 1, 4, 2, 8, 8, None, None, 0, None) == bad  # no result
    back = L.lgbm_b200_experts_matmul_backward
    assert back(p, 8, p, 4, 8, None, p, p, 1, 2, 4, 2, 8, 8, p, p, None, 0, None) == bad  # dw f16
    assert back(p, 7, p, 4, 8, None, p, p, 1, 1, 4, 2, 8, 8, p, p, None, 0, None) == length
    assert back(None, 8, p, 4, 8, None, p, p, 1, 1, 4, 2, 8, 8, p, p, None, 0, None) == bad
    assert back(p, 8, p, 4, 8, None, p, p, 1, 1, 4, 2, 8, 8, None, None, None, 0, None) == bad
    assert back(p, 8, p, 4, 8, None, None, p, 1, 1, 4, 2, 8, 8, p, None, None, 0, None) == bad
    assert back(p, 9, p, 4, 8, None, p, p, 1, 1, 4, 2, 8, 9, p, p, None, 0, None) == length

    w4 = L.lgbm_b200_experts_matmul_w4
    assert w4(p, 4, 8, None, p, p, None, 48, p, 1, 4, 2, 8, 8, p, None) == bad
    assert w4(p, 4, 8, None, p + 8, p, None, 32, p, 1, 4, 2, 8, 8, p, None) == bad
    assert w4(p, 4, 8, None, p, None, None, 32, p, 1, 4, 2, 8, 8, p, None) == bad
    assert w4(p, 4, 8, None, p, p, None, 32, p, 0, 4, 2, 8, 8, p, None) == bad

    comb = L.lgbm_b200_experts_combine
    assert comb(p, 3, 4, 8, 8, p, None, 2, 2, p, None) == bad
    assert comb(p, 0, 4, 8, 7, p, None, 2, 2, p, None) == bad
    assert comb(p, 0, 4, 8, 8, None, None, 2, 2, p, None) == bad
    cb = L.lgbm_b200_experts_combine_backward
    assert cb(p, p, 0, 5, 8, 8, 8, p, None, 2, 2, p, None, None) == length
    assert cb(p, None, 0, 4, 8, 8, 8, p, p, 2, 2, p, p, None) == bad
    drop = L.lgbm_b200_experts_dropout
    assert drop(p, None, 0, 1, 8, 8, 0, 1.5, 0, 0, p, None) == bad
    assert drop(p, None, 0, 1, 8, 8, 0, float("nan"), 0, 0, p, None) == bad
    assert drop(p, p, 0, 2, 8, 8, 7, 0.5, 0, 0, p, None) == bad
    assert drop(p, None, 0, 1 << 40, 1 << 40, 1 << 40, 0, 0.5, 0, 0, p, None) == bad
    assert drop(p, None, 0, 0, 8, 8, 0, 0.5, 0, 0, p, None) == capi.OK
    assert L.lgbm_b200_experts_errors(None) == bad


def test_workspace_only_where_an_operand_must_be_copied(capi):
    ws = capi.lib().lgbm_b200_experts_matmul_workspace
    p = 1 << 20
    assert ws(p, 64, None, p, 1000, 4, 64, 33) == 0
    assert ws(p, 64, None, p + 2, 1000, 4, 64, 33) > 0
    assert ws(p, 65, None, p, 1000, 4, 65, 33) > 0
    assert ws(p, 64, p, p, 1000, 4, 64, 33) > 0     # gathered rows
    assert ws(p, 65, p, p, 60, 4, 65, 33) == 0      # few rows are read where they are
    back = capi.lib().lgbm_b200_experts_matmul_backward_workspace
    one = back(p, 33, p, 64, None, p, 1000, 4, 64, 33, 1, 0)
    assert one > 0 and back(p, 33, p, 64, None, p, 1000, 4, 64, 33, 1, 1) == one  # dy once
    assert back(p, 40, p, 64, None, p, 1000, 4, 64, 33, 1, 1) == 0
