"""CPU checks of the gated and linear layers and of clipping: what must not reach a device is
refused with a status and a message before anything touches one."""

import ctypes

import pytest


@pytest.fixture(scope="module")
def capi():
    from lightgbm_rs_b200 import build

    build.build()
    from lightgbm_rs_b200 import _lib

    return _lib


P, N = 1 << 20, 1 << 20  # an address that is never read, workspace bytes enough

# complete calls, and (place, bytes off) of each array
CALLS = {
    "linear": ([P, 4, 8, P, P, P, P, 8, P, 1, 2, 4, 2, 8, 8, P, P, P, N, None],
               [(0, 1), (3, 2), (4, 1), (5, 1), (6, 1), (8, 2), (15, 1), (16, 16)]),
    "gated": ([P, 4, 8, P, P, P, 1, 2, 4, 2, 8, 8, P, P, P, N, None],
              [(0, 1), (3, 2), (4, 1), (5, 2), (12, 1), (13, 16)]),
    "linear_backward": ([P, 8, P, P, 4, 8, P, P, P, 1, 0, 2, 4, 2, 8, 8, P, P, P, P, N, None],
                        [(0, 1), (2, 16), (3, 1), (6, 2), (7, 1), (8, 2), (16, 1), (17, 2),
                         (18, 2)]),
    "gated_backward": ([P, 8, P, P, 4, 8, P, P, P, 1, 0, 2, 4, 2, 8, 8, P, P, P, N, None],
                       [(0, 1), (2, 16), (3, 1), (6, 2), (7, 1), (8, 2), (16, 1), (17, 2)]),
}


def call(capi, name, **changes):
    args = list(CALLS[name][0])
    for place, value in changes.items():
        args[int(place[1:])] = value
    return getattr(capi.lib(), "lgbm_b200_experts_" + name)(*args)


def test_arrays_off_their_elements_are_refused(capi):
    for name, (args, arrays) in CALLS.items():
        for place, off in arrays:
            got = call(capi, name, **{f"a{place}": args[place] + off})
            assert got == capi.INVALID_ARGUMENT, (name, place, capi.lib().lgbm_b200_last_error())


def test_arguments_are_refused_with_a_status(capi):
    bad, cap, length = capi.INVALID_ARGUMENT, capi.CAPABILITY_UNAVAILABLE, capi.LENGTH_MISMATCH
    half, wide = (1 << 27) + 8, (1 << 28) + 8
    for name, dtype, rows, experts, inner, outer, result in (
            ("linear", 9, 11, 12, 13, 14, 15), ("gated", 6, 8, 9, 10, 11, 12),
            ("linear_backward", 9, 12, 13, 14, 15, 16), ("gated_backward", 9, 12, 13, 14, 15, 16)):
        at = lambda **k: call(capi, name, **{f"a{i}": v for i, v in k.items()})  # noqa: E731
        put = lambda place, v: call(capi, name, **{f"a{place}": v})  # noqa: E731
        assert put(dtype, 0) == bad, name          # f32
        assert put(dtype, 7) == bad
        assert put(rows, -1) == bad
        assert put(experts, 0) == bad
        assert put(experts, 513) == cap
        assert put(inner, 0) == bad
        assert put(outer, 0) == bad
        assert put(outer, half if "gated" in name else wide) == cap
        assert put(rows, (1 << 31) - 1) == cap
        act = {"linear": 10, "gated": 7}.get(name, 11)
        assert put(act, 4) == bad and put(act, -1) == bad
        x = 3 if "backward" in name else 0
        assert put(x, None) == bad
        assert put(x + 2, 7) == length             # x's pitch
    assert call(capi, "linear", a15=None) == bad and call(capi, "gated", a12=None) == bad
    assert call(capi, "linear", a7=7) == length    # residual's pitch
    for name in ("linear_backward", "gated_backward"):
        assert call(capi, name, a0=None) == bad
        assert call(capi, name, a1=7) == length    # the gradient's pitch
        assert call(capi, name, a2=None) == bad    # pre
        assert call(capi, name, a10=2) == bad      # dw in f16 for bf16
        assert call(capi, name, a8=None) == bad
        nothing = {"a16": None, "a17": None, **({"a18": None} if "linear" in name else {})}
        assert call(capi, name, **nothing) == bad
        ws = {"linear_backward": "a20", "gated_backward": "a19"}[name]
        assert call(capi, name, **{ws: 0}) == length
        assert b"workspace" in capi.lib().lgbm_b200_last_error()
    assert call(capi, "linear_backward", a19=P + 8) == length  # workspace's alignment


def test_workspace_of_the_backward_passes(capi):
    lin = capi.lib().lgbm_b200_experts_linear_backward_workspace
    gat = capi.lib().lgbm_b200_experts_gated_backward_workspace
    p, relu = 1 << 20, 1
    args = (p, 40, p, 64, None, p)
    # without an activation dy itself is multiplied: nothing to keep but an operand's copies
    assert lin(*args, 0, 1024, 4, 64, 40, 1, 1, 0) == 0
    assert lin(p, 33, p, 64, None, p, 0, 1024, 4, 64, 33, 1, 0, 0) >= 1024 * 40 * 2
    assert lin(*args, relu, 1024, 4, 64, 40, 1, 1, 0) == 1024 * 40 * 2
    assert lin(*args, relu, 1024, 4, 64, 33, 1, 0, 0) >= 1024 * 40 * 2
    sums = lin(*args, 0, 1024, 4, 64, 40, 0, 0, 1)
    assert 4 * 40 * 4 < sums < 1 << 20
    assert lin(*args, relu, 1024, 4, 64, 40, 0, 0, 1) == 1024 * 40 * 2 + sums
    assert lin(*args, relu, 0, 4, 64, 40, 1, 1, 1) == 0
    assert gat(p, 64, None, p, 1024, 4, 64, 20, 1, 1) == 1024 * 40 * 2
    assert gat(p, 64, p, p, 1024, 4, 64, 20, 0, 1) >= 1024 * (40 + 64) * 2  # gathered x
    assert gat(p, 64, None, p, 1024, 4, 64, 0, 1, 1) == 0
    # a long reduction of few tiles, in parts: 2 of 576 and 448 in f32
    assert gat(p, 64, None, p, 100, 60, 64, 512, 1, 0) == 100 * 1024 * 2 + 2 * 100 * 64 * 4


class Item(ctypes.Structure):
    _fields_ = [("input", ctypes.c_void_p), ("out", ctypes.c_void_p), ("count", ctypes.c_int64),
                ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


def test_clipping_refuses(capi):
    L, bad, cap, length = (capi.lib(), capi.INVALID_ARGUMENT, capi.CAPABILITY_UNAVAILABLE,
                           capi.LENGTH_MISMATCH)

    def clip(items, most=1.0, norm=P, ws=P, size=N, n=None):
        a = (Item * max(1, len(items)))(*[Item(*i, 0) for i in items])
        return L.lgbm_b200_experts_clip_grads(a, len(items) if n is None else n, most, norm, ws,
                                              size, None)

    assert clip([(P, P, 5, 3)]) == bad              # dtype
    assert clip([(P, P, -1, 0)]) == bad
    assert clip([(None, P, 5, 0)]) == bad
    assert clip([(P, None, 5, 0)]) == bad
    assert clip([(P + 2, P, 5, 0)]) == bad          # off its elements
    assert clip([(P, P + 1, 5, 1)]) == bad
    assert clip([(P, P, 5, 0)], most=-1.0) == bad
    assert clip([(P, P, 5, 0)], most=float("nan")) == bad
    assert clip([(P, P, 5, 0)], norm=None) == bad
    assert clip([(P, P, 5, 0)], norm=P + 2) == bad
    assert clip([(P, P, 5, 0)], n=-1) == bad
    assert clip([(P, P, 1 << 43, 0)]) == cap
    assert clip([(P, P, 1 << 62, 1)]) == cap
    assert clip([(P, P, 1 << 20, 0)], size=0) == length
    assert clip([(P, P, 1 << 20, 0)], ws=P + 8) == length
    assert L.lgbm_b200_experts_grad_norm(None, 1, P, P, N, None) == bad
    small = (Item * 2)(Item(P, P, 100_000, 0, 0), Item(P, P, 3, 1, 0))
    many = (Item * 2000)(*[Item(P, P, 1, 0, 0)] * 2000)
    ws = L.lgbm_b200_experts_norm_workspace
    assert ws(small, 2) == 0 and ws(small, 0) == 0  # one cluster needs none
    assert 0 < ws(many, 65) < ws(many, 2000)
