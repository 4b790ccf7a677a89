"""CPU checks of the expert layers: what must not reach a device is refused before, and the
arithmetic that host and device share."""

import ctypes
import subprocess

import pytest


@pytest.fixture(scope="module")
def capi():
    from lightgbm_rs_b200 import build

    build.build()
    from lightgbm_rs_b200 import _lib

    return _lib


def test_arrays_off_their_elements_are_refused(capi):
    """Every array of every call in turn one byte (or half an element) off; the calls are complete
    otherwise, and none is passed on: a device would fault."""
    L, p = capi.lib(), 1 << 20
    n = 1 << 20  # workspace bytes, enough
    calls = {  # arguments, and (place, bytes off) of each array
        "route": ([p, 1, 100, 8, 8, 2, 1, p, p, p, p, p, p, n, None],
                  [(0, 1), (7, 2), (8, 2), (9, 2), (10, 2), (11, 2)]),
        "route_backward": ([p, p, p, p, 0, 4, 8, 8, 2, 1, p, None],
                           [(0, 2), (1, 2), (2, 2), (3, 2), (10, 2)]),
        "matmul": ([p, 4, 8, p, p, p, 1, 4, 2, 8, 8, p, p, n, None],
                   [(0, 1), (3, 2), (4, 1), (5, 2), (11, 1)]),
        "matmul_backward": ([p, 8, p, 4, 8, p, p, p, 1, 0, 4, 2, 8, 8, p, p, p, n, None],
                            [(0, 1), (2, 1), (5, 2), (6, 1), (7, 2), (14, 1), (15, 2)]),
        "matmul_w4": ([p, 4, 8, p, p, p, p, 32, p, 1, 4, 2, 8, 8, p, None],
                      [(0, 1), (3, 2), (4, 1), (5, 1), (8, 2), (14, 1)]),
        "combine": ([p, 0, 4, 8, 8, p, p, 2, 2, p, None], [(0, 2), (5, 2), (6, 2), (9, 2)]),
        "combine_backward": ([p, p, 0, 4, 8, 8, 8, p, p, 2, 2, p, p, None],
                             [(0, 2), (1, 2), (7, 2), (8, 2), (11, 2), (12, 2)]),
        "dropout": ([p, p, 0, 2, 8, 8, 8, 0.5, 0, 0, p, None], [(0, 2), (1, 2), (10, 2)]),
    }
    for name, (args, arrays) in calls.items():
        for place, off in arrays:
            bad = list(args)
            bad[place] += off
            got = getattr(L, "lgbm_b200_experts_" + name)(*bad)
            assert got == capi.INVALID_ARGUMENT, (name, place, L.lgbm_b200_last_error())
    # scratch is 16-byte aligned
    args = list(calls["route"][0])
    args[12] += 4
    assert L.lgbm_b200_experts_route(*args) == capi.LENGTH_MISMATCH


def compiled(tmp_path, body):
    """C++ around the library's own headers, as a shared object."""
    from lightgbm_rs_b200 import build

    src, so = str(tmp_path / "shim.cpp"), str(tmp_path / "shim.so")
    with open(src, "w") as f:
        f.write(body)
    subprocess.run([build.HOST_CXX, "-O1", "-std=c++17", "-shared", "-fPIC", f"-I{build.CSRC}",
                    "-o", so, src], check=True)
    return ctypes.CDLL(so)


def test_parts_of_a_weight_gradient_are_even(tmp_path):
    """Parts cover the rows in whole blocks of 64, and no smaller number of blocks would."""
    lib = compiled(tmp_path, '#include "experts_parts.h"\n'
                   'extern "C" int part_rows(int n, int parts, int block) {\n'
                   '  return lgbm_b200::experts::part_rows(n, parts, block);\n}\n')
    for parts in (1, 2, 3, 7, 24, 148):
        for n in [0, 1, 63, 64, 65, 64 * parts, 64 * parts * 5, 64 * parts * 5 + 1, 2063,
                  (1 << 31) - 65537]:
            each = lib.part_rows(n, parts, 64)
            assert each % 64 == 0 and each * parts >= n
            assert n == 0 or (each // 64 - 1) * parts < -(-n // 64)
    assert lib.part_rows(64 * 24 * 5, 24, 64) == 64 * 5  # not six blocks, four parts empty
