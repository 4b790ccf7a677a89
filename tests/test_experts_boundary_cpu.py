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


def test_philox_counter_words(tmp_path):
    """The device's generator, compiled for the host, against the published known answers and
    Python integers, with every word of the counter and the key in use: elements from 2^35 on have
    block numbers past 32 bits, more than a test can hold in memory."""
    lib = compiled(tmp_path, '#include "philox.h"\n'
                   'extern "C" void philox(uint64_t block, uint64_t offset, uint64_t seed,\n'
                   '                       uint32_t* out) {\n'
                   '  uint32_t w[4];\n'
                   '  lgbm_b200::experts::philox(block, offset, (uint32_t)seed,\n'
                   '                             (uint32_t)(seed >> 32), w);\n'
                   '  for (int i = 0; i < 4; ++i) out[i] = w[i];\n}\n')
    u64 = ctypes.c_uint64

    def words(block, offset, seed):
        out = (ctypes.c_uint32 * 4)()
        lib.philox(u64(block), u64(offset), u64(seed), out)
        return list(out)

    def integers(block, offset, seed):
        low = 0xFFFFFFFF
        c, k0, k1 = [block & low, block >> 32, offset & low, offset >> 32], seed & low, seed >> 32
        for _ in range(10):
            p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(q >> 32) ^ c[1] ^ k0, q & low, (p >> 32) ^ c[3] ^ k1, p & low]
            k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
        return c

    full = (1 << 64) - 1
    assert words(0, 0, 0) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert words(full, full, full) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    for block in (5, 1 << 32, (1 << 32) + 5, 0xFEDCBA9876543210):
        for offset in (0, 7, (3 << 32) + 1):
            for seed in (1, 0x0123456789ABCDEF):
                assert words(block, offset, seed) == integers(block, offset, seed)
    assert words(5, 0, 1) != words((1 << 32) + 5, 0, 1)


def test_streamed_or_copied_by_alignment(capi):
    """Weights that the tiles' loads cannot walk are streamed while that is the shorter way:
    workspace for their copy says which it is."""
    ws, p = capi.lib().lgbm_b200_experts_matmul_workspace, 1 << 20
    x = lambda inner: (p, (inner + 7) // 8 * 8, None)  # noqa: E731  aligned rows of x
    assert ws(*x(2001), p, 16, 32, 2001, 4096) == 0        # rows at 2 bytes: half the experts
    assert ws(*x(2001), p, 17, 32, 2001, 4096) > 0
    assert ws(*x(2000), p + 2, 17, 32, 2000, 4096) > 0     # the base counts too
    assert ws(*x(2002), p, 24 * 32, 32, 2002, 4096) == 0   # at 4 bytes: 24 an expert
    assert ws(*x(2002), p, 24 * 32 + 1, 32, 2002, 4096) > 0
    assert ws(*x(700), p, 12 * 255, 255, 700, 129) == 0    # half of the last block is empty
    assert ws(*x(700), p, 13 * 255, 255, 700, 129) > 0
    assert ws(*x(129), p, 32 * 64, 64, 129, 128) == 0      # small weights
    assert ws(*x(129), p, 32 * 64 + 1, 64, 129, 128) > 0


def test_waits_do_not_count_time_off_the_device(tmp_path):
    """A wait that is polled ends after two seconds; one that was switched out for minutes has lost a
    hundredth of its time; looks that are each late end it after a hundred of them."""
    lib = compiled(tmp_path, '#include "wait_budget.h"\n'
                   'using lgbm_b200::experts::WaitBudget;\n'
                   'extern "C" long looks(unsigned long long every, unsigned long long gap, long at) {\n'
                   '  unsigned long long now = 12345;\n'
                   '  WaitBudget b(now);\n'
                   '  for (long i = 1;; ++i) {\n'
                   '    now += i == at ? gap : every;\n'
                   '    if (!b.spend(now)) return i;\n'
                   '  }\n}\n')
    looks = lambda every, gap=0, at=-1: lib.looks(  # noqa: E731
        ctypes.c_ulonglong(every), ctypes.c_ulonglong(gap), ctypes.c_long(at))
    lib.looks.restype = ctypes.c_long
    assert looks(10_000) == 200_000
    assert looks(10_000, gap=300 * 10 ** 9, at=7) == 200_000 - 2000 + 1
    assert looks(10 ** 9) == 100
