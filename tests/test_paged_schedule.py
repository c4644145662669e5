"""How a paged attention launch divides its tiles, on the CPU: the schedule's arithmetic, compiled for the host from the kernels' own
header, against plain integers."""
import ctypes as C
import os
import random
import re
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "saetta_macqwen_b200", "csrc")
HOST = """
#include "paged_sched.cuh"
extern "C" uint64_t cut(uint64_t total, uint32_t c, uint32_t n) { return saetta::paged_cut(total, c, n); }
extern "C" uint32_t cta_of(uint64_t total, uint32_t ctas, uint64_t x) { return saetta::paged_cta_of(total, ctas, x); }
extern "C" uint64_t sum64(uint32_t n, uint32_t a, uint64_t b) { return saetta::tile_sum<64>(n, a, b); }
extern "C" uint64_t sum128(uint32_t n, uint32_t a, uint64_t b) { return saetta::tile_sum<128>(n, a, b); }
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("sched")
    (d / "host.cu").write_text(HOST)
    subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", CSRC, "-shared", "-Xcompiler", "-fPIC", "-o", str(d / "host.so"),
                    str(d / "host.cu")], check=True, capture_output=True)
    lib = C.CDLL(str(d / "host.so"))
    lib.cut.restype = C.c_uint64
    lib.cut.argtypes = [C.c_uint64, C.c_uint32, C.c_uint32]
    lib.cta_of.restype = C.c_uint32
    lib.cta_of.argtypes = [C.c_uint64, C.c_uint32, C.c_uint64]
    for f in (lib.sum64, lib.sum128):
        f.restype = C.c_uint64
        f.argtypes = [C.c_uint32, C.c_uint32, C.c_uint64]
    return lib


def totals(rng, n):
    yield from (1, 2, 148, 255, (1 << 24) - 1, 1 << 24, (1 << 32) + 7, (1 << 48) + 12345)
    for _ in range(n):
        yield rng.randrange(1, 1 << rng.randint(1, 50))


def test_shares_are_equal_and_cover_every_tile(host):
    rng = random.Random(1)
    for total in totals(rng, 3000):
        n = rng.randint(1, 255)
        for c in {0, n, rng.randint(0, n)}:
            assert host.cut(total, c, n) == total * c // n


def test_the_cta_of_a_tile_is_the_one_whose_share_holds_it(host):
    rng = random.Random(2)
    for total in totals(rng, 3000):
        n = rng.randint(1, min(255, total))
        for x in {0, total - 1, rng.randrange(total), total // 2}:
            c = host.cta_of(total, n, x)
            assert 0 <= c < n and total * c // n <= x < total * (c + 1) // n


@pytest.mark.parametrize("tpt", sorted({max(1, r // g) for r in (8, 16, 128) for g in range(1, 17)}))
def test_the_tiles_of_row_tiles(host, tpt):
    """Key tiles of the first n row tiles of tpt tokens, the first of which sees b - T + 1 keys."""
    rng = random.Random(tpt)
    for f, T in ((host.sum64, 64), (host.sum128, 128)):
        for n in (0, 1, 2, 7, 127, 128, 129, rng.randrange(1000), rng.randrange(1 << 16)):
            for b in (0, 1, T - 1, T, rng.randrange(1 << 20), rng.randrange(1 << 31)):
                assert f(n, tpt, b) == sum((tpt * i + b) // T for i in range(n))


def test_nothing_is_called_after_registers_were_given_back():
    """A callee compiled for the launch's registers may use some that its warp no longer has: these kernels call nothing at all."""
    for name in ("paged_sched.cuh", "paged_attend.cu", "paged_prefill.cu"):
        assert "__noinline__" not in open(os.path.join(CSRC, name)).read(), name


def test_two_rounds_join_the_parts_of_every_cta():
    """A round of the few-rows kernel holds kPdGroup + 1 parts at once, for as many CTAs as a launch may have."""
    hpp, attend = (open(os.path.join(CSRC, n)).read() for n in ("paged.hpp", "paged_attend.cu"))
    a, b = map(int, re.search(r"kPagedMaxCtas = (\d+) \* (\d+);", hpp).groups())
    group = int(re.search(r"kPdGroup = (\d+);", attend).group(1))
    for parts in range(1, a * b + 1):
        per = parts
        if parts > group:
            per = 2
            while per * per < parts:
                per += 1
        assert per <= group + 1 and (parts + per - 1) // per <= group + 1, parts
