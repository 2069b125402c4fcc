"""Which narrow product a call takes (csrc/narrow_rule.h), compiled for the CPU: both sides of its borders as they were measured."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sglang_b200", "csrc")
SHIM = """
#include "narrow_rule.h"
using namespace sglb200::narrow;
extern "C" int router(int64_t T, int64_t E, int64_t K) { return small_blocks(T, E, K); }
extern "C" int adapters(int64_t T, int64_t S, int64_t R, int64_t K, int64_t N) { return small_adapter_blocks(T, S, R, K, N); }
"""
# (T, E, K): us in blocks of 32 rows, of 128
ROUTER = {(256, 32, 1024): (3.1, 4.6), (128, 64, 1024): (3.2, 4.5), (512, 64, 1024): (4.0, 4.6), (4096, 16, 1024): (4.7, 4.5),
          (2048, 32, 1024): (4.7, 4.7), (256, 64, 2048): (4.3, 4.7), (512, 64, 2048): (4.7, 4.8), (1024, 64, 2048): (6.0, 5.4),
          (256, 256, 2048): (6.1, 5.5), (2048, 64, 2048): (8.0, 6.0), (768, 32, 4096): (4.9, 5.5), (1536, 32, 4096): (6.6, 5.7),
          (384, 64, 7168): (6.2, 6.7), (96, 256, 7168): (6.2, 6.6), (192, 160, 7168): (7.8, 6.7), (512, 64, 7168): (7.9, 6.8),
          (1536, 16, 4096): (4.9, 5.5), (192, 160, 4096): (6.1, 5.5), (2048, 32, 4096): (8.5, 6.3), (4096, 16, 4096): (8.5, 6.8), (1024, 16, 4096): (4.8, 5.4)}
# (T, slices, rank, K, columns): the same for three requests, sixteen, sixteen in any order
ADAPTERS = {(256, 1, 16, 7168, 2112): (11.2, 17.1, 11.3, 19.0, 12.8, 20.9), (1024, 1, 16, 7168, 2112): (14.9, 19.4, 15.1, 22.4, 18.7, 23.6),
            (192, 2, 32, 7168, 36864): (20.2, 22.4, 24.6, 39.5, 25.2, 41.0), (768, 2, 32, 7168, 36864): (48.8, 33.2, 71.5, 50.6, 72.8, 51.0),
            (96, 2, 64, 7168, 36864): (19.2, 21.6, 39.4, 42.0, 41.9, 42.8), (256, 2, 64, 7168, 36864): (36.0, 24.5, 46.6, 44.0, 64.0, 47.3),
            (128, 3, 64, 8192, 10240): (19.0, 20.2, 23.0, 31.7, 25.6, 33.5), (288, 3, 64, 8192, 10240): (28.7, 21.8, 36.6, 32.9, 37.8, 34.8),
            (257, 1, 128, 4096, 4096): (16.3, 18.3, 19.1, 20.9, 22.0, 22.2), (768, 1, 128, 4096, 4096): (28.4, 21.6, 30.4, 23.0, 32.7, 24.4),
            (257, 3, 16, 8192, 10240): (15.2, 20.4, 19.2, 25.5, 20.7, 27.2), (1024, 3, 16, 8192, 10240): (31.8, 27.3, 32.7, 29.3, 36.5, 30.7),
            (256, 1, 256, 4096, 6144): (28.0, 32.0, 31.0, 44.9, 42.4, 59.8), (1536, 1, 256, 4096, 6144): (98.7, 80.2, 104.3, 104.1, 119.9, 111.4),
            (512, 2, 32, 2048, 2048): (13.4, 15.5, 13.7, 15.3, 13.9, 16.3), (2048, 1, 8, 5120, 5120): (24.9, 23.2, 25.8, 25.0, 27.9, 29.2)}


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    d = tmp_path_factory.mktemp("narrow_rule")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I", CSRC, "-o", str(d / "shim.so"), str(d / "shim.cpp")])
    lib = ctypes.CDLL(str(d / "shim.so"))
    lib.router.argtypes, lib.adapters.argtypes = [ctypes.c_int64] * 3, [ctypes.c_int64] * 5
    return lib


def test_router_takes_the_faster_one(rule):
    for size, (small, tile) in ROUTER.items():
        taken = small if rule.router(*size) else tile
        assert taken <= 1.05 * min(small, tile), (size, small, tile)


def test_adapters_take_the_faster_one(rule):
    """On the average of the three ways in which requests lie, which the call does not know."""
    for size, us in ADAPTERS.items():
        small, tile = sum(us[0::2]), sum(us[1::2])
        taken = small if rule.adapters(*size) else tile
        assert taken <= 1.05 * min(small, tile), (size, us)


def test_more_rows_never_go_back_to_smaller_blocks(rule):
    for E, K in ((8, 8), (64, 1024), (256, 7168), (65536, 1 << 20), (1, 1 << 20)):
        taken = [rule.router(T, E, K) for T in list(range(1, 3000, 7)) + [1 << 20, (1 << 31) - 1024]]
        assert taken == sorted(taken, reverse=True)
    for S, R, K, N in ((1, 8, 8, 8), (2, 32, 7168, 36864), (8, 256, 1 << 20, (1 << 31) - 70000), (1, 256, 4096, 6144), (1, 128, 4096, 4096)):
        taken = [rule.adapters(T, S, R, K, N) for T in list(range(65, 5000, 7)) + [1 << 20, (1 << 31) - 70000]]
        assert taken == sorted(taken, reverse=True)
    assert not rule.adapters(65, 8, 256, 1 << 20, (1 << 31) - 70000) and not rule.router(1 << 20, 1 << 16, 1 << 20)


def test_the_kernels_for_many_rows_are_reached_at_ordinary_sizes(rule):
    """The sizes at which their bounded waits are tested (test_gpu_more_giveup.py)."""
    for size in ((600, 64, 1024), (2000, 256, 2048), (700, 512, 512)):
        assert not rule.router(*size)
    for size in ((1500, 1, 16, 512, 1024), (600, 1, 64, 512, 2560), (1500, 1, 128, 256, 136)):
        assert not rule.adapters(*size)
