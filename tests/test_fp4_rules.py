"""Which form of the 4-bit kernels a call takes (csrc/fp4_rules.h), compiled for the CPU; the cases of test_gpu_fp4_forms.py reach all of
them on a GPU of 148 SMs."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sglang_b200", "csrc")
SHIM = """
#include "fp4_rules.h"
using namespace sglb200::fp4;
extern "C" int columns(int64_t m, int64_t n, int64_t k, int64_t pairs) { return pair_columns(m, n, (k + 255) / 256, pairs); }
extern "C" void plan(int64_t slots, int64_t experts, int64_t k, int64_t rows, int up, int64_t sms, ExpertsPlan* p) {
  *p = plan_experts(slots, experts, k, rows, up, sms);
}
extern "C" int64_t smem(int steps, int cols, int stages) { return moe_smem(steps, cols, stages); }
"""
SMS, PAIRS_OF_A_GPU = 148, 74


class Plan(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("steps", "cols", "pass_rows", "warps_k", "sets", "stages")]


def compiled(folder):
    """The rules as a library: columns(m, n, k), plan(slots, experts, k, rows, up), smem(steps, cols, stages)."""
    with open(os.path.join(folder, "shim.cpp"), "w") as f:
        f.write(SHIM)
    so = os.path.join(folder, "shim.so")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I", CSRC, "-o", so, os.path.join(folder, "shim.cpp")])
    lib = ctypes.CDLL(so)
    i64, i32 = ctypes.c_int64, ctypes.c_int
    lib.columns.argtypes, lib.plan.argtypes, lib.smem.argtypes = [i64] * 4, [i64] * 4 + [i32, i64, ctypes.POINTER(Plan)], [i32] * 3
    lib.smem.restype = i64
    return lib


def plan(lib, slots, experts, k, rows, up, sms=SMS):
    p = Plan()
    lib.plan(slots, experts, k, rows, up, sms, ctypes.byref(p))
    return p


def forms(lib, T, E, topk, H, I):
    """(product, K in whole steps, eights of columns or "twice", K split over warps) of both products."""
    out = []
    for up, k, rows in ((1, H, 2 * I), (0, I, H)):
        p = plan(lib, T * topk, E, k, rows, up)
        assert p.stages >= 2
        eights = "twice" if not up and p.cols == 1 else 1 if p.cols <= 8 else 2 if p.cols <= 16 else 4
        out.append(("up" if up else "down", k % 256 == 0, eights, p.warps_k > 1))
    return out


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    return compiled(str(tmp_path_factory.mktemp("fp4_rules")))


def test_plans_fit_and_cover_the_work(rules):
    for slots in (1, 2, 7, 32, 100, 512, 1024):
        for experts in (1, 8, 256, 1024):
            for k in (32, 96, 256, 1056, 2048, 7168, 18432, 36864, 65536):
                for rows in (32, 512, 7168):
                    for up in (0, 1):
                        for sms in (148, 132, 1):
                            p = plan(rules, slots, experts, k, rows * (1 + up), up, sms)
                            assert p.steps == -(-k // 256) and 2 <= p.stages <= 6
                            assert rules.smem(p.steps, p.cols, p.stages) <= 227 * 1024
                            assert p.cols in (1, 2, 4, 8, 16, 32) and 1 <= p.pass_rows <= p.cols * (1 if up else 2)
                            if up:
                                assert p.pass_rows == p.cols
                            else:
                                assert p.pass_rows == max(1, p.cols // 2)
                            assert p.warps_k in (1, 2, 4, 8, 16) and p.warps_k <= p.steps
                            assert p.sets * (16 // p.warps_k) * 16 >= rows * (1 + up)


def test_rows_that_do_not_fit(rules):
    """69120 columns are the most that the header promises; what does not fit is refused before anything is launched."""
    from sglang_b200._lib import lib
    A, size = 4096, lib.sglb200_fused_experts_fp4_workspace_bytes  # A: an aligned address that is never touched
    for slots in (1, 4, 1024):
        for up in (0, 1):
            assert plan(rules, slots, 8, 69120, 64, up).stages >= 2 and plan(rules, slots, 8, 69120 + 32, 64, up).stages == 0
    for H, I in ((69120 + 32, 64), (64, 69120 + 32), (1 << 30, 32)):
        rc = lib.sglb200_fused_experts_fp4(A, 0, A, A, None, A, A, None, A, A, A, 2, 2, 8, H, I, 1.0, A, size(2, 2, H, I), None)
        assert rc == -1 and b"too many" in lib.sglb200_last_error()


def test_the_widths_of_pairs_tiles(rules):
    for m in (129, 257, 700, 4096, 9000):
        for n in (8, 104, 640, 2112, 10240, 36864):
            for k in (32, 1056, 7168):
                for pairs in (74, 66, 1):
                    assert rules.columns(m, n, k, pairs) in (128, 192, 256)
    # figures of the rule's comment
    assert rules.columns(4096, 36864, 7168, PAIRS_OF_A_GPU) == 256 and rules.columns(1024, 10240, 8192, PAIRS_OF_A_GPU) == 192
    assert rules.columns(1024, 2112, 7168, PAIRS_OF_A_GPU) == 128


def test_the_gpu_tests_reach_every_form(rules):
    from tests.test_gpu_fp4_experts_terms import TWICE
    from tests.test_gpu_fp4_forms import EXPERTS, PAIRS
    from tests.test_gpu_fp4_moe import CASES
    reached = {f for c in CASES + EXPERTS for f in forms(rules, *c)} | {f for T, E, I in TWICE for f in forms(rules, T, E, 1, 32, I)}
    for whole in (False, True):
        for split in (False, True):
            for eights in (1, 2, 4):
                assert ("up", whole, eights, split) in reached
                assert ("down", whole, eights, split) in reached
        assert any(f[:3] == ("down", whole, "twice") for f in reached)
    for m, n, k, columns in PAIRS:
        assert rules.columns(m, n, k, PAIRS_OF_A_GPU) == columns
        assert -(-m // 64) * -(-n // 128) > SMS  # (pairs, not rows)
        assert -(-m // 256) * -(-n // columns) > PAIRS_OF_A_GPU  # several tiles a pair
    assert {c for *_, c in PAIRS} == {128, 192, 256}
