"""Numbers that a sum or a product of 64 bits does not hold, at the C entry of `lora_add` (no GPU needed: all are refused)."""
import ctypes

A = 4096  # an aligned address that is never touched
BIG = (1 << 63) - 1


def _call(**kw):
    from sglang_b200._lib import lib
    a = {**dict(x=A, a=A, b=A, base=A, out=A, T=4, L=2, R=16, N=64, K=128, ldx=128, ldb=64, ldo=64, sizes=(64,), ws=A, bytes=1 << 30), **kw}
    sizes = (ctypes.c_int64 * len(a["sizes"]))(*a["sizes"])
    rc = lib.sglb200_lora_add(a["x"], a["a"], a["b"], a["base"], a["out"], 0, A, None, None, a["T"], a["L"], a["R"], a["N"], a["K"], a["ldx"],
                              a["ldb"], a["ldo"], len(a["sizes"]), sizes, a["ws"], a["bytes"], None)
    return rc, lib.sglb200_last_error().decode()


def test_slices_whose_sum_wraps_around():
    for sizes in ((1, BIG, BIG, 65), (BIG, BIG, 66), (BIG, 66, BIG), (32, BIG, BIG, 34)):
        assert (sum(sizes) + (1 << 63)) % (1 << 64) - (1 << 63) == 64
        rc, what = _call(sizes=sizes)
        assert rc == -1 and "more than 64 columns" in what, (sizes, rc, what)
