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


def test_strides_that_offsets_do_not_hold():
    """64-bit offsets are rows x stride x 2 bytes: strides of 2^40 values and more are refused, before anything is multiplied by them."""
    from sglang_b200._lib import lib
    for T in (1, 4, 5, 100):
        for kw in (dict(ldb=1 << 62, ldo=1 << 62), dict(ldb=1 << 40), dict(ldo=(1 << 63) - 8), dict(ldx=1 << 62)):
            rc, what = _call(T=T, **kw)
            assert rc == -1 and "too large" in what, (T, kw, rc, what)
        assert lib.sglb200_router_logits(A, A, 0, A, T, 8, 64, 1 << 62, None) == -1 and "too large" in lib.sglb200_last_error().decode()
    assert _call(T=1 << 30, ldb=1 << 31, ldo=1 << 31)[0] == -1
    assert _call(ldb=(1 << 40) - 8, ldo=(1 << 40) - 8, ldx=(1 << 40) - 8, ws=None)[0] == -4  # (the next check speaks)
