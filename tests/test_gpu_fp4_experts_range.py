"""The experts of a few tokens at the ends of the ranges: factors, and rows whose power of two is not the usual one."""
import numpy as np
import pytest
import torch

from oracle import fp4_oracle as F
from tests.test_gpu_fp4_moe import _layer, _run, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("a13,a2,xs", [(2.0**100, 1.0, 2.0**-100), (2.0**-100, 1.0, 2.0**100), (2.0**100, 2.0**-60, 2.0**-85), (1.0, 2.0**100, 2.0**-60),
                                       (2.0**-60, 2.0**100, 2.0**20), (2.0**-80, 2.0**-20, 2.0**110)])
def test_large_and_small_factors(a13, a2, xs):
    """A factor is 1 / the weights' global scale, 2^-100 to 2^100, beside rows that make up for it."""
    x, w13, w2, weights, ids = _layer(6, 4, 2, 256, 160, torch.bfloat16, 21)
    w13, w2 = (w[:2] + (np.full(4, a, dtype=np.float32),) + w[3:] for w, a in ((w13, a13), (w2, a2)))
    # gates and ups that add up: the largest weights, all of one sign, and a row beside them that is not negative
    codes, scode = np.full_like(w13[0], 0x77), np.full_like(w13[1], 0x7E)
    w13 = (codes, scode, w13[2], F.dequantize(codes, scode, 16))
    x = x.abs()
    x = (x.double() * xs).to(torch.bfloat16)
    with np.errstate(over="ignore"):
        out, first, second = _want(x, w13, w2, weights, ids)
    got = _run(x, w13, w2, weights, ids)
    # the tolerance of test_gpu_fp4_moe without its absolute term: every value is far from the ends of bf16
    e1, e2 = (256 / 16 + 12) * 2.0**-23 + 2.0**-20, 2.0**-20 + (160 / 16 + 20) * 2.0**-23
    tol = e1 * first + e2 * second + 2.0**-8 * 1.001 * np.abs(out)
    assert 1e-30 < np.abs(out).max() < 1e37
    assert (np.abs(got.double().cpu().numpy() - out) <= tol).all()
