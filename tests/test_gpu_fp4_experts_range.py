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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_of_all_magnitudes(dtype):
    """Rows that are staged under another power of two than the usual one, as x and as h, each with an expert of its own whose factor brings the
    output back to ordinary numbers; 2^6 would flush the small ones to zero and take the large ones to infinity."""
    powers = [-60, -45, -30, -20, -12, -7, -3, 0, 4, 7, 9, 12, 16, 30, 45, 58] if dtype == torch.bfloat16 else [-9, -7, -5, -3, 0, 2, 4, 6, 8, 10]
    n = len(powers)
    x, w13, w2, weights, _ = _layer(n, n, 1, 512, 288, dtype, 22)
    x = (x.double() * 2.0 ** torch.tensor(powers, dtype=torch.float64)[:, None]).to(dtype)
    # silu(v) is v / 2 for small v: h goes as the square either way
    w13 = w13[:2] + (np.full(n, 1e-2, dtype=np.float32),) + w13[3:]
    w2 = w2[:2] + ((2.0 ** (-2.0 * np.array(powers)) * 1e-2).astype(np.float32),) + w2[3:]
    ids = torch.arange(n, dtype=torch.int32)[:, None]
    with np.errstate(over="ignore"):
        out, first, second = _want(x, w13, w2, weights, ids)
    got = _run(x, w13, w2, weights, ids).double().cpu().numpy()
    # as above; fp16 outputs may be subnormal: half of their step
    e1, e2 = (512 / 16 + 12) * 2.0**-23 + 2.0**-20, 2.0**-20 + (288 / 16 + 20) * 2.0**-23
    tol = e1 * first + e2 * second + torch.finfo(dtype).eps / 2 * 1.001 * np.abs(out)
    if dtype == torch.float16:
        tol += 2.0**-25
    err = np.abs(got - out)
    assert (np.abs(out).max(1) > 1e-3).all() and (np.abs(out).max(1) < 6e4).all()
    for row, p in enumerate(powers):
        assert (err[row] <= tol[row]).all(), (p, (err[row] / tol[row]).max())
        assert (err[row] ** 2).mean() <= (torch.finfo(dtype).eps / 2) ** 2 * (out[row] ** 2).mean(), p


@pytest.mark.parametrize("H,I", [(69120, 32), (69088, 64), (64, 69120), (32, 69088)])
def test_longest_rows(H, I):
    """The most columns of either product, where one row at a time is staged."""
    from tests.test_gpu_fp4_experts_terms import _check
    args = _layer(3, 1, 1, H, I, torch.bfloat16, 23)
    _check(_run(*args), _want(*args), H, I, torch.bfloat16)
