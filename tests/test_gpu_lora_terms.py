"""The two 16-bit terms in which h = A x enters the adapters' second product (`lora_add`)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
BITS = {"bf16": 8, "fp16": 11}
# tokens and ranks that reach every form of the second product: up to 64 tokens, sorted blocks of 32 rows and of 128, ranks of one to eight spans
FORMS = [(1, 8), (1, 256), (7, 32), (40, 64), (64, 128), (90, 16), (200, 40), (200, 256), (257, 128), (1100, 16), (1500, 64), (700, 128), (600, 200)]


def _run(base, x, a, b, ids, scalings=None):
    from sglang_b200 import ops
    d = [t.cuda() for t in (base, x, a, b, ids)]
    return ops.lora_add(*d, None if scalings is None else scalings.cuda()).cpu()


def _pairs(T, R, dtype, seed, spread):
    """x and A whose h is exact in float32 and takes all 2 p bits of two terms of p: h_r = 2^-m_r (u + 2^-p v), u and v of p bits.
    (x, a, h float64 [T, R], m)"""
    g = torch.Generator().manual_seed(seed)
    p = BITS[dtype]
    u = torch.randint(1 << (p - 1), 1 << p, (T, R), generator=g) * (torch.randint(0, 2, (T, R), generator=g) * 2 - 1)
    v = torch.randint(-(1 << p) + 1, 1 << p, (T, R), generator=g) | 1
    x = torch.stack([u.double() * 2.0 ** (1 - p), v.double() * 2.0 ** (1 - 2 * p)], -1).view(T, 2 * R)
    m = torch.randint(0, spread + 1, (R,), generator=g)
    m[0] = 0
    a = torch.zeros(2, R, 2 * R, dtype=torch.float64)
    r = torch.arange(R)
    a[:, r, 2 * r] = a[:, r, 2 * r + 1] = 2.0 ** -m.double()
    assert torch.equal(x.to(DT[dtype]).double(), x)
    return x.to(DT[dtype]), a.to(DT[dtype]), x @ a[0].t(), m


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,R", FORMS)
@pytest.mark.parametrize("spread", [0, 14])
def test_no_bit_of_two_terms_is_lost(T, R, dtype, spread):
    """Every out is the sum of two h (times the power of two that makes up for 2^-m) plus base = -(that sum, rounded): what is left are the
    bits behind the first p, which two terms hold and out holds as well.  h is up to 2^-`spread` of its row's largest.

    The products are exact; a partial sum is a whole number of units of 2^(1 - 2 p) below 2^(2 p + 1) of them, at most 2^23: float32 holds it."""
    N = 200
    x, a, h, m = _pairs(T, R, dtype, T + R + spread, spread)
    g = torch.Generator().manual_seed(T * R)
    first = torch.randint(0, R, (2, N), generator=g)
    second = (first + torch.randint(1, R, (2, N), generator=g)) % R
    sign = torch.randint(0, 2, (2, N, 2), generator=g).double() * 2 - 1
    b = torch.zeros(2, N, R, dtype=torch.float64)
    b.scatter_(2, first[..., None], sign[..., :1] * 2.0 ** m[first][..., None].double())
    b.scatter_(2, second[..., None], sign[..., 1:] * 2.0 ** m[second][..., None].double())
    ids = (torch.arange(T) * 2 // T).to(torch.int32) if T % 2 else torch.randint(0, 2, (T,), generator=g).to(torch.int32)
    sums = torch.einsum("tr,tnr->tn", h, b[ids.long()]) if T * N * R < 3e7 else torch.stack([h[t] @ b[ids[t]].t() for t in range(T)])
    base = -sums.to(DT[dtype])
    want = sums + base.double()
    assert torch.equal(want.to(DT[dtype]).double(), want) and want.ne(0).any()
    got = _run(base, x, a, b.to(DT[dtype]), ids)
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,R", FORMS)
def test_random_values_against_what_two_terms_keep(T, R, dtype):
    """base = -(the sum, rounded) again, so that the error of the sum is not hidden behind the rounding of out.

    K = 64: the first product is 4 instructions and the sum of at most 64 parts, each off by at most 2 units of 2^-24 (2 x 4 + 64).  Two terms are
    off by 2^-16 of h (8 bits and 8) or 2^-22 (11 and 11), and by half of float16's smallest step, 2^-25, where the row's largest is at
    least 2^14.  The second product is an instruction per 16 values of the rank and term, each off by 2 units of 2^-23 at most."""
    K, N, L = 64, 136, 3
    g = torch.Generator().manual_seed(T * 3 + R)
    x = torch.randn(T, K, generator=g).to(DT[dtype])
    a = (torch.randn(L, R, K, generator=g) * torch.exp2(torch.randint(-6, 1, (L, R, 1), generator=g).float())).to(DT[dtype])
    b, ids = torch.randn(L, N, R, generator=g).to(DT[dtype]), torch.randint(0, L, (T,), generator=g).to(torch.int32)
    scalings = torch.tensor([1.0, 0.5, 2.0])
    want, tol = torch.empty(T, N, dtype=torch.float64), torch.empty(T, N, dtype=torch.float64)
    for l in range(L):
        rows = ids == l
        xd, ad, bd, s = x[rows].double(), a[l].double(), b[l].double(), float(scalings[l])
        h = xd @ ad.t() * s
        want[rows] = h @ bd.t()
        of_h = (2 * 4 + 64) * 2.0**-24 * s * (xd.abs() @ ad.abs().t())
        of_h += 2.0 ** (-2 * BITS[dtype]) * h.abs() + (2.0**-39 * h.abs().amax(1, keepdim=True) if dtype == "fp16" else 0)
        tol[rows] = of_h @ bd.abs().t() + (R + 15) // 16 * 2 * 2 * 2.0**-23 * (h.abs() @ bd.abs().t())
    base = -want.to(DT[dtype])
    want += base.double()
    eps = torch.finfo(DT[dtype]).eps / 2
    tol = tol * 1.01 + eps * (want.abs() + tol) + torch.finfo(DT[dtype]).tiny * eps
    err = (_run(base, x, a, b, ids, scalings).double() - want).abs()
    assert (err <= tol).all(), (err / tol).max()
