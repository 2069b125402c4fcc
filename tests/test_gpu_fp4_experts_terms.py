"""The experts' intermediate h between the two products: kept as two fp16 terms, 23 bits, against the definition in float64."""
import numpy as np
import pytest
import torch

from oracle import fp4_oracle as F
from tests.test_gpu_fp4_moe import _layer, _run, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,I", [(1, 4, 32), (2, 1, 64), (3, 1, 96), (4, 1, 256), (5, 1, 256), (8, 1, 160), (9, 1, 512), (17, 1, 2048), (33, 2, 288),
                                   (64, 16, 768), (200, 4, 256)])
def test_differences_of_nearly_equal_values(T, E, I, dtype):
    """h_i = silu(3) * (4096 + d_i) with d_i of a few units, and every output the difference of two of them: 11 bits would lose it."""
    H = 64
    rng = np.random.default_rng(T + I)
    steps = np.array([0, 1, 2, 3, 4, 5, 6, 7])  # codes of 0, 0.5, .. 6
    d = rng.choice(steps, size=(E, I))
    c13 = np.zeros((E, 2 * I, H), dtype=np.int64)
    c13[:, :I, 2] = 2                    # gate: 1 * x[2]
    c13[:, I:, 0], c13[:, I:, 1] = 2, d  # up: 1 * x[0] + d * x[1]
    c2 = np.zeros((E, H, I), dtype=np.int64)
    a, b = rng.integers(0, I, size=(2, E, H))
    e, n = np.meshgrid(np.arange(E), np.arange(H), indexing="ij")
    c2[e, n, a] = 2                      # 1
    c2[e, n, b] = np.where(a == b, 0, 10)  # -1
    one = lambda c: np.full(c.shape[:2] + (c.shape[2] // 16,), 0x38, dtype=np.uint8)  # noqa: E731
    w13, w2 = ((F.pack(c), one(c), None) for c in (c13, c2))
    x = torch.zeros(T, H)
    unit = 2.0 ** torch.from_numpy(rng.integers(-2, 3, size=T)).float()  # a row's power of two
    x[:, 0], x[:, 1], x[:, 2] = 4096 * unit, unit, 3
    ids = torch.from_numpy(rng.integers(0, E, size=(T, 1))).to(torch.int32)
    got = _run(x.to(dtype), w13, w2, torch.ones(T, 1), ids).double().cpu().numpy()
    silu3 = 3 / (1 + np.exp(-3.0))
    i = ids[:, 0].numpy()
    value = F.E2M1[d]
    pick = lambda at: np.take_along_axis(value[i], at[i], 1)  # noqa: E731
    want = silu3 * (pick(a) - pick(b)) * unit.numpy()[:, None].astype(np.float64)
    # per value of h: its product is rounded (2^-24), its terms leave 2^-23, and a sum of two of them takes at most four additions of
    # 2^-23 of the larger; the activation's 2^-21 is common to both
    tol = 7 * 2.0**-23 * 4102 * silu3 * unit.numpy()[:, None] + (2.0**-21 + torch.finfo(dtype).eps / 2) * 1.01 * np.abs(want)
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


def _check(got, want, H, I, dtype):
    out, first, second = want
    # first sums: as in test_gpu_fp4_moe; h: an activation good to 2^-20, two terms that leave 2^-23 of a value (and 2^-37 of the row's
    # largest, within the 2^-13 of it that `second` holds a multiple of); second sums: a unit of 2^-23 for every 8 columns of the larger and as
    # many of the lesser terms' 2^-11, the addition of both, eight between warps, a token's slots and two factors
    e1 = (H / 16 + 12) * 2.0**-23 + 2.0**-20
    e2 = 2.0**-23 + 2.0**-20 + (I / 16 * (1 + 2.0**-11) + 21) * 2.0**-23
    tol = e1 * first + e2 * second + torch.finfo(dtype).eps / 2 * np.abs(out) * 1.001 + torch.finfo(dtype).tiny
    err = np.abs(got.double().cpu().numpy() - out)
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,topk,H,I", [(1, 8, 2, 32, 64), (5, 1, 1, 32, 96), (9, 2, 2, 64, 160), (17, 1, 1, 96, 256), (40, 8, 4, 64, 512),
                                          (64, 4, 2, 128, 288), (170, 3, 3, 32, 1056)])
def test_few_columns(T, E, topk, H, I, dtype):
    """Short sums, whose rounding does not hide that of h."""
    args = _layer(T, E, topk, H, I, dtype, 3 * T + E)
    _check(_run(*args), _want(*args), H, I, dtype)


TWICE = [(1, 1, 36096), (3, 2, 36000), (5, 1, 40992)]


@pytest.mark.parametrize("T,E,I", TWICE)
def test_more_columns_than_fit_with_both_terms(T, E, I):
    """Second products whose rows fit shared memory with one term only: the weights are taken twice."""
    args = _layer(T, E, 1, 32, I, torch.bfloat16, I)
    want = _want(*args)
    _check(_run(*args), want, 32, I, torch.bfloat16)
    x = args[0]
    x[0, 3] = float("nan")
    got = _run(*args)
    assert torch.isnan(got[0]).all()
    _check(got[1:], tuple(w[1:] for w in want), 32, I, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,I", [(1024, 7168, 1024), (300, 7168, 1024), (1024, 3616, 1024)])
def test_long_sums(T, H, I, dtype):
    """First products whose up sums climb over half of K and come back to zero: a sum that the matrix instructions carried all the way,
    which cut off what does not fit instead of rounding it, would be left with a share of its peak."""
    from sglang_b200 import ops
    half = H // 2
    gen = torch.Generator().manual_seed(H + T)
    x = torch.randint(128, 256, (T, half), generator=gen).float() / 128
    x[:, 0] = 4
    x = torch.cat([x, x], 1).to(dtype).cuda()
    up = torch.randint(1, 8, (I, half), generator=gen)  # codes of 0.5 to 6, under scales of 2^-4 to 2
    scales = torch.randint(0x18, 0x40, (I, half // 16), generator=gen)
    c13 = torch.zeros(2 * I, H, dtype=torch.uint8)
    c13[:I, 0] = 7  # gate: 6 * 4
    c13[I:] = torch.cat([up, up + 8], 1).to(torch.uint8)
    c2 = torch.zeros(H, I, dtype=torch.uint8)
    c2[torch.arange(I), torch.arange(I)] = 2  # output n is h of n
    one = lambda n, k: torch.full((1, n, k // 16), 0x38, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # noqa: E731
    s13 = torch.cat([torch.full((I, H // 16), 0x38), torch.cat([scales, scales], 1)]).to(torch.uint8).cuda().view(torch.float8_e4m3fn)[None]
    pack = lambda c: torch.from_numpy(F.pack(c.numpy())).cuda()[None]  # noqa: E731
    got = ops.fused_experts_fp4(x, pack(c13), pack(c2), s13, one(H, I), torch.ones(T, 1, device="cuda"),
                                torch.zeros(T, 1, dtype=torch.int32, device="cuda")).double()
    peak = x[:, :half].double() @ torch.from_numpy(F.E2M1[up] * np.repeat(F.E4M3[scales], 16, 1)).cuda().t()
    # A step of 256 columns is 16 instructions, each off by at most 2^-23 of the step's sum so far, which is at most 256 / half of the peak;
    # then a float32 addition of 2^-24 of the sum for each step, and four between warps.  silu(24) is 24 to 2^-34.
    steps = -(-H // 256)
    tol = 24.01 * peak * 2.0**-23 * (steps * 16 * min(1.0, 256 / half) + steps / 2 + 4)
    assert (got[:, I:] == 0).all()
    assert (got[:, :I].abs() <= tol).all(), (got[:, :I].abs() / tol).max()
