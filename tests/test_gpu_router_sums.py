"""How exact the router's sums are (`router_logits`): K in parts that begin from zero, against float64."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _bound(T, E, K):
    """Of the sum of the products' magnitudes, in 2^-24: an instruction cuts off less than a unit (2^-23, 2 here) of its sum and as much of the
    16 products that it adds; a float32 addition is off by half a unit (1).  Sums in tensor memory take 256 columns, 16 instructions, and
    meet over K / 256 additions (a partial sum is as large as its share of the columns: half of them count); the small kernel's 64 warps take
    two instructions for every 32 columns of theirs.  Up to eight parts of a cluster, and eight of a CTA, are added up at the end."""
    if T * E > 32768:
        return 4 * 16 + (K // 256) / 2 + 1 + 8
    return 4 * 2 * -(-K // (32 * 64)) + 8 + 8


# both kernels: one with 64 parts of K (a tile or few), one with pieces of 256 columns, with K in one piece and split over a cluster
SIZES = [(1, 16, 65536), (8, 16, 65536), (32, 16, 16384), (600, 64, 65536), (2100, 256, 16384), (5000, 200, 8192), (257, 256, 32768)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("one_sign", [True, False])
@pytest.mark.parametrize("T,E,K", SIZES)
def test_sums_of_long_rows(T, E, K, one_sign, dtype):
    """Products of one sign: what is cut off adds up, and one sum over all of K would lose a third of a unit for each of its K / 16 instructions,
    1365 in 2^-24 for 65536 columns."""
    from sglang_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(T + E + K)
    x, w = torch.randn(T, K, generator=g, device="cuda"), torch.randn(E, K, generator=g, device="cuda") * 0.05
    if one_sign:
        x, w = x.abs(), w.abs()
    x, w = x.to(DT[dtype]), w.to(DT[dtype])
    got = ops.router_logits(x, w)
    wd = w.double().t().contiguous()
    worst = 0.0
    for i in range(0, T, 512):
        xd = x[i : i + 512].double()
        worst = max(worst, ((got[i : i + 512].double() - xd @ wd).abs() / (xd.abs() @ wd.abs())).max().item())
    assert worst <= _bound(T, E, K) * 2.0**-24, (worst * 2**24, _bound(T, E, K))


@pytest.mark.parametrize("T", [1, 3, 9, 70, 700])
def test_a_row_without_a_leading_dimension(T):
    from sglang_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, 1024, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(40, 1024, generator=g, device="cuda").to(torch.bfloat16)
    for row in (x[0], x[T - 1], x[T // 2]):
        got = ops.router_logits(row, w)
        assert got.shape == (40,) and got.dtype == torch.float32
        err = (got.double() - w.double() @ row.double()).abs()
        assert (err <= _bound(1, 40, 1024) * 2.0**-24 * (w.double().abs() @ row.double().abs())).all()
        assert torch.equal(got, ops.router_logits(row[None], w)[0])
