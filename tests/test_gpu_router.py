"""The router's product (`router_logits`) against float64."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _check(x, w):
    from sglang_b200 import ops
    got = ops.router_logits(x, w)
    K = x.shape[-1]
    assert got.dtype == torch.float32 and got.shape == x.shape[:-1] + (w.shape[0],)
    want = x.double() @ w.double().t()
    mass = x.double().abs() @ w.double().abs().t()
    # products of 16-bit numbers are exact in float32; an instruction adds 16 of them to a sum and cuts off at most two units of what it
    # adds up, and up to 64 parts of K are added up after that
    tol = ((K + 15) // 16 * 2 + 64) * 2.0**-24 * mass
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (err <= tol).all(), (err / tol).max()


SIZES = [(1, 256, 7168), (1, 1, 8), (2, 8, 256), (7, 160, 5120), (8, 33, 1000), (9, 64, 2048), (16, 17, 24), (17, 128, 2048), (64, 128, 2048),
         (65, 256, 7168), (130, 160, 1288), (511, 160, 5120), (1000, 96, 264), (2049, 256, 1024), (300, 512, 4096), (5, 1000, 520)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,E,K", SIZES)
def test_router(T, E, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(T + E + K)
    x = torch.randn(T, K, generator=g, device="cuda").to(DT[dtype])
    w = (torch.randn(E, K, generator=g, device="cuda") * 0.02).to(DT[dtype])
    _check(x, w)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,E,K", SIZES + [(8192, 256, 7168), (4100, 40, 8184)])
def test_whole_numbers_are_exact(T, E, K, dtype):
    """Sums of small whole numbers, none of which is rounded: every term of every sum has to be there once."""
    from sglang_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(T * 3 + E + K)
    x = torch.randint(-3, 4, (T, K), generator=g, device="cuda").to(DT[dtype])
    w = torch.randint(-3, 4, (E, K), generator=g, device="cuda").to(DT[dtype])
    got = ops.router_logits(x, w)
    assert torch.equal(got.double(), x.double() @ w.double().t())


@pytest.mark.parametrize("T", [3, 70, 700, 1300])
def test_rows_apart_and_leading_dimensions(T):
    from sglang_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(T)
    wide = torch.randn(T, 1024 + 64, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(40, 1024, generator=g, device="cuda").to(torch.bfloat16)
    _check(wide[:, 64:], w)
    x = wide[:, :1024].contiguous()
    assert torch.equal(ops.router_logits(x.view(1, T, 1024), w)[0], ops.router_logits(x, w))
    assert torch.equal(ops.router_logits(x[0], w), ops.router_logits(x, w)[0]) or T > 8  # (another split of K: another rounding)


def test_no_tokens():
    from sglang_b200 import ops
    assert tuple(ops.router_logits(torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16)).shape) == (0, 4)


@pytest.mark.parametrize("T", [4, 100, 600, 1500])
def test_infinities_and_nan_stay_in_their_rows(T):
    from sglang_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, 512, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(24, 512, generator=g, device="cuda").to(torch.bfloat16)
    want = ops.router_logits(x, w)
    x[1, 5], x[2, 7] = float("nan"), float("inf")
    got = ops.router_logits(x, w)
    keep = [t for t in range(T) if t not in (1, 2)]
    assert torch.equal(got[keep], want[keep]) and got[1].isnan().all() and not got[2].isfinite().any()


@pytest.mark.parametrize("E", [8, 512])
def test_offsets_beyond_32_bits(E):
    from sglang_b200 import ops
    T, K, apart = 130, 64, (1 << 24) + 512  # the last rows begin behind 2^31 values
    wide = torch.empty(T * apart, device="cuda", dtype=torch.bfloat16).view(T, apart)
    g = torch.Generator(device="cuda").manual_seed(E)
    x = torch.randn(T, K, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(E, K, generator=g, device="cuda").to(torch.bfloat16)
    wide[:, :K] = x
    assert torch.equal(ops.router_logits(wide[:, :K], w), ops.router_logits(x, w))
