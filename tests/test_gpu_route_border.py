"""Experts that cannot be told apart in float32 at the border of the picks, exact ties among them (`route_topk`)."""
import numpy as np
import pytest
import torch

from oracle import more_oracle as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0**-23


def _ids(x, topk, scoring="softmax", bias=None, groups=1, kept=1, top=1):
    from sglang_b200 import ops
    return ops.route_topk(x.cuda(), topk, scoring, None if bias is None else bias.cuda(), groups, kept, top)[1].cpu()


def _check(x, topk, scoring="softmax", bias=None, groups=1, kept=1, top=1):
    got = _ids(x, topk, scoring, bias, groups, kept, top)
    _, want = O.route(x.double().numpy(), topk, scoring, None if bias is None else bias.double().numpy(), groups, kept, top)
    np.testing.assert_array_equal(got.numpy(), want)


def _sorted_ids(x, topk, scoring, bias):
    """Without groups, one bias for all: larger c in float64 first, then the larger logit, then the lower expert."""
    xd, by_logit = torch.sort(x.double(), dim=-1, descending=True, stable=True)
    c = (torch.sigmoid(xd) if scoring == "sigmoid" else torch.softmax(xd, -1)) + bias.double()[0]
    return by_logit.gather(1, torch.sort(c, dim=-1, descending=True, stable=True)[1])[:, :topk].to(torch.int32)


@pytest.mark.parametrize("first,want", [([1, 1, 1 + U], 2), ([1, 1 + U, 1 + U, 1 + 2 * U], 3), ([1, 1, 1, 1 + U], 3), ([1, 1, 1, 1], 0),
                                        ([1, 1 + U, 1, 1], 1), ([1 + U, 1, 1 + U, 1], 0)])
def test_one_pick_of_a_few(first, want):
    x = torch.full((5, 64), -1.0)
    x[:, : len(first)] = torch.tensor(first, dtype=torch.float64).float()
    x[1] = x[1].flip(0)  # the same in other lanes
    x[2] = x[2].roll(31)
    x[3] = x[3].view(16, 4).t().reshape(-1)  # one to a lane
    assert _ids(x, 1)[0, 0] == want
    for scoring in ("softmax", "sigmoid"):
        _check(x, 1, scoring)
        _check(x, 1, scoring, None, 4, 2, 1)
        _check(x, 1, scoring, torch.full((64,), 0.25), 8, 3, 2)


@pytest.mark.parametrize("topk", [1, 2, 8, 29, 30, 31, 32])
@pytest.mark.parametrize("tie", [2, 3, 4, 33, 60])
def test_a_larger_one_behind_a_run_of_equal_ones(topk, tie):
    """`topk` - 1 picks beyond doubt, then `tie` equal experts, then one a unit or a few larger or smaller."""
    E = 128
    for step in (-3, -1, 1, 2):
        x = torch.full((3, E), -4.0)
        x[:, :tie] = 1.0
        x[:, tie + 3] = 1.0 + step * U
        x[:, E - topk + 1 :] = 8.0 + torch.arange(topk - 1).float()
        x[1] = x[1].view(4, 32).t().reshape(-1)
        x[2] = x[2].flip(0)
        _check(x, topk)
        for bias in (torch.zeros(E), torch.full((E,), -0.5)):
            _check(x, topk, "sigmoid", bias)
        _check(x, min(topk, 8), "softmax", torch.full((E,), 0.5), 4, 3, 2)


@pytest.mark.parametrize("topk", [2, 3, 5, 8])
def test_equal_ones_between_close_ones(topk):
    """P ? Q, Q = R, R ? S at every place around the border, in any order of the indices."""
    g = torch.Generator().manual_seed(topk)
    for shift in range(4):
        rows = []
        for _ in range(12):
            offs = torch.tensor([1.0, 0.0, 0.0, -1.0, 0.0, 1.0])[torch.randperm(6, generator=g)] * U * (1 + shift)
            x = torch.full((96,), -3.0)
            x[:topk - 1] = 6.0 + torch.arange(topk - 1).float()
            x[topk : topk + 6] = 1.0 + offs
            x[topk : topk + shift] = 5.0 - shift
            rows.append(x[torch.randperm(96, generator=g)])
        x = torch.stack(rows)
        _check(x, topk)
        _check(x, topk, "sigmoid", torch.full((96,), 0.125))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_fewer_experts_than_looks(scoring):
    """Rows whose last available experts are equal or close: nothing is behind them."""
    x = torch.full((4, 40), -float("inf"))
    x[0, [3, 9]] = 1.0
    x[1, [3, 9, 20]] = torch.tensor([1.0, 1.0, 1.0 + U])
    x[2, [3, 9, 20, 39]] = torch.tensor([1.0, 1.0, 1.0, 1.0 + U])
    x[3, [0, 1]] = torch.tensor([1.0, 1.0 + U])
    for topk in (1, 2, 3, 4, 6):
        _check(x, topk, scoring)
        _check(x, topk, scoring, torch.zeros(40))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("mean,std", [(8, 1), (10, 1), (0, 6), (12, 2)])
@pytest.mark.parametrize("constant", [0.0, 0.5])
def test_saturated_sigmoids_and_one_bias_for_all(dtype, mean, std, constant):
    """Large scores share their leading bits, and 16-bit logits have equal pairs everywhere."""
    x = (torch.randn(2000, 256, generator=torch.Generator().manual_seed(mean * 7 + std)) * std + mean).to(DT[dtype])
    bias = torch.full((256,), constant)
    for topk in (1, 6, 8):
        assert torch.equal(_ids(x, topk, "sigmoid", bias), _sorted_ids(x, topk, "sigmoid", bias))
    _check(x[:120], 8, "sigmoid", bias, 8, 4, 2)
    _check(x[:120], 8, "sigmoid", bias, 8, 4, 1)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("topk", [1, 8, 30])
def test_softmax_and_one_bias_for_all(dtype, topk):
    x = (torch.randn(2000, 256, generator=torch.Generator().manual_seed(topk)) * 5).to(DT[dtype])
    bias = torch.full((256,), 0.5)
    want = _sorted_ids(x, topk, "softmax", bias)
    # (scores below 2^-53 of the bias are equal to float64, and which goes first is not asked here)
    s = torch.softmax(x.double(), -1)
    asked = s.gather(1, want.long())[:, -1] > 2.0**-40
    assert asked.any()
    assert torch.equal(_ids(x, topk, "softmax", bias)[asked], want[asked])


@pytest.mark.parametrize("topk", [1, 2, 8, 31])
def test_logits_from_a_few_values(topk):
    """Rows of a few neighbouring float32 values: runs of equal and close ones of every length, at every border."""
    g = torch.Generator().manual_seed(topk)
    for E in (33, 64, 256, 1000):
        for spread in (2, 4, 40):
            x = 1.0 + torch.randint(0, spread, (300, E), generator=g) * U
            x = torch.where(torch.rand(300, E, generator=g) < 0.5, x, -x - 1.0).float()
            want = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :topk].to(torch.int32)
            assert torch.equal(_ids(x, topk), want)
