"""Scores that float64 does not tell apart (`route_topk`): where the biases are equal the logits decide, as without a bias."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _ids(x, topk, scoring, bias=None, groups=1, kept=1, top=1):
    from sglang_b200 import ops
    return ops.route_topk(x.cuda(), topk, scoring, None if bias is None else bias.cuda(), groups, kept, top)[1].cpu()


def _logits(T, E, std, dtype, seed):
    x = torch.randn(T, E, generator=torch.Generator().manual_seed(seed)) * std
    x[0] = 60.0  # all of them saturated, and equal
    x[1] = 60.0 + torch.arange(E) % 7
    x[2] = torch.arange(E) * 0.5
    return x.to(DT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("scoring,std", [("sigmoid", 30.0), ("sigmoid", 400.0), ("softmax", 400.0)])
@pytest.mark.parametrize("E,topk", [(33, 33), (64, 8), (256, 8), (1000, 32)])
def test_one_bias_for_all_leaves_the_order_of_the_logits(E, topk, scoring, std, dtype):
    topk = min(topk, 32)
    x = _logits(40, E, std, dtype, E)
    want = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][:, :topk].to(torch.int32)
    assert torch.equal(_ids(x, topk, scoring), want)
    for constant in (0.0, 0.5, -3.0):
        assert torch.equal(_ids(x, topk, scoring, torch.full((E,), constant)), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("scoring,std", [("sigmoid", 30.0), ("softmax", 400.0)])
@pytest.mark.parametrize("E,topk,groups,kept", [(64, 6, 8, 3), (256, 8, 8, 4), (96, 4, 3, 2), (512, 8, 32, 5)])
def test_groups_by_their_best(E, topk, groups, kept, scoring, std, dtype):
    x = _logits(40, E, std, dtype, E + 1)
    want = _ids(x, topk, scoring, None, groups, kept)
    f = x.float().view(40, groups, -1)
    stay = torch.sort(f.amax(-1), dim=-1, descending=True, stable=True)[1][:, :kept]
    keep = torch.zeros(40, groups, dtype=torch.bool).scatter_(1, stay, True)
    by_hand = torch.sort(f.masked_fill(~keep[..., None], -torch.inf).view(40, E), dim=-1, descending=True, stable=True)[1][:, :topk]
    assert torch.equal(want, by_hand.to(torch.int32))
    assert torch.equal(_ids(x, topk, scoring, torch.zeros(E), groups, kept), want)
    assert torch.equal(_ids(x, topk, scoring, torch.full((E,), 2.0), groups, kept), want)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_two_classes_of_biases(scoring):
    """Odd experts a bias of 4 and even ones none: each class in the order of its logits, the favoured one first."""
    x = _logits(40, 128, 300.0, "fp32", 5)
    bias = torch.zeros(128)
    bias[1::2] = 4.0
    odd = torch.sort(x[:, 1::2], dim=-1, descending=True, stable=True)[1][:, :10] * 2 + 1
    assert torch.equal(_ids(x, 10, scoring, bias), odd.to(torch.int32))
    bias[1::2] = -4.0
    even = torch.sort(x[:, 0::2], dim=-1, descending=True, stable=True)[1][:, :10] * 2
    assert torch.equal(_ids(x, 10, scoring, bias), even.to(torch.int32))
