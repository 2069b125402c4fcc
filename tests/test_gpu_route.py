"""Routing (`route_topk`) against its definition in float64: ids equal, weights within the roundings that they meet."""
import math

import numpy as np
import pytest
import torch

from oracle import more_oracle as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _check(x, topk, scoring="softmax", bias=None, groups=1, kept=1, top=1, renorm=True, factor=1.0):
    from sglang_b200 import ops
    w, ids = ops.route_topk(x.cuda(), topk, scoring, None if bias is None else bias.cuda(), groups, kept, top, renorm, factor)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32 and tuple(w.shape) == tuple(ids.shape) == (x.shape[0], topk)
    xn = x.double().numpy()
    want_w, want_i = O.route(xn, topk, scoring, None if bias is None else bias.double().numpy(), groups, kept, top, renorm, factor)
    np.testing.assert_array_equal(ids.cpu().numpy(), want_i)
    # a difference of two logits (half a unit of up to 300, beyond which the exponential is 0), an exponential (2 units), a sum of E
    # or topk such terms (up to 10 roundings), a quotient and three products or sums: relative to the weight
    fin = np.abs(xn[np.isfinite(xn)])
    reach = min(300.0, 2 * float(fin.max())) if fin.size else 0.0
    rel = (reach / 2 + 2 + 2 + 10 + 4) * 2.0**-23
    np.testing.assert_allclose(w.cpu().double().numpy(), want_w, rtol=rel, atol=abs(factor) * 2.0**-126)


def _logits(T, E, seed, dtype="fp32", std=1.5):
    return (torch.randn(T, E, generator=torch.Generator().manual_seed(seed)) * std).to(DT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,topk,groups,kept", [(1, 256, 8, 8, 4), (3, 160, 6, 8, 3), (70, 64, 6, 1, 1), (33, 7, 7, 1, 1), (257, 96, 10, 16, 5),
                                                  (9, 1024, 32, 4, 2), (5, 1, 1, 1, 1), (40, 66, 4, 3, 2), (17, 512, 3, 32, 7), (300, 128, 8, 2, 1)])
def test_route(T, E, topk, groups, kept, scoring, dtype):
    x = _logits(T, E, T * 1000 + E, dtype)
    bias = torch.randn(E, generator=torch.Generator().manual_seed(E)) * (0.1 if scoring == "sigmoid" else 0.2 / E)
    for b, top, renorm in ((None, 1, True), (None, 2, False), (bias, 2, True), (bias, 1, False)):
        _check(x, topk, scoring, b, groups, kept, top, renorm, factor=2.5)


def test_many_rows():
    x = _logits(5001, 256, 5)
    bias = torch.randn(256, generator=torch.Generator().manual_seed(6)) * 0.1
    _check(x, 8, "sigmoid", bias, 8, 4, 2, True, 2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 3)])
def test_scores_that_float32_cannot_tell_apart(scoring, groups, kept):
    """The bias undoes the scores up to its own rounding: the order of c is that of those roundings, 2^-26 apart and less."""
    for seed in range(20):
        x = _logits(1, 64, seed)
        xd = x.double()
        s = torch.softmax(xd, -1) if scoring == "softmax" else torch.sigmoid(xd)
        bias = (0.75 - s[0]).float()
        for top in (1, 2):
            _check(x.repeat(3, 1), 8, scoring, bias, groups, kept, top)


@pytest.mark.parametrize("topk", [1, 5, 30, 31, 32])
def test_neighbours_at_the_border_of_the_picks(topk):
    """Runs of experts a few float32 units apart, in any order, of which the border of the picks cuts one."""
    for seed in range(6):
        g = torch.Generator().manual_seed(100 + seed)
        base = (torch.arange(96) // 3).float()[torch.randperm(96, generator=g)] * 0.125 - 2.0
        x = base + torch.randint(-2, 3, (3, 96), generator=g) * 2.0**-23
        _check(x, topk, "softmax")
        _check(x, topk, "sigmoid", groups=4, kept=2, top=2)
        _check(x, topk, "softmax", groups=8, kept=4, top=1)
        bias = (torch.randint(0, 4, (96,), generator=g) * 0.25 - torch.sigmoid(x[0].double())).float()
        _check(x, topk, "sigmoid", bias)
        _check(x, topk, "softmax", bias * 0.01, 4, 2, 2, renorm=False)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_sums_of_large_biases_that_cancel(scoring):
    """A group's two largest c of opposite signs: their sum is far smaller than what each is rounded by."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(20, 32, generator=g)
    bias = torch.full((32,), -5000.0)
    bias[0::4], bias[1::4] = 1000.0, -1000.0 + torch.arange(8) * 2.0**-13
    _check(x, 4, scoring, bias, 8, 3, 2)


def test_logits_far_from_zero():
    """Differences that float32 logits hold in their last bits, far below a score's."""
    g = torch.Generator().manual_seed(4)
    x = (3.0e4 + torch.randint(0, 40, (30, 64), generator=g) * 2.0**-9).float()
    for top in (1, 2):
        _check(x, 6, "softmax", None, 8, 3, top)
        _check(-x, 6, "softmax", None, 8, 3, top)
    x = torch.where(torch.rand(30, 64, generator=g) < 0.7, x - 2000.0, x)  # most scores are nothing even in float64
    _check(x, 6, "softmax", None, 8, 3, 1)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_ties_go_to_the_lower_index(scoring):
    x = torch.zeros(4, 64)
    x[1, 5::7] = 1.0
    x[2] = -0.0
    x[2, ::2] = 0.0
    x[3] = torch.arange(64) // 16
    for bias in (None, torch.zeros(64), torch.full((64,), -0.25)):
        _check(x, 9, scoring, bias, 8, 3, 2)
        _check(x, 9, scoring, bias, 1, 1, 1, renorm=False)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept,top", [(1, 1, 1), (4, 2, 1), (4, 2, 2)])
def test_masked_experts_and_rows(scoring, groups, kept, top):
    """-inf, NaN and the type's lowest value among the logits; rows with less than topk experts, and with none."""
    for dtype in ("bf16", "fp16", "fp32"):
        x = _logits(8, 32, 3, dtype)
        low = torch.finfo(DT[dtype]).min
        x[0, :] = -math.inf
        x[1, :] = math.nan
        x[2, 1:] = -math.inf
        x[3, ::2], x[3, 1::4] = -math.inf, math.nan
        x[4, :] = low
        x[5, 3:] = low
        x[6, 7], x[6, 9] = math.inf, math.inf
        x[7, 16:] = -math.inf
        bias = torch.randn(32, generator=torch.Generator().manual_seed(1)) * 0.1
        off = bias.clone()
        off[4], off[20], off[6] = -math.inf, math.nan, -math.inf
        for b in (None, bias, off):
            for renorm in (True, False):
                _check(x, 6, scoring, b, groups, kept, top, renorm)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_scores_too_small_for_float32_keep_their_shares(scoring):
    x = torch.full((2, 16), -200.0)
    x[:, 3], x[:, 5] = -199.0, -201.0
    if scoring == "softmax":  # the largest logit is out of the kept groups by its bias
        x[:, 15] = 0.0
    bias = torch.zeros(16)
    bias[15] = -100.0
    _check(x, 4, scoring, bias, 1, 1, 1)


def test_rows_that_do_not_begin_on_16_bytes_and_other_device_state():
    """An odd number of experts, a view into a larger buffer, and a stream of its own."""
    from sglang_b200 import ops
    for dtype in ("bf16", "fp16", "fp32"):
        buf = _logits(1, 1 + 37 * 61, 9, dtype)[0]
        x = buf[1:].view(37, 61)
        side = torch.cuda.Stream()
        xd = buf.cuda()[1:].view(37, 61)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            w, ids = ops.route_topk(xd, 5)
        side.synchronize()
        want_w, want_i = O.route(x.double().numpy(), 5, "softmax")
        np.testing.assert_array_equal(ids.cpu().numpy(), want_i)


def test_no_rows():
    from sglang_b200 import ops
    w, ids = ops.route_topk(torch.zeros(0, 64, device="cuda"), 4)
    assert tuple(w.shape) == tuple(ids.shape) == (0, 4)


def test_offsets_beyond_32_bits():
    from sglang_b200 import ops
    T, E = (1 << 21) + 77, 1024
    x = torch.zeros(T, E, device="cuda", dtype=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(1)
    tail = torch.randn(100, E, generator=g, device="cuda").to(torch.bfloat16)
    x[-100:] = tail
    w, i = ops.route_topk(x, 3)
    want_w, want_i = ops.route_topk(tail, 3)
    assert torch.equal(i[-100:], want_i) and torch.equal(w[-100:], want_w)
    assert i[:-100].eq(torch.arange(3, device="cuda", dtype=torch.int32)).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,kept", [(32, 32, 5), (2, 2, 1), (31, 31, 31)])
def test_groups_of_one_expert(E, groups, kept, scoring):
    x = _logits(50, E, E)
    for b, top in ((None, 1), (None, 2), (torch.linspace(-0.3, 0.3, E), 2)):
        _check(x, min(kept, 4), scoring, b, groups, kept, top, True)
