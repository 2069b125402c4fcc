"""The 4-bit quantizers and the way back, against the definition in float64: codes and scales bit for bit."""
import numpy as np
import pytest
import torch

from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rows(rows, hidden, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, hidden, generator=g)
    x = torch.where(torch.rand(rows, hidden, generator=g) < 0.01, x * 30, x)
    x = torch.where(torch.rand(rows, 1, generator=g) < 0.1, torch.zeros(()), x)  # rows of zeros
    return x.to(dtype)


def _scale(g):
    return None if g is None else torch.tensor([g], device="cuda", dtype=torch.float32)


def _check(x, g, group, q, s):
    rows, hidden = x.shape
    want_q, want_s = F.quantize(x.double().numpy(), 1.0 if g is None else np.float32(g), group)
    s = s.view(torch.uint8).cpu().numpy()
    assert np.array_equal(F.unblocked(s, rows, hidden // group), want_s)
    assert np.array_equal(q.cpu().numpy(), want_q)
    pad = -(-(hidden // group) // 4) * 4
    assert not F.unblocked(s, rows, pad)[:, hidden // group :].any()  # groups past the last


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,hidden", [(1, 16), (1, 7168), (3, 48), (127, 272), (129, 2112), (300, 64), (33, 18432), (2100, 4112)])
@pytest.mark.parametrize("g", [None, 44.8, 32.0, 0.37])
def test_quant_16(dtype, rows, hidden, g):
    from sglang_b200 import ops
    x = _rows(rows, hidden, dtype, rows + hidden)
    q, s = ops.per_token_group_quant_fp4(x.cuda(), _scale(g))
    assert q.dtype == torch.uint8 and s.dtype == torch.float8_e4m3fn
    _check(x, g, 16, q, s)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,hidden", [(1, 32), (1, 7168), (5, 96), (129, 2112), (300, 64), (2100, 4128)])
def test_quant_32(dtype, rows, hidden):
    from sglang_b200 import ops
    x = _rows(rows, hidden, dtype, rows + hidden)
    q, s = ops.per_token_group_quant_fp4(x.cuda(), None, 32)
    assert s.dtype == torch.float8_e8m0fnu
    _check(x, None, 32, q, s)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [16, 32])
def test_borders_and_special_values(dtype, group):
    """Values on and next to every border, under scales on and next to theirs; subnormals, the largest finite values; groups with
    a NaN or an infinity."""
    from sglang_b200 import ops
    rng = np.random.default_rng(3)
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    rows = []
    for scale in [1.0, 1.125, 0.875, 13.0, 2.0**-6, 2.0**-9, 448.0]:
        for jitter in [0.0, 2.0**-8, -(2.0**-8), 2.0**-10, 2.0**-20, -(2.0**-22)]:
            v = rng.choice(borders, size=64) * rng.choice([-1.0, 1.0], size=64) * scale * (1 + jitter)
            v[::group] = 6 * scale
            rows.append(v)
    tiny, huge = float(torch.finfo(dtype).tiny), float(torch.finfo(dtype).max)
    rows += [np.full(64, tiny), np.full(64, tiny / 2), np.linspace(-tiny, tiny, 64), np.linspace(0, huge, 64), np.full(64, -0.0)]
    for bad in (np.nan, np.inf, -np.inf):
        v = rng.standard_normal(64)
        v[5] = bad
        rows.append(v)
    x = torch.from_numpy(np.stack(rows)).to(dtype)
    for g in [None] if group == 32 else [None, 1.0, 44.8, 1.0 / 3.0, 7.4666667, 2.0**30]:
        q, s = ops.per_token_group_quant_fp4(x.cuda(), _scale(g), group)
        _check(x, g, group, q, s)
        v = ops.per_token_group_dequant_fp4(q, s, _scale(g), torch.float32).cpu()
        held = torch.isfinite(x).view(len(x), -1, group).all(-1, keepdim=True).expand(-1, -1, group).reshape(x.shape)
        assert torch.isnan(v[~held]).all() and not torch.isnan(v[held]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,g", [(16, None), (16, 44.8), (32, None)])
@pytest.mark.parametrize("rows,hidden", [(1, 32), (131, 2112), (257, 160), (2100, 4128)])
def test_dequant(dtype, group, g, rows, hidden):
    from sglang_b200 import ops
    rng = np.random.default_rng(hidden)
    codes = rng.integers(0, 256, size=(rows, hidden // 2)).astype(np.uint8)
    scode = rng.integers(0 if group == 16 else 110, 127 if group == 16 else 135, size=(rows, hidden // group)).astype(np.uint8)
    t = torch.float8_e4m3fn if group == 16 else torch.float8_e8m0fnu
    s = ops.fp4_blocked_scales(torch.from_numpy(scode).cuda().view(t))
    got = ops.per_token_group_dequant_fp4(torch.from_numpy(codes).cuda(), s, _scale(g), dtype).double().cpu().numpy()
    want = F.dequantize(codes, scode, group) / np.float64(np.float32(1.0 if g is None else g))
    # s / g and code * (s / g) in float32: each off by at most 2^-24 of the value; then one rounding to the output's type
    tol = (2 * 2.0**-24 + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0)) * np.abs(want)
    # below the type's normal range a rounding is half a subnormal step
    tol += torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("group,g", [(16, None), (16, 6.72), (32, None)])
@pytest.mark.parametrize("rows,d", [(1, 32), (64, 2048), (129, 352), (7, 18432)])
def test_silu_and_mul_quant(dtype, group, g, rows, d):
    from sglang_b200 import ops
    x = _rows(rows, 2 * d, dtype, rows + d)
    x[0, :16] = torch.tensor([0.0, -0.0, 100.0, -100.0, 20.0, -20.0, 88.0, -88.0] * 2)
    q, s = ops.silu_and_mul_quant_fp4(x.cuda(), _scale(g), group)
    h = F.silu_and_mul(x.double().numpy())
    gg = 1.0 if g is None else np.float32(g)
    scode = F.unblocked(s.view(torch.uint8).cpu().numpy(), rows, d // group)
    # h in float32: the exponential is off by at most 2 units of 2^-23, the sum, the quotient and the product by half a unit
    # each; e^-x / (1 + e^-x) <= 1 carries the first over: 3.5 units, here 4 = 2^-21 of the value
    eps = 2.0**-21
    lo_s, hi_s = F.group_scales(h * (1 - eps), gg, group)[0], F.group_scales(h * (1 + eps), gg, group)[0]
    assert ((lo_s <= scode) & (scode <= hi_s)).all()
    got = F.unpack(q.cpu().numpy())
    sv = F.scale_values(scode, group)
    lo, hi = (F.value_codes(h * f, sv, gg, group) % 8 for f in (1 - eps, 1 + eps))
    assert ((lo <= got % 8) & (got % 8 <= hi)).all()
    nonzero = (got % 8 > 0)
    assert np.array_equal(got[nonzero] >= 8, h[nonzero] < 0)


def test_batched_shapes_empty_and_streams():
    from sglang_b200 import ops
    x = _rows(30, 64, torch.bfloat16, 1)
    q, s = ops.per_token_group_quant_fp4(x.view(2, 15, 64).cuda())
    assert tuple(q.shape) == (2, 15, 32)
    _check(x, None, 16, q.view(30, 32), s)
    assert tuple(ops.per_token_group_dequant_fp4(q, s).shape) == (2, 15, 64)
    q, s = ops.per_token_group_quant_fp4(torch.empty(0, 64, device="cuda", dtype=torch.bfloat16))
    assert q.shape == (0, 32) and s.shape == (0, 4)
    assert ops.per_token_group_dequant_fp4(q, s).shape == (0, 64)
    side = torch.cuda.Stream()
    big = torch.randn(4096, 8192, device="cuda").bfloat16()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y = big * 2
        q, s = ops.per_token_group_quant_fp4(y)
        back = ops.per_token_group_dequant_fp4(q, s)
    side.synchronize()
    again = ops.per_token_group_quant_fp4(big * 2)
    assert torch.equal(again[0], q) and torch.equal(ops.per_token_group_dequant_fp4(*again), back)


def test_values_that_begin_on_16_bytes():
    """A view that is 16-byte but not 32-byte aligned takes narrower loads and stores."""
    from sglang_b200 import ops
    for dtype, off in ((torch.bfloat16, 8), (torch.float32, 4)):
        x = _rows(70, 96, dtype, 4)
        flat = torch.empty(70 * 96 + off, dtype=dtype, device="cuda")
        flat[off:] = x.flatten().cuda()
        view = flat[off:].view(70, 96)
        assert view.data_ptr() % 32 == 16
        q, s = ops.per_token_group_quant_fp4(view)
        _check(x, None, 16, q, s)
        q, s = ops.per_token_group_quant_fp4(view, None, 32)
        _check(x, None, 32, q, s)
    y = torch.empty(70 * 96 + 8, dtype=torch.bfloat16, device="cuda")[8:].view(70, 96)
    from sglang_b200._lib import check, lib
    check(lib.sglb200_per_token_group_dequant_fp4(q.data_ptr(), s.data_ptr(), None, y.data_ptr(), 0, 70, 96, 32,
                                                  torch.cuda.current_stream().cuda_stream))
    assert torch.equal(y, ops.per_token_group_dequant_fp4(q, s))


def test_rows_past_the_last_are_left_as_they_were():
    from sglang_b200._lib import check, lib
    x = torch.randn(5, 64, device="cuda").bfloat16()
    q = torch.full((6, 32), 0xAB, dtype=torch.uint8, device="cuda")
    s = torch.full((128, 4), 0xCD, dtype=torch.uint8, device="cuda")
    check(lib.sglb200_per_token_group_quant_fp4(x.data_ptr(), 0, q.data_ptr(), s.data_ptr(), None, 5, 64, 16,
                                                torch.cuda.current_stream().cuda_stream))
    assert (q[5] == 0xAB).all()
    assert (F.unblocked(s.cpu().numpy(), 128, 4)[5:] == 0xCD).all()


def test_gpu_refusals():
    from sglang_b200 import ops
    x = torch.randn(4, 64, device="cuda").bfloat16()
    for bad, err in [(lambda: ops.per_token_group_quant_fp4(x.t()), "contiguous"),
                     (lambda: ops.per_token_group_quant_fp4(x[:, :40].contiguous()), "divisible"),
                     (lambda: ops.per_token_group_quant_fp4(x, torch.ones(2, device="cuda")), "global_scale"),
                     (lambda: ops.per_token_group_quant_fp4(x, torch.ones(1)), "global_scale"),
                     (lambda: ops.per_token_group_quant_fp4(x, torch.ones(1, device="cuda"), 32), "global scale"),
                     (lambda: ops.per_token_group_quant_fp4(x.double()), "dtype"),
                     (lambda: ops.silu_and_mul_quant_fp4(x.float()), "dtype"),
                     (lambda: ops.silu_and_mul_quant_fp4(x[:, :63].contiguous()), "odd"),
                     (lambda: ops.per_token_group_quant_fp4(torch.randn(65 * 64, device="cuda").bfloat16()[1:65]), "16-byte")]:
        with pytest.raises(RuntimeError, match=err):
            bad()
    q, s = ops.per_token_group_quant_fp4(x)
    with pytest.raises(RuntimeError, match="shape"):
        ops.per_token_group_dequant_fp4(q[:, :16].contiguous(), torch.cat([s, s]))
    with pytest.raises(RuntimeError, match="uint8"):
        ops.per_token_group_dequant_fp4(q.to(torch.int32), s)
    with pytest.raises(RuntimeError, match="dtype"):
        ops.per_token_group_dequant_fp4(q, s, None, torch.float64)
