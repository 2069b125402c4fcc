"""The 4-bit quantizers at sizes where a warp takes two tasks, and beyond one launch, against the definition in float64."""
import numpy as np
import pytest
import torch

from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _rows_for_two_tasks(columns, group):
    """Rows (68 past a block of 128) with which a warp takes two tasks: 64 warps of two for every SM; a task is a block of four groups in eight
    rows, or four where a group has 32 columns."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    blocks = -(-columns // group // 4)
    per_128_rows = (16 if group == 16 else 32) * blocks
    return -(-sms * 128 // per_128_rows) * 128 + 68


def _scale(g):
    return None if g is None else torch.tensor([g], device="cuda")


def _x(rows, columns, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, columns, generator=gen)
    return (x * 2.0 ** torch.randint(-3, 4, (rows, 1), generator=gen)).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,g,columns", [(16, 44.8, 4112), (16, None, 18480), (32, None, 4128)])
def test_quant(dtype, group, g, columns):
    from sglang_b200 import ops
    rows = _rows_for_two_tasks(columns, group)
    x = _x(rows, columns, dtype, 1)
    q, s = ops.per_token_group_quant_fp4(x.cuda(), _scale(g), group)
    want_q, want_s = F.quantize(x.double().numpy(), 1.0 if g is None else float(np.float32(g)), group)
    s = s.view(torch.uint8).cpu().numpy()
    assert np.array_equal(F.unblocked(s, rows, columns // group), want_s)
    assert np.array_equal(q.cpu().numpy(), want_q)
    assert not F.unblocked(s, rows, -(-columns // group // 4) * 4)[:, columns // group :].any()


@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("group,g,columns", [(16, 6.72, 4112), (32, None, 4128)])
def test_silu_and_mul_quant(dtype, group, g, columns):
    from sglang_b200 import ops
    rows = _rows_for_two_tasks(columns, group)
    x = _x(rows, 2 * columns, dtype, 2)
    q, s = ops.silu_and_mul_quant_fp4(x.cuda(), _scale(g), group)
    h = F.silu_and_mul(x.double().numpy())
    want_q, want_s = F.quantize(h, 1.0 if g is None else float(np.float32(g)), group)
    assert np.array_equal(F.unblocked(s.view(torch.uint8).cpu().numpy(), rows, columns // group), want_s)
    assert np.array_equal(q.cpu().numpy(), want_q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group,g,columns", [(16, 44.8, 4112), (32, None, 4128)])
def test_dequant(dtype, group, g, columns):
    from sglang_b200 import ops
    rows = _rows_for_two_tasks(columns, group)
    rng = np.random.default_rng(3)
    codes = rng.integers(0, 256, size=(rows, columns // 2)).astype(np.uint8)
    scode = rng.integers(40 if group == 16 else 115, 90 if group == 16 else 135, size=(rows, columns // group)).astype(np.uint8)
    t = torch.float8_e4m3fn if group == 16 else torch.float8_e8m0fnu
    s = ops.fp4_blocked_scales(torch.from_numpy(scode).cuda().view(t))
    got = ops.per_token_group_dequant_fp4(torch.from_numpy(codes).cuda(), s, _scale(g), dtype).double().cpu().numpy()
    want = F.dequantize(codes, scode, group) / np.float64(np.float32(1.0 if g is None else g))
    # s / g and code * (s / g) in float32: each off by at most 2^-24 of the value; then one rounding to the output's type
    tol = (2 * 2.0**-24 + (torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0)) * np.abs(want) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert (np.abs(got - want) <= tol).all()


def test_more_rows_than_a_launch_takes():
    """A launch takes 2^30 bytes of scales, 2^28 rows of one group: five more are a launch of their own.  Rows repeat, so that every part has
    to give what the first one gives."""
    from sglang_b200 import ops
    base, times, more = 1 << 20, 1 << 8, 5
    for silu in (False, True):
        x = _x(base, 32 if silu else 16, torch.bfloat16, 4).cuda()
        quantizer = ops.silu_and_mul_quant_fp4 if silu else ops.per_token_group_quant_fp4
        q, s = quantizer(x)
        want_q, want_s = q.clone(), s.view(torch.uint8).clone()
        big = torch.cat([x.repeat(times, 1), x[:more]])
        q, s = quantizer(big)
        del big
        s = s.view(torch.uint8)
        for part in range(times):
            assert torch.equal(q[part * base : (part + 1) * base], want_q)
            assert torch.equal(s[part * base : (part + 1) * base], want_s)
        assert torch.equal(q[times * base :], want_q[:more])
        assert np.array_equal(F.unblocked(s[times * base :].cpu().numpy(), more, 4), F.unblocked(want_s[:128].cpu().numpy(), more, 4))
        back = ops.per_token_group_dequant_fp4(q, s.view(torch.float8_e4m3fn))
        want = ops.per_token_group_dequant_fp4(want_q, want_s.view(torch.float8_e4m3fn))
        for part in range(times):
            assert torch.equal(back[part * base : (part + 1) * base], want)
        assert torch.equal(back[times * base :], want[:more])
        del q, s, back
        torch.cuda.empty_cache()
