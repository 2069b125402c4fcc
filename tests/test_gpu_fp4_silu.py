"""silu(gate) * up inside the 4-bit operators, where float32 by itself is not enough."""
import numpy as np
import pytest
import torch

from oracle import fp4_oracle as F
from tests.test_gpu_fp4_moe import _run

pytestmark = pytest.mark.gpu


def _held(x, g, group):
    """(codes, scale codes) of the operator as numpy."""
    from sglang_b200 import ops
    q, s = ops.silu_and_mul_quant_fp4(x.cuda(), None if g is None else torch.tensor([g], device="cuda"), group)
    rows, d = x.shape[0], x.shape[1] // 2
    return q.cpu().numpy(), F.unblocked(s.view(torch.uint8).cpu().numpy(), rows, d // group)


@pytest.mark.parametrize("group,g", [(16, None), (16, 2.0**20), (32, None)])
def test_gates_below_minus_87(group, g):
    """e^-gate leaves float32 from 88.7 on, its reciprocal from 87.3; times a large `up` the product is an ordinary number."""
    gates = np.array([-86.5, -87.0, -87.5, -88.0, -88.5, -89.0, -90.0, -92.0, -95.0, -100.0, -101.0, -103.0, -104.0, -110.0, -120.0, -150.0])
    rows = []
    for top in (1e38, 3e36, 1e30):
        for first in (0, 3, 8):
            gate = np.resize(gates[first:], 64)
            up = np.where(np.arange(64) % 3 == 1, -1.0, 1.0) * top * (1 + np.arange(64) % 7 / 8)
            rows.append(np.concatenate([gate, up]))
    rows.append(np.concatenate([np.full(64, -88.0), np.full(64, 1e38)]))
    x = torch.from_numpy(np.stack(rows)).to(torch.bfloat16)
    codes, scales = _held(x, g, group)
    want = F.silu_and_mul(x.double().numpy())
    assert np.abs(want[-1]).min() > 40  # (an ordinary number)
    # float32: an activation and a product good to 2^-21, which can move a value over a border that it is next to
    gg, eps = 1.0 if g is None else np.float32(g), 2.0**-21
    lo, hi = F.group_scales(want * (1 - eps), gg, group)[0], F.group_scales(want * (1 + eps), gg, group)[0]
    assert ((lo <= scales) & (scales <= hi)).all()
    sv = F.scale_values(scales, group)
    got = F.unpack(codes)
    lo, hi = (F.value_codes(want * f, sv, gg, group) % 8 for f in (1 - eps, 1 + eps))
    assert ((lo <= got % 8) & (got % 8 <= hi)).all()
    assert (got[-1] % 8 > 0).all()


@pytest.mark.parametrize("gate", [-86, -88, -96, -100])
def test_experts_gates_below_minus_87(gate):
    """The same between the experts' products: 2688 * 2^17 = 3.5e8 times silu."""
    H, I = 64, 96
    c13, s13 = np.zeros((1, 2 * I, H), dtype=np.int64), np.full((1, 2 * I, H // 16), 0x38, dtype=np.uint8)
    c13[:, :I, 18], s13[:, :I, 1] = 15, 0x48   # gate: -6 * 4 * x[18]
    c13[:, I:, 0], s13[:, I:, 0] = 7, 0x7E     # up: 6 * 448 * x[0]
    c2, s2 = np.zeros((1, H, I), dtype=np.int64), np.full((1, H, I // 16), 0x38, dtype=np.uint8)
    c2[0, :, :H] = 2 * np.eye(H, dtype=np.int64)
    x = torch.zeros(3, H)
    x[:, 0], x[:, 18] = 2.0**17, -gate / 24
    x = x.bfloat16()
    w13, w2 = (F.pack(c13), s13, None), (F.pack(c2), s2, None)
    got = _run(x, w13, w2, torch.ones(3, 1), torch.zeros(3, 1, dtype=torch.int32)).double().cpu().numpy()
    a = -24 * x[0, 18].double().item()
    want = a * np.exp(a) / (1 + np.exp(a)) * 2688 * 2.0**17
    assert 1e-36 < abs(want)
    # x[18] has 8 bits and is 2^-15 of its row's largest, so it and the gate are exact; the activation is good to 2^-20
    assert (np.abs(got - want) <= (2.0**-8 + 2.0**-19) * abs(want)).all(), (got[0, :3], want)


def _near(targets, dtype, within):
    """(gate, up) of `dtype` whose silu(gate) * up lies within that share of a target's magnitude, though never on it."""
    gate = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype).double()
    gate = gate[torch.isfinite(gate) & (gate.abs() < 80) & (gate.abs() > 2.0**-10)].numpy()
    s = gate / (1 + np.exp(-gate))
    found = []
    for t in targets:
        up = torch.from_numpy(t / s).to(dtype).double().numpy()
        off = np.abs(s * up / t - 1)
        for i in np.nonzero((off < within) & (off > 2.0**-44) & (np.abs(up) > 2.0**-10))[0]:
            found.append((gate[i], up[i]))
    return found


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,g", [(16, None), (16, 6.72), (32, None)])
def test_values_next_to_borders(dtype, group, g):
    """Codes and scales are those of the unrounded product, also where it lies nearer to a border than float32 resolves."""
    gg = 1.0 if g is None else float(np.float32(g))
    rows = []
    scales = [1.0, 1.125, 1.25, 1.375, 1.5, 1.625, 1.75, 1.875] if group == 16 else [1.0]
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    for s in scales:  # a group whose largest value has this scale, and one next to a border of codes
        for gate, up in _near(borders * s / gg, dtype, 2.0**-22):
            row = np.zeros(2 * group)
            row[0], row[group] = 24.0, 6 * s / gg / 24
            row[5], row[group + 5] = gate, up
            rows.append(row)
    if group == 16:  # the largest value next to a border of scales
        targets = 6 * (F.E4M3[40:90] + F.E4M3[41:91]) / 2 / gg
    else:
        targets = 2.0 ** np.arange(-20, 12)
    for gate, up in _near(targets, dtype, 2.0**-22):
        row = np.zeros(2 * group)
        row[9], row[group + 9] = gate, up
        row[2::3], row[group + 2 :: 3] = 1.0, row[group + 2 :: 3] + 2.0**-6
        rows.append(row)
    x = torch.from_numpy(np.stack(rows)).to(dtype)
    codes, scode = _held(x, g, group)
    want_codes, want_scode = F.quantize(F.silu_and_mul(x.double().numpy()), gg, group)
    wrong = (codes != want_codes).any(1) | (scode != want_scode).any(1)
    print(f"{len(rows)} rows, {wrong.sum()} wrong")
    assert not wrong.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,g", [(16, None), (16, 6.72), (32, None)])
@pytest.mark.parametrize("rows,d", [(1, 64), (130, 352), (2600, 2112)])
def test_bit_for_bit(dtype, group, g, rows, d):
    """Ordinary rows, among them gates whose silu is the gate itself, so that products are short numbers and lie on borders."""
    gen = torch.Generator().manual_seed(rows + d)
    x = torch.randn(rows, 2 * d, generator=gen)
    x = torch.where(torch.rand(x.shape, generator=gen) < 0.02, x * 40, x)
    x[0] = torch.randint(-60, 60, (2 * d,), generator=gen).float() / 2
    x = x.to(dtype)
    codes, scode = _held(x, g, group)
    h = F.silu_and_mul(x.double().numpy())
    want_codes, want_scode = F.quantize(h, 1.0 if g is None else float(np.float32(g)), group)
    assert np.array_equal(scode, want_scode) and np.array_equal(codes, want_codes)


@pytest.mark.parametrize("group,g", [(16, 6.72), (32, None)])
def test_rows_that_begin_on_16_bytes(group, g):
    """A view that is 16-byte but not 32-byte aligned, with gates that float32 does not do for in some groups of many warps."""
    gen = torch.Generator().manual_seed(31)
    x = torch.randn(200, 2 * 288, generator=gen)
    x[::3, 5:288:40] = -90.0
    x[::3, 288 + 5 :: 40] = 1e36
    x = x.bfloat16()
    flat = torch.empty(x.numel() + 8, dtype=torch.bfloat16, device="cuda")
    flat[8:] = x.flatten().cuda()
    view = flat[8:].view(x.shape)
    assert view.data_ptr() % 32 == 16
    from sglang_b200 import ops
    scale = None if g is None else torch.tensor([g], device="cuda")
    q, s = ops.silu_and_mul_quant_fp4(view, scale, group)
    want_q, want_s = F.quantize(F.silu_and_mul(x.double().numpy()), 1.0 if g is None else float(np.float32(g)), group)
    assert np.array_equal(F.unblocked(s.view(torch.uint8).cpu().numpy(), 200, 288 // group), want_s)
    assert np.array_equal(q.cpu().numpy(), want_q)
    again, _ = ops.silu_and_mul_quant_fp4(x.cuda(), scale, group)
    assert torch.equal(again, q)
