"""silu(gate) * up inside the 4-bit operators, where float32 by itself is not enough."""
import numpy as np
import pytest
import torch

from oracle import fp4_oracle as F
from tests.test_gpu_fp4_moe import _run

pytestmark = pytest.mark.gpu


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
