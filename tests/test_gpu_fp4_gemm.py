"""The product of 4-bit operands against the definition in float64."""
import time

import numpy as np
import pytest
import torch

from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu

SCALE_T = {16: torch.float8_e4m3fn, 32: torch.float8_e8m0fnu}


def _operand(rows, k, group, seed, device="cuda"):
    """Random codes and scales: (codes, scales in blocked order with anything in the rows past the last, values in float64)."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 256, size=(rows, k // 2)).astype(np.uint8)
    lo, hi = (40, 70) if group == 16 else (122, 132)
    scode = rng.integers(lo, hi, size=(rows, k // group)).astype(np.uint8)
    b = F.blocked(scode, fill=0)
    gb = b.shape[1] // 4
    spare = np.setdiff1d(np.arange(-(-rows // 128) * 128), np.arange(rows))
    if len(spare):  # rows past the last: NaN scales
        r, c = np.meshgrid(spare, np.arange(gb * 4), indexing="ij")
        b.reshape(-1)[((r // 128) * gb + c // 4) * 512 + r % 32 * 16 + r // 32 % 4 * 4 + c % 4] = F.NAN_CODE[group]
    values = torch.from_numpy(F.dequantize(codes, scode, group))
    return torch.from_numpy(codes).to(device), torch.from_numpy(b).to(device).view(SCALE_T[group]), values


def _check(M, N, K, group, dtype, alpha=None, bias=False, seed=0):
    from sglang_b200 import ops
    a, sa, av = _operand(M, K, group, seed + 1)
    b, sb, bv = _operand(N, K, group, seed + 2)
    al = None if alpha is None else torch.tensor([alpha], device="cuda")
    bi = torch.randn(N, generator=torch.Generator().manual_seed(seed)).to(dtype) if bias else None
    got = ops.w4a4_group_fp4_matmul(a, b, sa, sb, al, dtype, None if bi is None else bi.cuda())
    assert got.dtype == dtype and tuple(got.shape) == (M, N)
    av, bv = av.cuda(), bv.cuda()
    f = 1.0 if alpha is None else float(np.float32(alpha))
    want, mass = (av @ bv.t()) * f, (av.abs() @ bv.abs().t()) * abs(f)
    if bi is not None:
        want = want + bi.cuda().double()
    # products are exact; an instruction adds 64 of them to the sum and errs by at most 2^-22 of what it adds up; partial sums of
    # up to 16 parts of K, the factor and the bias: 19 roundings of 2^-24 more; then one rounding to the output's type
    tol = ((K + 63) // 64 * 2.0**-22 + 19 * 2.0**-24) * mass + torch.finfo(dtype).eps / 2 * 1.01 * (want.abs() + 2.0**-20 * mass)
    tol += torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), (err / tol).max()
    assert ops.gemm_status() == 0


@pytest.mark.parametrize("group", [16, 32])
@pytest.mark.parametrize("M,N,K", [(1, 8, 32), (1, 128, 64), (3, 136, 96), (16, 2112, 7168), (17, 264, 288), (32, 1000, 4096), (33, 512, 1056),
                                   (64, 384, 544), (65, 256, 512), (128, 768, 256), (129, 392, 2080), (300, 1000, 1056), (515, 2112, 1536), (9000, 104, 544)])
def test_matmul(M, N, K, group):
    _check(M, N, K, group, torch.bfloat16, alpha=2.0**-10)


@pytest.mark.parametrize("M,N,K,group", [(1, 2112, 7168, 16), (40, 1920, 736, 32), (257, 1024, 8192, 32), (1000, 520, 992, 16)])
def test_matmul_fp16_bias_alpha(M, N, K, group):
    _check(M, N, K, group, torch.float16, alpha=3.1e-4, bias=True, seed=7)


@pytest.mark.parametrize("M,N,K", [(1, 4096, 256), (1, 24, 18432), (64, 7168, 16384), (2048, 2304, 7168), (4096, 3200, 512), (8, 36864, 7168)])
def test_matmul_large(M, N, K):
    _check(M, N, K, 16, torch.bfloat16, alpha=2.0**-12, bias=True, seed=3)


# tiles of 256 rows by pairs of CTAs: 256, 192 and 128 columns, ragged ends of every kind, one tile and several a pair
@pytest.mark.parametrize("group", [16, 32])
@pytest.mark.parametrize("M,N,K,columns", [(257, 10240, 1056, 192), (129, 20000, 288, 256), (1024, 5000, 544, 256), (1100, 1928, 96, 128),
                                           (8200, 520, 32, 128), (3000, 9224, 2080, 256), (513, 9432, 1312, 192)])
def test_matmul_pairs(M, N, K, columns, group):
    _check(M, N, K, group, torch.bfloat16, alpha=2.0**-10, bias=group == 16, seed=columns)


@pytest.mark.parametrize("group", [16, 32])
@pytest.mark.parametrize("M,N,K", [(5, 136, 160), (64, 256, 1024), (200, 320, 608), (700, 1040, 1024), (2048, 4104, 1024), (300, 9432, 544)])
def test_matmul_exact(M, N, K, group):
    """Scales of one and values that are multiples of a half: every partial sum is a multiple of 1/4 below 2^22, so float32 sums
    are exact and the output is the exact sum, rounded once."""
    from sglang_b200 import ops
    rng = np.random.default_rng(5)
    out = []
    for rows in (M, N):
        codes = rng.integers(0, 256, size=(rows, K // 2)).astype(np.uint8)
        scode = np.full((rows, K // group), 0x38 if group == 16 else 127, dtype=np.uint8)
        s = ops.fp4_blocked_scales(torch.from_numpy(scode).cuda().view(SCALE_T[group]))
        out.append((torch.from_numpy(codes).cuda(), s, torch.from_numpy(F.dequantize(codes, scode, group)).cuda()))
    (a, sa, av), (b, sb, bv) = out
    got = ops.w4a4_group_fp4_matmul(a, b, sa, sb)
    assert torch.equal(got, (av @ bv.t()).bfloat16())


def test_one_hot_scales():
    """Each operand all ones, one group of one row scaled apart: lands in that row (column) of the output and nowhere else."""
    from sglang_b200 import ops
    M, N, K = 200, 264, 544
    for group, one, two in ((16, 0x38, 0x40), (32, 127, 128)):
        codes = torch.full((N, K // 2), 0x22, dtype=torch.uint8, device="cuda")  # 1.0
        plain = np.full((N, K // group), one, dtype=np.uint8)
        s = ops.fp4_blocked_scales(torch.from_numpy(plain).cuda().view(SCALE_T[group]))
        for r in (0, 31, 32, 95, 127, 128, 199):
            for c in (0, 3, 4, K // group - 1):
                t = plain[:M].copy()
                t[r, c] = two
                st = ops.fp4_blocked_scales(torch.from_numpy(t).cuda().view(SCALE_T[group]))
                want = torch.full((M, N), float(K), device="cuda", dtype=torch.float16)
                want[r] += group
                got = ops.w4a4_group_fp4_matmul(codes[:M].contiguous(), codes, st, s, None, torch.float16)
                assert torch.equal(got, want), (group, r, c)
                got = ops.w4a4_group_fp4_matmul(codes, codes[:M].contiguous(), s, st, None, torch.float16)
                assert torch.equal(got, want.t().contiguous()), (group, r, c)


def test_nan_scales_stay_in_their_row():
    from sglang_b200 import ops
    for M in (40, 300):
        x = torch.randn(M, 512, device="cuda").bfloat16()
        w = torch.randn(256, 512, device="cuda").bfloat16()
        bq, bs = ops.per_token_group_quant_fp4(w)
        good = ops.w4a4_group_fp4_matmul(*_swap(ops.per_token_group_quant_fp4(x), (bq, bs)))
        x[7, 100] = float("nan")
        got = ops.w4a4_group_fp4_matmul(*_swap(ops.per_token_group_quant_fp4(x), (bq, bs)))
        assert torch.isnan(got[7]).all()
        keep = torch.arange(M, device="cuda") != 7
        assert torch.equal(got[keep], good[keep])


def _swap(a, b):
    return a[0], b[0], a[1], b[1]


def test_quantise_multiply_activate_multiply():
    """A gated MLP as a user runs it, against the same chain with every 4-bit operand taken as the quantizers leave it."""
    from sglang_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(11)
    for T, H, I in ((1, 512, 352), (70, 512, 352), (260, 1024, 768)):
        x = torch.randn(T, H, device="cuda", generator=g).bfloat16()
        gx, gw, gh = (torch.tensor([v], device="cuda") for v in (448 * 6 / 6.0, 448 * 6 / 0.12, 448 * 6 / 40.0))
        w13 = (torch.randn(2 * I, H, device="cuda", generator=g) * 0.02).bfloat16()
        w2 = (torch.randn(H, I, device="cuda", generator=g) * 0.02).bfloat16()
        q13, s13 = ops.per_token_group_quant_fp4(w13, gw)
        q2, s2 = ops.per_token_group_quant_fp4(w2, gw)
        xq, xs = ops.per_token_group_quant_fp4(x, gx)
        h13 = ops.w4a4_group_fp4_matmul(xq, q13, xs, s13, 1 / (gx * gw))
        hq, hs = ops.silu_and_mul_quant_fp4(h13, gh)
        out = ops.w4a4_group_fp4_matmul(hq, q2, hs, s2, 1 / (gh * gw))
        deq = lambda q, s, f: ops.per_token_group_dequant_fp4(q, s, f, torch.float32).double()  # noqa: E731
        w13d, w2d = deq(q13, s13, gw), deq(q2, s2, gw)
        want13 = deq(xq, xs, gx) @ w13d.t()
        # one rounding to bf16 of each, and float32 sums
        assert (h13.double() - want13).abs().max() <= 2.0**-8 * want13.abs().max()
        hd = deq(hq, hs, gh)
        want = hd @ w2d.t()
        assert (out.double() - want).abs().max() <= 2.0**-8 * want.abs().max()
        exact = F.silu_and_mul(h13.double().cpu().numpy())
        # half an e2m1 step of a group's largest value is a sixth of it, its scale's rounding a sixteenth of that more
        amax = np.repeat(np.abs(exact).reshape(T, -1, 16).max(-1), 16, -1)
        assert (np.abs(hd.cpu().numpy() - exact) <= amax * (1 / 6 + 1 / 16)).all()


@pytest.mark.parametrize("M,N,K", [(16, 7168, 4096), (64, 1024, 8192), (300, 512, 1024), (2048, 4096, 2048), (300, 10240, 4096)])
def test_wait_runs_out_and_recovers(M, N, K):
    from sglang_b200 import ops
    from sglang_b200._lib import check, lib
    a, sa, _ = _operand(M, K, 16, 1)
    b, sb, _ = _operand(N, K, 16, 2)
    good = ops.w4a4_group_fp4_matmul(a, b, sa, sb)
    torch.cuda.synchronize()
    assert ops.gemm_status() == 0
    lib.sglb200_gemm_set_wait_probes(0xFFFFFFFF)
    try:
        t0 = time.perf_counter()
        ops.w4a4_group_fp4_matmul(a, b, sa, sb)
        torch.cuda.synchronize()
        assert time.perf_counter() - t0 < 5.0
        assert ops.gemm_status() == 1
    finally:
        lib.sglb200_gemm_set_wait_probes(0)
        check(lib.sglb200_gemm_status_clear())
    again = ops.w4a4_group_fp4_matmul(a, b, sa, sb)
    torch.cuda.synchronize()
    assert ops.gemm_status() == 0 and torch.equal(again, good)


def test_captured_and_replayed_on_two_streams():
    """Two captured graphs and eager calls between them, each with inputs of its own."""
    from sglang_b200 import ops
    sets = []
    for seed, (M, N, K) in enumerate([(8, 2112, 7168), (520, 10240, 2048)]):
        a, sa, _ = _operand(M, K, 16, 2 * seed)
        b, sb, _ = _operand(N, K, 16, 2 * seed + 1)
        want = ops.w4a4_group_fp4_matmul(a, b, sa, sb)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.w4a4_group_fp4_matmul(a, b, sa, sb)
        sets.append((a, b, sa, sb, want, graph, out))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        sets[0][5].replay()
        with torch.cuda.stream(side):
            sets[1][5].replay()
            eager = ops.w4a4_group_fp4_matmul(*sets[0][:4])
        torch.cuda.synchronize()
        assert torch.equal(sets[0][6], sets[0][4]) and torch.equal(sets[1][6], sets[1][4]) and torch.equal(eager, sets[0][4])
        for s in sets:
            s[6].zero_()


def test_refusals():
    from sglang_b200 import ops
    a, sa, _ = _operand(4, 64, 16, 0)
    b, sb, _ = _operand(16, 64, 16, 1)
    a32, sa32, _ = _operand(4, 64, 32, 0)
    for bad, err in [(lambda: ops.w4a4_group_fp4_matmul(a, b, sa32, sb), "group sizes"),
                     (lambda: ops.w4a4_group_fp4_matmul(a, b, sa, sb, None, torch.float32), "output dtype"),
                     (lambda: ops.w4a4_group_fp4_matmul(a, b[:, :16].contiguous(), sa, sb), "shape|matching"),
                     (lambda: ops.w4a4_group_fp4_matmul(a, b, sa[:64], sb), "shape"),
                     (lambda: ops.w4a4_group_fp4_matmul(a, b, sa, sb, torch.ones(1)), "alpha"),
                     (lambda: ops.w4a4_group_fp4_matmul(a, b, sa, sb, None, torch.bfloat16, torch.ones(3, device="cuda")), "bias"),
                     (lambda: ops.w4a4_group_fp4_matmul(a.cpu(), b, sa, sb), "CUDA"),
                     (lambda: ops.w4a4_group_fp4_matmul(a, _operand(12, 64, 16, 1)[0], sa, _operand(12, 64, 16, 1)[1]), "divisible")]:
        with pytest.raises(RuntimeError, match=err):
            bad()
    a, sa, _ = _operand(4, 48, 16, 0)
    b, sb, _ = _operand(16, 48, 16, 1)
    with pytest.raises(RuntimeError, match="divisible"):
        ops.w4a4_group_fp4_matmul(a, b, sa, sb)
    a, sa, _ = _operand(4, 64, 16, 0)
    b, sb, _ = _operand(16, 64, 16, 1)
    assert ops.w4a4_group_fp4_matmul(a[:0], b, sa[:0], sb).shape == (0, 16)
