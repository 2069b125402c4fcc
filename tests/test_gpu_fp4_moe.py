"""The routed experts of a few tokens on 4-bit weights, against the definition in float64."""
import numpy as np
import pytest
import torch

from oracle import fp4_oracle as F

pytestmark = pytest.mark.gpu


def _weights(E, n, k, seed):
    """Random codes, plausible scales, a factor per expert; and the values in float64 (without the factor)."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 256, size=(E, n, k // 2)).astype(np.uint8)
    scode = rng.integers(30, 90, size=(E, n, k // 16)).astype(np.uint8)
    alpha = (rng.random(E) * 0.5 + 0.5).astype(np.float32) * np.float32(1e-3)
    return codes, scode, alpha, F.dequantize(codes, scode, 16)


def _cuda(codes, scode, alpha):
    return (torch.from_numpy(codes).cuda(), torch.from_numpy(scode).cuda().view(torch.float8_e4m3fn),
            None if alpha is None else torch.from_numpy(alpha).cuda())


def _layer(T, E, topk, H, I, dtype, seed, alpha=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g)
    x = torch.where(torch.rand(T, H, generator=g) < 0.01, x * 20, x).to(dtype)
    w13, w2 = _weights(E, 2 * I, H, seed + 1), _weights(E, H, I, seed + 2)
    if not alpha:
        w13, w2 = (w[:2] + (None,) + w[3:] for w in (w13, w2))
    ids = torch.stack([torch.randperm(E, generator=g)[:topk] for _ in range(T)]).to(torch.int32)
    weights = torch.rand(T, topk, generator=g)
    return x, w13, w2, weights, ids


def _run(x, w13, w2, weights, ids, factor=1.0):
    from sglang_b200 import ops
    c13, s13, a13 = _cuda(*w13[:3])
    c2, s2, a2 = _cuda(*w2[:3])
    return ops.fused_experts_fp4(x.cuda(), c13, c2, s13, s2, weights.cuda(), ids.cuda(), a13, a2, factor)


def _want(x, w13, w2, weights, ids, factor=1.0):
    """(output, sum of magnitudes that rounding errors scale with), float64."""
    x = x.double().numpy()
    T, H = x.shape
    E, I = len(w2[3]), w2[3].shape[2]
    a13, a2 = (np.ones(E) if w[2] is None else w[2].astype(np.float64) for w in (w13, w2))
    out, first, second = np.zeros((T, H)), np.zeros((T, H)), np.zeros((T, H))
    for t in range(T):
        for j, e in enumerate(ids[t].tolist()):
            if not 0 <= e < E:
                continue
            f = float(weights[t, j]) * a2[e] * factor
            gu = a13[e] * (w13[3][e] @ x[t])
            gate, up = gu[:I], gu[I:]
            mass = a13[e] * (np.abs(w13[3][e]) @ np.abs(x[t]))
            sig = 1 / (1 + np.exp(-gate))
            h = gate * sig * up
            # |d silu| <= 1.1: what an error of the first sums does to h
            dh = 1.1 * mass[:I] * np.abs(up) + np.abs(gate * sig) * mass[I:]
            out[t] += f * (w2[3][e] @ h)
            w = np.abs(w2[3][e]) * abs(f)
            first[t] += w @ dh
            second[t] += w @ np.abs(h) + 2.0**-13 * (w @ np.full(I, np.abs(h).max()))
    return out, first, second


def _check(got, want, H, I, dtype):
    out, first, second = want
    # first sums: H products that are exact, float32 additions (at most one unit of 2^-23 of the running magnitude for every 16
    # columns, and eight more between warps), the factor; bf16 activations below 2^-18 of their row's largest are off by 2^-26 of it
    e1 = (H / 16 + 12) * 2.0**-23 + 2.0**-20
    # h: rounded to fp16 (2^-12) after an activation good to 2^-21; second sums likewise; the sum over a token's slots and two factors
    e2 = 2.0**-12 + 2.0**-20 + (I / 16 + 20) * 2.0**-23
    tol = e1 * first + e2 * second + torch.finfo(dtype).eps / 2 * np.abs(out) * 1.001 + torch.finfo(dtype).tiny
    err = np.abs(got.double().cpu().numpy() - out)
    assert (err <= tol).all(), (err / tol).max()
    # the bound above is a sum of worst cases; the typical error is that of one rounding to the output's type
    rms = np.sqrt((err**2).mean() / (out**2).mean())
    assert rms <= torch.finfo(dtype).eps / 2, rms


CASES = [(1, 8, 2, 256, 128), (1, 256, 8, 512, 96), (3, 4, 4, 288, 352), (16, 16, 4, 1024, 512), (33, 8, 2, 512, 160), (64, 4, 1, 416, 1056),
         (5, 3, 1, 7168, 64), (7, 6, 2, 64, 2048), (128, 8, 8, 128, 64), (2, 1, 1, 32, 32),
         # rows' scales on two bytes, on four, on eight; several turns of the ring, ragged sets of tiles
         (6, 4, 2, 4128, 288), (6, 4, 2, 4160, 320), (6, 4, 2, 4224, 416), (1, 64, 8, 3104, 1056), (50, 6, 3, 2080, 800),
         # experts of many rows, whose slots are split among CTAs: few slots, one expert, the same experts for all, the most slots
         (31, 1, 1, 2080, 256), (64, 1, 1, 4096, 256), (64, 2, 2, 2080, 800), (128, 3, 3, 1056, 96), (1024, 5, 1, 544, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,topk,H,I", CASES)
def test_experts(T, E, topk, H, I, dtype):
    args = _layer(T, E, topk, H, I, dtype, T + E)
    _check(_run(*args), _want(*args), H, I, dtype)


def test_without_factors_and_with_a_scaling_factor():
    args = _layer(4, 8, 2, 256, 128, torch.bfloat16, 5, alpha=False)
    _check(_run(*args, 2.5), _want(*args, 2.5), 256, 128, torch.bfloat16)


def test_filtered_ids_and_repeated_ids():
    x, w13, w2, weights, ids = _layer(9, 8, 4, 256, 128, torch.bfloat16, 6)
    ids[0] = -1            # nothing of this rank
    ids[1, 2] = -1
    ids[2] = torch.tensor([3, 3, 3, 5])  # an expert three times
    ids[3, 0] = 8          # past the last
    ids[4, 1] = 2**31 - 1
    ids[5, 1] = -(2**31)
    got = _run(x, w13, w2, weights, ids)
    _check(got, _want(x, w13, w2, weights, ids), 256, 128, torch.bfloat16)
    assert not got[0].any()
    assert not _run(x, w13, w2, weights, torch.full_like(ids, -1)).any()
    wide = ids.to(torch.int64)
    wide[4, 1], wide[5, 1], wide[1, 2] = 2**40 + 1, -(2**40) + 1, 2**32
    assert torch.equal(_run(x, w13, w2, weights, wide), got)


def test_all_tokens_to_one_expert():
    for T in (7, 8, 9, 40, 1024):
        x, w13, w2, weights, ids = _layer(T, 2, 1, 160, 96, torch.bfloat16, 8)
        ids[:] = 1
        _check(_run(x, w13, w2, weights, ids), _want(x, w13, w2, weights, ids), 160, 96, torch.bfloat16)


def test_one_token_to_many_experts():
    x, w13, w2, weights, ids = _layer(1, 1024, 1024, 64, 32, torch.bfloat16, 9)
    _check(_run(x, w13, w2, weights, ids), _want(x, w13, w2, weights, ids), 64, 32, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_wide_range_of_activations(dtype):
    """Rows of very small and very large magnitudes, and both in one row."""
    x, w13, w2, weights, ids = _layer(8, 4, 2, 512, 128, dtype, 10)
    top = 1e4 if dtype == torch.float16 else 1e30
    x = x.float()
    x[0] *= 1e-6 if dtype == torch.float16 else 1e-30
    x[1, 3] = top
    x[2] = 0
    x[3, ::2] *= 1e-4
    x = x.to(dtype)
    w13 = w13[:2] + ((w13[2] * 1e-3).astype(np.float32) if dtype == torch.float16 else w13[2],) + w13[3:]
    keep = torch.tensor([0, 2, 3, 4, 5, 6, 7] + ([1] if dtype == torch.float16 else []))
    got = _run(x, w13, w2, weights, ids)
    with np.errstate(over="ignore", invalid="ignore"):
        want = _want(x, w13, w2, weights, ids)
    _check(got[keep.cuda()], tuple(w[keep.numpy()] for w in want), 512, 128, dtype)
    assert not got[2].any()


def test_not_finite_activations_stay_in_their_row():
    x, w13, w2, weights, ids = _layer(10, 2, 2, 256, 128, torch.bfloat16, 12)
    good = _run(x, w13, w2, weights, ids)
    x[3, 7], x[6, 9] = float("nan"), float("inf")
    got = _run(x, w13, w2, weights, ids)
    assert torch.isnan(got[3]).all() and not torch.isfinite(got[6]).any()
    keep = torch.tensor([0, 1, 2, 4, 5, 7, 8, 9]).cuda()
    assert torch.equal(got[keep], good[keep])


def test_results_do_not_depend_on_the_batch_and_repeat():
    """From run to run; and alone as among others, where K is split alike."""
    x, w13, w2, weights, ids = _layer(32, 16, 4, 512, 256, torch.bfloat16, 13)
    many = _run(x, w13, w2, weights, ids)
    for _ in range(3):
        assert torch.equal(_run(x, w13, w2, weights, ids), many)
    for t in (0, 17, 31):
        assert torch.equal(_run(x[t : t + 1], w13, w2, weights[t : t + 1], ids[t : t + 1])[0], many[t])


def test_captured_graphs_streams_and_the_router_in_front():
    """Routing, then the experts, captured twice in one pool and replayed on two streams between eager calls."""
    from sglang_b200 import ops
    _, w13, w2, _, _ = _layer(1, 16, 4, 512, 256, torch.bfloat16, 14)
    c13, s13, a13 = _cuda(*w13[:3])
    c2, s2, a2 = _cuda(*w2[:3])

    def layer(x, logits):
        w = torch.empty(x.shape[0], 4, device="cuda")
        ids = torch.empty(x.shape[0], 4, device="cuda", dtype=torch.int32)
        ops.topk_softmax_out(w, ids, logits, True)
        return ops.fused_experts_fp4(x, c13, c2, s13, s2, w, ids, a13, a2), w, ids

    sets = []
    for T in (3, 24):
        x, logits = torch.randn(T, 512, device="cuda").bfloat16(), torch.randn(T, 16, device="cuda")
        want, w, ids = layer(x, logits)
        full = _want(x.cpu(), w13, w2, w.cpu(), ids.cpu())
        _check(want, full, 512, 256, torch.bfloat16)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=sets[0][3].pool() if sets else None):
            out = layer(x, logits)[0]
        sets.append((x, logits, want, graph, out))
    for _ in range(3):  # (graphs of one pool run one after the other)
        for x, logits, want, graph, out in sets:
            graph.replay()
            assert torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            a = layer(*sets[0][:2])[0]
        b = layer(*sets[1][:2])[0]
        torch.cuda.synchronize()
        assert torch.equal(a, sets[0][2]) and torch.equal(b, sets[1][2])


def test_quantised_weights_of_a_checkpoint():
    """Weights as a quantizer leaves them, scales in rows' order: the layer against the dequantised one."""
    g = torch.Generator().manual_seed(15)
    E, H, I, T = 4, 512, 256, 6
    x = torch.randn(T, H, generator=g).bfloat16()
    ws = []
    for n, k in ((2 * I, H), (H, I)):
        w = torch.randn(E, n, k, generator=g).numpy() * 0.02
        gs = [np.float32(448 * 6 / np.abs(v).max()) for v in w]
        q = [F.quantize(v, s, 16) for v, s in zip(w, gs)]
        codes, scode = np.stack([a for a, _ in q]), np.stack([b for _, b in q])
        ws.append((codes, scode, np.array([1 / s for s in gs], dtype=np.float32), F.dequantize(codes, scode, 16)))
    ids = torch.stack([torch.randperm(E, generator=g)[:2] for _ in range(T)]).to(torch.int32)
    weights = torch.rand(T, 2, generator=g)
    _check(_run(x, *ws, weights, ids), _want(x, *ws, weights, ids), H, I, torch.bfloat16)


@pytest.mark.parametrize("T,E,topk,H,I", [(1, 64, 8, 7168, 512), (40, 4, 2, 2048, 1024)])
def test_wait_runs_out_and_recovers(T, E, topk, H, I):
    import time

    from sglang_b200 import ops
    from sglang_b200._lib import check, lib
    args = _layer(T, E, topk, H, I, torch.bfloat16, 16)
    good = _run(*args)
    torch.cuda.synchronize()
    assert ops.gemm_status() == 0
    lib.sglb200_gemm_set_wait_probes(0xFFFFFFFF)
    try:
        t0 = time.perf_counter()
        _run(*args)
        torch.cuda.synchronize()
        assert time.perf_counter() - t0 < 10.0
        assert ops.gemm_status() == 1
    finally:
        lib.sglb200_gemm_set_wait_probes(0)
        check(lib.sglb200_gemm_status_clear())
    assert torch.equal(_run(*args), good) and ops.gemm_status() == 0


def test_refusals():
    from sglang_b200 import ops
    x, w13, w2, weights, ids = _layer(4, 8, 2, 256, 128, torch.bfloat16, 5)
    c13, s13, a13 = _cuda(*w13[:3])
    c2, s2, a2 = _cuda(*w2[:3])
    x, weights, ids = x.cuda(), weights.cuda(), ids.cuda()

    def call(x=x, c13=c13, c2=c2, s13=s13, s2=s2, weights=weights, ids=ids, a13=a13, a2=a2):
        return ops.fused_experts_fp4(x, c13, c2, s13, s2, weights, ids, a13, a2)

    for bad, err in [(dict(x=x.float()), "dtype"), (dict(x=x.cpu()), "CUDA"), (dict(x=x.t()), "contiguous"),
                     (dict(x=x[:, :128].contiguous()), "do not fit"), (dict(s13=s13[:, :1].contiguous()), "w13_scale"),
                     (dict(c2=c2[:, :, :32].contiguous()), "do not fit"), (dict(a13=a13[:3]), "w13_alpha"), (dict(a2=a2.double()), "w2_alpha"),
                     (dict(ids=ids[:3]), "topk"), (dict(ids=ids.float()), "int32"), (dict(ids=ids.to(torch.int16)), "int32"), (dict(weights=weights[:, :1].contiguous()), "topk"),
                     (dict(x=x.repeat(200, 1), ids=ids.repeat(200, 1), weights=weights.repeat(200, 1)), "at most 1024")]:
        with pytest.raises(RuntimeError, match=err):
            call(**bad)
    assert call(x=x[:0], ids=ids[:0], weights=weights[:0]).shape == (0, 256)
    assert not call(ids=ids[:, :0].contiguous(), weights=weights[:, :0].contiguous()).any()
