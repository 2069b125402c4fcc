"""Low-rank adapters (`lora_add`) against their definition in float64."""
import numpy as np
import pytest
import torch

from oracle import more_oracle as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(T, K, slices, R, L, dtype, seed, ids="mixed", whole=False, ranks=None):
    g = torch.Generator().manual_seed(seed)
    N, S = sum(slices), len(slices)
    if whole:  # few whole numbers, so that nothing is rounded on the way
        x = torch.zeros(T, K)
        at = torch.randint(0, K, (T, 4), generator=g)
        x.scatter_(1, at, torch.randint(-2, 3, (T, 4), generator=g).float())
        a = torch.randint(-1, 2, (L, S * R, K), generator=g).float()
        b = torch.zeros(L, N, R)
        b.scatter_(2, torch.randint(0, R, (L, N, 3), generator=g), torch.randint(-2, 3, (L, N, 3), generator=g).float())
        base = torch.randint(-20, 21, (T, N), generator=g).float()
        scalings = torch.randint(1, 3, (L,), generator=g).float()
    else:
        x = torch.randn(T, K, generator=g)
        a, b = torch.randn(L, S * R, K, generator=g) / K**0.5, torch.randn(L, N, R, generator=g) * 0.1
        base, scalings = torch.randn(T, N, generator=g), torch.rand(L, generator=g) * 2 - 0.5
    if ids == "mixed":  # each token its own; some name none, in either direction
        i = torch.randint(-2, L + 2, (T,), generator=g)
    elif ids == "runs":
        i = (torch.arange(T) * 5 // T) % (L + 1) - 1
    elif ids == "none":
        i = torch.full((T,), -1)
    else:
        i = torch.full((T,), int(ids))
    t = {"base": base, "x": x, "a": a, "b": b}
    t = {k: v.to(DT[dtype]) for k, v in t.items()}
    return {**t, "ids": i.to(torch.int32), "scalings": scalings, "ranks": ranks, "slices": tuple(slices)}


def _want(c):
    R = c["b"].shape[2]
    ranks = np.full(c["a"].shape[0], R) if c["ranks"] is None else c["ranks"].numpy()
    f = lambda t: t.double().numpy()
    a, b = f(c["a"]), f(c["b"])
    return O.lora_add(f(c["base"]), f(c["x"]), a, b, c["ids"].numpy(), f(c["scalings"]), ranks, c["slices"])


def _run(c, **kw):
    from sglang_b200 import ops
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    return ops.lora_add(d["base"], d["x"], d["a"], d["b"], d["ids"], d["scalings"], d["ranks"], d["slices"], **kw)


def _check(c, got):
    want, mass = _want(c)
    dtype, K, R = c["x"].dtype, c["x"].shape[1], c["b"].shape[2]
    assert got.dtype == dtype and got.shape == c["base"].shape
    g = got.cpu().double().numpy()
    # h: an instruction adds 16 exact products to a float32 sum and cuts off at most two units, then up to 64 parts; two terms of h keep it
    # to 2^-16 (bf16) of the row's largest, which R of them can be short of; the second product likewise; then one rounding to the type
    eps = torch.finfo(dtype).eps
    rel = ((K + 15) // 16 * 2 + 64 + (R + 15) // 16 * 4 + 8) * 2.0**-24
    live = (c["ids"].numpy() >= 0) & (c["ids"].numpy() < c["a"].shape[0])
    most = np.zeros(len(live))  # the most that one h of a token can be, through the largest weights
    for t in np.nonzero(live)[0]:
        l = c["ids"][t]
        rows = np.abs(np.nan_to_num(c["a"][l].double().numpy())) @ np.abs(c["x"][t].double().numpy())
        most[t] = rows.max() * np.abs(np.nan_to_num(c["b"][l].double().numpy())).max() * R * abs(float(c["scalings"][l]))
    tol = rel * mass + 2.0**-16 * most[:, None] + (np.abs(want) + 2.0**-16 * most[:, None]) * eps / 2 * 1.01 + float(torch.finfo(dtype).tiny) * eps
    err = np.abs(g - want)
    assert np.isfinite(g).all() and (err <= tol).all(), (err / tol).max()
    np.testing.assert_array_equal(g[~live], c["base"].double().numpy()[~live])


SIZES = [(1, 256, [64], 8, 1), (1, 7168, [2112], 16, 4), (5, 264, [100], 24, 3), (64, 512, [256, 256], 32, 16), (70, 1000, [96, 33, 64], 8, 40),
         (130, 512, [264, 8, 8], 64, 3), (33, 136, [72], 128, 2), (20, 64, [40, 24], 256, 5), (200, 128, [1000], 16, 1), (513, 192, [320], 40, 7),
         (17, 2048, [777], 200, 2)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("ids", ["mixed", "runs"])
@pytest.mark.parametrize("T,K,slices,R,L", SIZES)
def test_lora(T, K, slices, R, L, ids, dtype):
    c = _case(T, K, slices, R, L, dtype, T + K, ids)
    _check(c, _run(c))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("ids", ["mixed", "runs", "0"])
@pytest.mark.parametrize("T,K,slices,R,L", SIZES + [(1500, 256, [512, 264], 64, 4), (1100, 264, [136], 128, 2), (2100, 128, [96, 40, 32], 16, 9)])
def test_whole_numbers_are_exact(T, K, slices, R, L, ids, dtype):
    """Values that every step holds exactly: each weight of each adapter has to meet its token once."""
    c = _case(T, K, slices, R, L, dtype, 7 * T + K, ids, whole=True)
    want, mass = _want(c)
    keep = np.abs(want) <= 256  # (what 8 bits hold)
    assert keep.mean() > 0.99
    got = _run(c).cpu().double().numpy()
    np.testing.assert_array_equal(got[keep], want[keep])


@pytest.mark.parametrize("ids", ["mixed", "runs"])
@pytest.mark.parametrize("T", [3, 90, 1200])
def test_ranks_of_their_own_and_what_lies_beyond(T, ids):
    """Adapters of smaller rank in buffers of the largest: whatever an earlier adapter left there, NaN as well, is not used."""
    L, R, K, slices = 6, 32, 256, (72, 56)
    ranks = torch.tensor([32, 0, 5, 16, 31, 8], dtype=torch.int32)
    c = _case(T, K, slices, R, L, "bf16", T, ids, ranks=ranks)
    for l, r in enumerate(ranks.tolist()):
        c["b"][l, :, r:] = float("nan")
        for s in range(len(slices)):
            c["a"][l, s * R + r : (s + 1) * R] = float("inf")
    got = _run(c)
    for l, r in enumerate(ranks.tolist()):  # (the oracle multiplies whole rows)
        c["b"][l, :, r:] = 0
        for s in range(len(slices)):
            c["a"][l, s * R + r : (s + 1) * R] = 0
    _check(c, got)


@pytest.mark.parametrize("T", [1, 40, 1100])
def test_no_adapter_anywhere(T):
    c = _case(T, 128, [96], 16, 2, "bf16", T, "none")
    assert torch.equal(_run(c).cpu(), c["base"])


@pytest.mark.parametrize("T", [1, 40, 1100])
@pytest.mark.parametrize("N", [96, 77])
def test_in_place_and_rows_apart(T, N):
    """Into base itself; and rows of a wider buffer, whose other columns stay."""
    from sglang_b200 import ops
    c = _case(T, 128, [N], 16, 3, "bf16", T + N, "mixed")
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    want = _run(c)
    mine = d["base"].clone()
    got = ops.lora_add(mine, d["x"], d["a"], d["b"], d["ids"], d["scalings"], out=mine)
    assert got.data_ptr() == mine.data_ptr() and torch.equal(mine, want)
    for lead in (8, 3):
        wide_x, wide = torch.randn(T, 128 + 40, device="cuda").to(torch.bfloat16), torch.randn(T, N + 40, device="cuda").to(torch.bfloat16)
        wide_x[:, 16:144], wide[:, lead : lead + N] = d["x"], d["base"]
        before = wide.clone()
        view = wide[:, lead : lead + N]
        ops.lora_add(view, wide_x[:, 16:144], d["a"], d["b"], d["ids"], d["scalings"], out=view)
        assert torch.equal(view, want)
        assert torch.equal(wide[:, :lead], before[:, :lead]) and torch.equal(wide[:, lead + N :], before[:, lead + N :])
        apart = ops.lora_add(before[:, lead : lead + N], d["x"], d["a"], d["b"], d["ids"], d["scalings"])
        assert torch.equal(apart, want)


def test_magnitudes_that_leave_float16():
    """h beyond float16's range, and h below its smallest, against weights that bring the sums back."""
    c = _case(40, 256, [64], 16, 3, "fp16", 5, "mixed")
    for big in (200.0, 2.0**-14):
        d = dict(c, x=(c["x"].float() * big).half(), a=(c["a"].float() * (64 if big > 1 else 2.0**-6)).half())
        d["scalings"] = c["scalings"] / (big * (64 if big > 1 else 2.0**-6))
        _check(d, _run(d))


def test_infinities_and_nan_stay_in_their_rows():
    c = _case(100, 128, [72], 16, 3, "bf16", 8, "1")
    want = _run(c)
    c["x"][5, 3], c["x"][70, 9], c["base"][9, 4] = float("nan"), float("inf"), float("nan")
    got = _run(c)
    keep = [t for t in range(100) if t not in (5, 9, 70)]
    assert torch.equal(got[keep], want[keep]) and got[5].isnan().all() and not got[70].isfinite().any()
    assert got[9, 4].isnan() and torch.equal(got[9, 5:], want[9, 5:])


def test_leading_dimensions_and_no_tokens():
    from sglang_b200 import ops
    c = _case(24, 128, [72], 16, 3, "bf16", 9, "mixed")
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    got = ops.lora_add(d["base"].view(4, 6, 72), d["x"].view(4, 6, 128), d["a"], d["b"], d["ids"].view(4, 6), d["scalings"])
    assert torch.equal(got.view(24, 72), _run(c))
    none = ops.lora_add(d["base"][:0], d["x"][:0], d["a"], d["b"], d["ids"][:0])
    assert tuple(none.shape) == (0, 72)


@pytest.mark.parametrize("T", [64, 65, 257, 3000])
def test_most_adapters_and_slices(T):
    c = _case(T, 64, [8, 16, 24, 8, 40, 8, 8, 16], 8, 1024, "bf16", T, "mixed", whole=True)
    want, _ = _want(c)
    np.testing.assert_array_equal(_run(c).cpu().double().numpy(), want)


@pytest.mark.parametrize("T", [1, 70, 2100])
def test_offsets_beyond_32_bits(T):
    """An adapter behind 2^31 others' weights; 2100 tokens' rows of base and out pass 2^31 values as well."""
    from sglang_b200 import ops
    L, N, R, K = 40, 1 << 20, 56, 64
    g = torch.Generator(device="cuda").manual_seed(T)
    b = torch.zeros(L, N, R, device="cuda", dtype=torch.bfloat16)
    a = torch.zeros(L, R, K, device="cuda", dtype=torch.bfloat16)
    b[L - 1] = torch.randint(-1, 2, (N, R), generator=g, device="cuda").to(torch.bfloat16)
    a[L - 1, torch.arange(R), torch.arange(R)] = 1  # h = the first R of x
    x = torch.randint(-1, 2, (T, K), generator=g, device="cuda").to(torch.bfloat16)
    base = torch.zeros(T, N, device="cuda", dtype=torch.bfloat16)
    base[:, ::7] = 3
    ids = torch.full((T,), L - 1, dtype=torch.int32, device="cuda")
    got = ops.lora_add(base, x, a, b, ids)
    for c0 in (0, N // 2 + 24, N - 1000):
        cols = slice(c0, c0 + 1000)
        want = base[:, cols].double() + x[:, :R].double() @ b[L - 1, cols].double().t()
        assert torch.equal(got[:, cols].double(), want)


def test_columns_of_one_buffer():
    """base and out side by side in one buffer."""
    from sglang_b200 import ops
    c = _case(90, 128, [72], 16, 3, "bf16", 11, "mixed")
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    both = torch.zeros(90, 160, device="cuda", dtype=torch.bfloat16)
    both[:, :72] = d["base"]
    ops.lora_add(both[:, :72], d["x"], d["a"], d["b"], d["ids"], d["scalings"], out=both[:, 80:152])
    assert torch.equal(both[:, 80:152], _run(c)) and torch.equal(both[:, :72], d["base"]) and both[:, 72:80].eq(0).all()
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.lora_add(both[:, :72], d["x"], d["a"], d["b"], d["ids"], d["scalings"], out=both[:, 8:80])
