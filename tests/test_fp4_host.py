"""What the 4-bit operators refuse, and their host-side pieces (no GPU needed)."""
import numpy as np
import pytest
import torch

from oracle import fp4_oracle as F


def _err():
    from sglang_b200._lib import lib
    return lib.sglb200_last_error().decode()


QUANTIZERS = ["sglb200_per_token_group_quant_fp4", "sglb200_silu_and_mul_quant_fp4"]


@pytest.mark.parametrize("name", QUANTIZERS)
def test_quantizers_refuse(name):
    from sglang_b200._lib import lib
    fn, A = getattr(lib, name), 4096  # A: an aligned address that is never touched
    assert fn(A, 0, A, A, None, 4, 64, 64, None) == -2 and "group_size" in _err()
    assert fn(A, 0, A, A, None, 4, 72, 16, None) == -1 and "not divisible" in _err()
    assert fn(A, 0, A, A, None, 4, 48, 32, None) == -1 and "not divisible" in _err()
    assert fn(A, 0, A, A, None, 4, 0, 16, None) == -1
    assert fn(A, 0, A, A, None, -1, 64, 16, None) == -1
    assert fn(A, 0, A, A, None, 4, (1 << 20) + 32, 32, None) == -1 and "2^20" in _err()
    assert fn(A, 0, A, A, A, 4, 64, 32, None) == -1 and "no global scale" in _err()
    assert fn(A, 0, A, A, A + 2, 4, 64, 16, None) == -1 and "aligned" in _err()
    assert fn(A, 3, A, A, None, 4, 64, 16, None) == -2 and "dtype" in _err()
    assert fn(None, 0, A, A, None, 4, 64, 16, None) == -1 and "null" in _err()
    assert fn(A + 8, 0, A, A, None, 4, 64, 16, None) == -1 and "16-byte" in _err()
    assert fn(A, 0, A, A, None, 0, 64, 16, None) == 0  # no rows: nothing to do
    if "silu" in name:
        assert fn(A, 2, A, A, None, 4, 64, 16, None) == -2 and "dtype" in _err()


def test_dequantizer_refuses():
    from sglang_b200._lib import lib
    fn, A = lib.sglb200_per_token_group_dequant_fp4, 4096
    assert fn(A, A, None, A, 0, 4, 64, 8, None) == -2
    assert fn(A, A, None, A, 0, 4, 40, 16, None) == -1
    assert fn(A, A, A, A, 0, 4, 64, 32, None) == -1
    assert fn(A, A, None, A, 5, 4, 64, 16, None) == -2
    assert fn(A, None, None, A, 0, 4, 64, 16, None) == -1
    assert fn(A, A, None, A + 4, 0, 4, 64, 16, None) == -1
    assert fn(A, A, None, A, 0, 0, 64, 16, None) == 0


def test_python_forms_refuse_cpu_tensors_and_bad_arguments():
    from sglang_b200 import ops
    x = torch.zeros(4, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.per_token_group_quant_fp4(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.silu_and_mul_quant_fp4(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.per_token_group_dequant_fp4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(128, 4).to(torch.float8_e4m3fn))
    with pytest.raises(NotImplementedError, match="group_size"):
        ops.per_token_group_quant_fp4(x, None, 128)
    with pytest.raises(RuntimeError, match="float8"):
        ops.fp4_blocked_scales(torch.zeros(4, 4))


@pytest.mark.parametrize("rows,groups", [(1, 1), (3, 5), (128, 4), (129, 7), (300, 132)])
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e8m0fnu])
def test_blocked_scales(rows, groups, dtype):
    from sglang_b200 import ops
    codes = np.random.default_rng(rows).integers(0, 255, size=(rows, groups)).astype(np.uint8)
    got = ops.fp4_blocked_scales(torch.from_numpy(codes).view(dtype))
    assert got.dtype == dtype and tuple(got.shape) == ops.fp4_scale_shape(rows, groups * 16)
    got = got.view(torch.uint8).numpy()
    assert np.array_equal(got, F.blocked(codes))
    assert np.array_equal(F.unblocked(got, rows, groups), codes)


def test_oracle_format():
    """Known answers of the format: every code round-trips, ties go to the even mantissa, magnitudes saturate."""
    x = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, 0.2500001, 4.99, 5.01, 6.9, 0.0, -6.0]])
    codes, s = F.quantize(x * 1.0, 1.0, 16)
    # amax 6.9 / 6 = 1.15 -> e4m3 1.125
    assert s[0, 0] == 0x39
    full = x.copy()
    full[0, 13] = 6.0
    codes, s = F.quantize(full, 1.0, 16)
    assert s[0, 0] == 0x38
    v = F.dequantize(codes, s, 16)[0]
    assert v.tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, -0.0, -1.0, 0.5, 4.0, 6.0, 6.0, 0.0, -6.0]
    codes, s = F.quantize(np.array([[7.9] + [1.0] * 31]), 1.0, 32)
    assert s[0, 0] == 127 and F.dequantize(codes, s, 32)[0, 0] == 6.0
    codes, s = F.quantize(np.array([[8.0] + [1.0] * 31]), 1.0, 32)
    assert s[0, 0] == 128 and F.dequantize(codes, s, 32)[0, 0] == 8.0
    t = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(t, F.E4M3)


def test_product_refuses():
    from sglang_b200._lib import lib
    A = 4096

    def call(M=4, N=16, K=64, group=16, dt=0, a=A, b=A, sa=A, sb=A, alpha=None, c=A, bias=None):
        return lib.sglb200_group_fp4_scaled_mm(a, b, sa, sb, alpha, c, bias, M, N, K, group, dt, None)

    assert call(group=64) == -2 and "group_size" in _err()
    assert call(dt=2) == -2 and "output dtype" in _err()
    assert call(K=48) == -1 and "divisible" in _err()
    assert call(N=12) == -1 and "divisible" in _err()
    assert call(K=0) == -1 and call(N=0) == -1 and call(M=-1) == -1
    assert call(K=(1 << 20) + 32) == -1 and "too large" in _err()
    assert call(M=(1 << 31)) == -1 and "too large" in _err()
    assert call(sa=None) == -1 and "null" in _err()
    assert call(c=A + 8) == -1 and "16-byte" in _err()
    assert call(bias=A + 2) == -1 and "16-byte" in _err()
    assert call(alpha=A + 1) == -1 and "alpha" in _err()
    assert call(M=0) == 0


def test_experts_refuse():
    from sglang_b200._lib import lib
    A = 4096
    size = lib.sglb200_fused_experts_fp4_workspace_bytes

    def call(T=2, k=2, E=8, H=256, I=128, dt=0, x=A, w13=A, s13=A, a13=None, w2=A, s2=A, a2=None, w=A, ids=A, out=A, ws=A, ws_bytes=None):
        if ws_bytes is None:
            ws_bytes = size(T, k, H, I)
        return lib.sglb200_fused_experts_fp4(x, dt, w13, s13, a13, w2, s2, a2, w, ids, out, T, k, E, H, I, 1.0, ws, ws_bytes, None)

    assert size(0, 2, 256, 128) == 0 and size(2, 2, 256, 128) >= 4 * (256 + 128) * 4
    assert call(dt=2) == -2
    assert call(H=240) == -1 and "divisible" in _err()
    assert call(I=80) == -1 and "divisible" in _err()
    assert call(E=0) == -1 and call(E=1025) == -1 and "experts" in _err()
    assert call(T=600) == -1 and "at most" in _err()
    assert call(T=1 << 40, k=1 << 40, ws_bytes=0) == -1 and "at most" in _err()
    assert call(k=0, ws_bytes=0) == -1 and call(T=-1, ws_bytes=0) == -1
    assert call(ids=None) == -1 and "null" in _err()
    assert call(x=A + 8) == -1 and "16-byte" in _err()
    assert call(ws=None) == -4 and "workspace" in _err()
    assert call(ws_bytes=16) == -4 and call(ws=A + 8) == -4
    assert call(T=0) == 0


def _code(name):
    """A source file without its comments."""
    import os
    import re
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sglang_b200", "csrc", name)
    return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S))


def test_tensor_memory_is_taken_after_the_kernel_in_front_and_before_the_one_behind():
    """A CTA that held tensor memory while it waits for the kernel in front could keep that kernel's last CTAs from getting theirs;
    one that let the next kernel in before it has its own could be kept waiting by it."""
    for name, kernel, alloc in (("fp4_gemm.cu", "fp4_rows_kernel(", "tmem_alloc("), ("fp4_pair.cu", "fp4_pair_kernel(", "pair_tmem_alloc(")):
        body = _code(name)
        body = body[body.index(kernel):]
        wait, take, let_in = (body.index(w) for w in ("grid_dependency_wait()", alloc, "launch_dependents()"))
        assert wait < take < let_in
        assert min(body.index("tma_load" if "rows" in kernel else "pair_load_2d("), body.index("p.alpha")) > let_in


def test_the_down_launch_reads_nothing_of_the_up_launch_before_its_wait():
    body = _code("fp4_moe.cu")
    body = body[body.index("fp4_experts_kernel(const __grid_constant__"):]
    products = body[body.index("const int wk = warp % warps_k"):]
    wait = products.index("if constexpr (!kUp) ptx::grid_dependency_wait();")
    assert wait < products.index("stage_rows") and wait < products.index("sum_slots") and wait < products.index("p.h")
    assert "p.x" not in body[:body.index("const int wk = warp % warps_k")] and "act_row" not in body[:body.index("const int wk = warp % warps_k")]
    # every thread of the down launch waits: a launch is over only when the one in front of it is
    assert body.count("if constexpr (!kUp) ptx::grid_dependency_wait();") == 3
    up = body[:body.index("route(p, ctl)")]
    assert up.index("grid_dependency_wait()") < up.index("launch_dependents()") < up.index("p.done[i] = 0")
