"""Tensor-level entry points: torch tensors in, C-ABI calls out.

Each function validates what the reference op validates (`CHECK_INPUT`,
`TORCH_CHECK`), hands raw device pointers plus the current CUDA stream to
`libsglang_b200.so`, and raises `RuntimeError` on a rejected call.  Nothing
here computes on the host and nothing synchronises the device.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from ._lib import check, host, lib

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
FP8_MIN = -448.0
ALIGN_BLOCK = 128  # row-block of the grouped GEMM; moe_align must be called with this block size

_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _cuda_contig(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def _dt(t: torch.Tensor, allow=(torch.bfloat16, torch.float16)) -> int:
    if t.dtype not in allow:
        raise RuntimeError(f"unsupported dtype {t.dtype}")
    return _DT[t.dtype]


# --------------------------------------------------------------------------------------------
# quantizer
# --------------------------------------------------------------------------------------------


def per_token_group_quant_fp8_out(
    x: torch.Tensor,
    x_q: torch.Tensor,
    x_s: torch.Tensor,
    group_size: int,
    eps: float = 1e-10,
    fp8_min: float = FP8_MIN,
    fp8_max: float = FP8_MAX,
) -> None:
    """Writes codes into `x_q` and scales into `x_s` (any 2-D strides: row-major or the
    M-major "column_major_scales" view)."""
    _cuda_contig(x, "input")
    _cuda_contig(x_q, "output_q")
    if x_q.dtype != FP8:
        raise RuntimeError("output_q must be float8_e4m3fn")
    if x_s.dtype != torch.float32 or not x_s.is_cuda:
        raise RuntimeError("output_s must be a float32 CUDA tensor")
    hidden = x.shape[-1]
    tokens = x.numel() // hidden if hidden else 0
    if x_q.numel() != x.numel():
        raise RuntimeError("output_q has the wrong number of elements")
    groups = hidden // group_size if group_size else 0
    if x_s.numel() == 0 and tokens == 0:
        return
    s2 = x_s.reshape(tokens, groups) if x_s.is_contiguous() else x_s
    if s2.dim() != 2 or s2.shape[0] != tokens or s2.shape[1] != groups:
        raise RuntimeError(f"output_s has shape {tuple(x_s.shape)}, expected [{tokens}, {groups}]")
    check(
        lib.sglb200_per_token_group_quant_fp8(
            x.data_ptr(), _dt(x, _DT), x_q.data_ptr(), s2.data_ptr(), tokens, hidden, int(group_size),
            float(eps), float(fp8_min), float(fp8_max), s2.stride(0), s2.stride(1), _stream(x),
        )
    )


def per_token_group_quant_fp8(
    x: torch.Tensor, group_size: int = 128, eps: float = 1e-10, column_major_scales: bool = False,
    scale_tma_aligned: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    out = host.quant(x, group_size, eps, column_major_scales, scale_tma_aligned)
    if out is not None:
        return out
    x_q = torch.empty_like(x, dtype=FP8)
    tokens = x.numel() // x.shape[-1]
    groups = x.shape[-1] // group_size
    if column_major_scales:
        pad = (tokens + 3) // 4 * 4 if scale_tma_aligned else tokens
        x_s = torch.empty((groups, pad), device=x.device, dtype=torch.float32).t()[:tokens, :]
    else:
        x_s = torch.empty(x.shape[:-1] + (groups,), device=x.device, dtype=torch.float32)
    if tokens > 0:
        per_token_group_quant_fp8_out(x, x_q, x_s, group_size, eps)
    return x_q, x_s


# --------------------------------------------------------------------------------------------
# 4-bit floating point
# --------------------------------------------------------------------------------------------

_FP4_SCALE = {16: torch.float8_e4m3fn, 32: torch.float8_e8m0fnu}


def _fp4_group(group_size: int, what: str) -> int:
    if group_size not in _FP4_SCALE:
        raise NotImplementedError(f"{what}: group_size must be 16 (e4m3 scales) or 32 (e8m0 scales), not {group_size}")
    return int(group_size)


def _scalar_f32(t: Optional[torch.Tensor], like: torch.Tensor, name: str) -> int:
    if t is None:
        return 0
    if not t.is_cuda or t.dtype != torch.float32 or t.numel() != 1 or t.device != like.device:
        raise RuntimeError(f"{name} must be one float32 on the device of the other tensors")
    return t.data_ptr()


def fp4_scale_shape(rows: int, hidden: int, group_size: int = 16) -> Tuple[int, int]:
    """Shape of the scales of [rows, hidden] values in blocked order: whole blocks of 128 rows x 4 groups."""
    return (rows + 127) // 128 * 128, (hidden // group_size + 3) // 4 * 4


def fp4_blocked_scales(scales: torch.Tensor) -> torch.Tensor:
    """Scales [rows, groups] in rows' order (as a checkpoint stores a weight's) -> blocked order, padded with zeros: what
    the 4-bit products read.  Laid out once, when the weight is loaded."""
    if scales.dim() != 2 or scales.dtype not in _FP4_SCALE.values():
        raise RuntimeError("fp4_blocked_scales: scales must be float8_e4m3fn or float8_e8m0fnu [rows, groups]")
    rows, groups = scales.shape
    mb, gb = (rows + 127) // 128, (groups + 3) // 4
    padded = torch.zeros(mb * 128, gb * 4, dtype=torch.uint8, device=scales.device)
    padded[:rows, :groups] = scales.contiguous().view(torch.uint8)
    return padded.view(mb, 4, 32, gb, 4).permute(0, 3, 2, 1, 4).reshape(mb * 128, gb * 4).view(scales.dtype)


def _quant_fp4(x, global_scale, group_size, silu, what):
    group = _fp4_group(group_size, what)
    _cuda_contig(x, "input")
    if x.dim() < 1 or x.shape[-1] == 0 or (silu and x.shape[-1] % 2):
        raise RuntimeError(f"{what}: the last dimension is empty" + (" or odd" if silu else ""))
    hidden = x.shape[-1] // (2 if silu else 1)
    rows = x.numel() // x.shape[-1]
    q = torch.empty(x.shape[:-1] + (hidden // 2,), device=x.device, dtype=torch.uint8)
    s = torch.empty(fp4_scale_shape(rows, hidden, group), device=x.device, dtype=_FP4_SCALE[group])
    g = _scalar_f32(global_scale, x, "global_scale")
    fn = lib.sglb200_silu_and_mul_quant_fp4 if silu else lib.sglb200_per_token_group_quant_fp4
    with torch.cuda.device(x.device):
        check(fn(x.data_ptr(), _dt(x, _DT if not silu else (torch.bfloat16, torch.float16)), q.data_ptr(), s.data_ptr(), g, rows,
                 hidden, group, _stream(x)))
    return q, s


def per_token_group_quant_fp4(
    x: torch.Tensor, global_scale: Optional[torch.Tensor] = None, group_size: int = 16,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [..., hidden] -> (codes uint8 [..., hidden / 2], scales in blocked order, `fp4_scale_shape`).

    `group_size` 16: s = e4m3(amax * global_scale / 6), code = e2m1(x * global_scale / s); `global_scale` is one float32 on
    the device (None: 1), customarily 448 * 6 / the tensor's largest magnitude.  `group_size` 32: s = 2^(floor(log2 amax) - 2),
    code = e2m1(x / s), no global scale.  A group that holds a NaN or an infinity gets the scale NaN."""
    out = host.quant_fp4(x, global_scale, group_size)
    return out if out is not None else _quant_fp4(x, global_scale, group_size, False, "per_token_group_quant_fp4")


def silu_and_mul_quant_fp4(
    x: torch.Tensor, global_scale: Optional[torch.Tensor] = None, group_size: int = 16,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """silu(x[..., :d]) * x[..., d:], unrounded, quantised as `per_token_group_quant_fp4` does; x [..., 2d]."""
    out = host.silu_mul_quant_fp4(x, global_scale, group_size)
    return out if out is not None else _quant_fp4(x, global_scale, group_size, True, "silu_and_mul_quant_fp4")


def _fp4_scales_ok(codes: torch.Tensor, scales: torch.Tensor, name: str) -> int:
    """The group size that the type of `scales` says, once their shape fits codes [..., hidden / 2]."""
    _cuda_contig(codes, name)
    _cuda_contig(scales, f"{name}'s scales")
    if codes.dtype != torch.uint8 or codes.dim() < 1 or codes.shape[-1] == 0:
        raise RuntimeError(f"{name} must be uint8 [..., hidden / 2]")
    group = next((g for g, t in _FP4_SCALE.items() if t == scales.dtype), None)
    if group is None:
        raise RuntimeError(f"{name}'s scales must be float8_e4m3fn (groups of 16) or float8_e8m0fnu (groups of 32)")
    hidden = codes.shape[-1] * 2
    want = fp4_scale_shape(codes.numel() // codes.shape[-1], hidden, group)
    if hidden % group or tuple(scales.shape) != want or scales.device != codes.device:
        raise RuntimeError(f"{name}'s scales have shape {tuple(scales.shape)}, expected {want} in blocked order")
    return group


def per_token_group_dequant_fp4(
    codes: torch.Tensor, scales: torch.Tensor, global_scale: Optional[torch.Tensor] = None,
    dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """The values code * s / global_scale [..., hidden] of codes [..., hidden / 2] with scales in blocked order."""
    out = host.dequant_fp4(codes, scales, global_scale, dtype)
    if out is not None:
        return out
    group = _fp4_scales_ok(codes, scales, "codes")
    if dtype not in _DT:
        raise RuntimeError(f"unsupported dtype {dtype}")
    hidden = codes.shape[-1] * 2
    out = torch.empty(codes.shape[:-1] + (hidden,), device=codes.device, dtype=dtype)
    g = _scalar_f32(global_scale, codes, "global_scale")
    with torch.cuda.device(codes.device):
        check(lib.sglb200_per_token_group_dequant_fp4(codes.data_ptr(), scales.data_ptr(), g, out.data_ptr(), _DT[dtype],
                                                      codes.numel() // codes.shape[-1], hidden, group, _stream(codes)))
    return out


# --------------------------------------------------------------------------------------------
# activation / reduction / gather
# --------------------------------------------------------------------------------------------


def silu_and_mul_out(out: torch.Tensor, x: torch.Tensor) -> None:
    _cuda_contig(x, "input")
    _cuda_contig(out, "out")
    d = x.shape[-1] // 2
    rows = x.numel() // x.shape[-1] if x.shape[-1] else 0
    if out.dtype != x.dtype or out.numel() != rows * d:
        raise RuntimeError("silu_and_mul: out must have input's dtype and half its last dimension")
    check(lib.sglb200_silu_and_mul(out.data_ptr(), x.data_ptr(), _dt(x), rows, d, _stream(x)))


def silu_and_mul_quant_fp8(
    x: torch.Tensor, group_size: int = 128, eps: float = 1e-10, num_rows: Optional[torch.Tensor] = None
) -> Tuple[torch.Tensor, torch.Tensor]:
    """[rows, 2d] -> (codes [rows, d], scales [rows, d/group]).  `num_rows` (device int32 scalar)
    limits the rows processed; the remaining rows of the outputs are left untouched."""
    out = host.silu_mul_quant(x, group_size, eps, num_rows)
    if out is not None:
        return out
    _cuda_contig(x, "input")
    d = x.shape[-1] // 2
    rows = x.numel() // x.shape[-1]
    q = torch.empty(x.shape[:-1] + (d,), device=x.device, dtype=FP8)
    s = torch.empty(x.shape[:-1] + (d // group_size,), device=x.device, dtype=torch.float32)
    nr = num_rows.data_ptr() if num_rows is not None else None
    check(
        lib.sglb200_silu_and_mul_quant_fp8(
            x.data_ptr(), _dt(x), q.data_ptr(), s.data_ptr(), rows, d, int(group_size), float(eps), nr, _stream(x)
        )
    )
    return q, s


def silu_and_mul_masked_quant_fp8_out(x: torch.Tensor, out_q: torch.Tensor, out_s: torch.Tensor, masked_m: torch.Tensor,
                                      group_size: int = 128, eps: float = 1e-10) -> None:
    """Masked expert layout: x [E, T_pad, 2d]; rows t < masked_m[e] of expert e are activated and quantised into
    out_q [E, T_pad, d] / out_s [E, T_pad, d/group] (float32), every other row of the outputs is left untouched."""
    for t, n in ((x, "input"), (out_q, "output"), (out_s, "output_scale"), (masked_m, "masked_m")):
        _cuda_contig(t, n)
    if x.dim() != 3 or x.shape[-1] % 2:
        raise RuntimeError("silu_and_mul_masked_quant: input must be [experts, padded tokens, 2d]")
    E, T, d2 = x.shape
    d = d2 // 2
    if out_q.dtype != FP8 or tuple(out_q.shape) != (E, T, d):
        raise RuntimeError("silu_and_mul_masked_quant: output must be float8_e4m3fn [experts, padded tokens, d]")
    if out_s.dtype != torch.float32 or tuple(out_s.shape) != (E, T, d // group_size):
        raise RuntimeError("silu_and_mul_masked_quant: output_scale must be float32 [experts, padded tokens, d/group]")
    if masked_m.dtype != torch.int32 or tuple(masked_m.shape) != (E,):
        raise RuntimeError("silu_and_mul_masked_quant: masked_m must be int32 [experts]")
    check(lib.sglb200_silu_and_mul_masked_quant_fp8(x.data_ptr(), _dt(x), out_q.data_ptr(), out_s.data_ptr(), E, T, d,
                                                    int(group_size), float(eps), masked_m.data_ptr(), _stream(x)))


def moe_sum_reduce_out(x: torch.Tensor, out: torch.Tensor, routed_scaling_factor: float) -> None:
    _cuda_contig(x, "input")
    _cuda_contig(out, "output")
    if x.dim() != 3 or out.dim() != 2 or out.shape[0] != x.shape[0] or out.shape[1] != x.shape[2]:
        raise RuntimeError("moe_sum_reduce: input [tokens, topk, hidden], output [tokens, hidden]")
    if out.dtype != x.dtype:
        raise RuntimeError("moe_sum_reduce: dtype mismatch")
    t, k, h = x.shape
    check(lib.sglb200_moe_sum_reduce(x.data_ptr(), out.data_ptr(), _dt(x), t, k, h, float(routed_scaling_factor), _stream(x)))


def moe_sum_reduce_masked_out(x: torch.Tensor, topk_ids: torch.Tensor, out: torch.Tensor,
                              routed_scaling_factor: float) -> None:
    """moe_sum_reduce over the slots whose id in `topk_ids` [tokens, topk] (int32) is not negative."""
    _cuda_contig(x, "input")
    _cuda_contig(out, "output")
    _cuda_contig(topk_ids, "topk_ids")
    if x.dim() != 3 or out.dim() != 2 or out.shape[0] != x.shape[0] or out.shape[1] != x.shape[2]:
        raise RuntimeError("moe_sum_reduce: input [tokens, topk, hidden], output [tokens, hidden]")
    if out.dtype != x.dtype or topk_ids.dtype != torch.int32 or tuple(topk_ids.shape) != tuple(x.shape[:2]):
        raise RuntimeError("moe_sum_reduce: dtype or shape mismatch")
    t, k, h = x.shape
    check(lib.sglb200_moe_sum_reduce_masked(x.data_ptr(), topk_ids.data_ptr(), out.data_ptr(), _dt(x), t, k, h,
                                            float(routed_scaling_factor), _stream(x)))


def gather_sum_rows(src: torch.Tensor, slot: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """out[t] = scale * sum_j src[slot[t, j]] (float32 accumulation); slots outside [0, len(src)) are skipped."""
    _cuda_contig(src, "src")
    _cuda_contig(slot, "slot")
    if src.dim() != 2 or slot.dim() != 2 or slot.dtype != torch.int64:
        raise RuntimeError("gather_sum_rows: src [rows, hidden], slot [tokens, per_token] int64")
    out = torch.empty((slot.shape[0], src.shape[1]), dtype=src.dtype, device=src.device)
    check(lib.sglb200_gather_sum_rows(src.data_ptr(), slot.data_ptr(), out.data_ptr(), _dt(src), slot.shape[0],
                                      slot.shape[1], src.shape[0], src.shape[1], float(scale), _stream(src)))
    return out


def shuffle_mul_sum_out(input: torch.Tensor, output: torch.Tensor, permutation: torch.Tensor,
                        factors: Optional[torch.Tensor] = None) -> None:
    """output[t] = sum_j factors[t, j] * input[permutation[t * topk + j]] (float32 accumulation)."""
    _cuda_contig(input, "input")
    _cuda_contig(output, "output")
    _cuda_contig(permutation, "permutation")
    tokens, hidden = output.shape
    if permutation.dtype != torch.int32 or tokens == 0 or permutation.numel() % max(tokens, 1):
        raise RuntimeError("apply_shuffle_mul_sum: permutation must be int32 with tokens * topk entries")
    topk = permutation.numel() // tokens
    if input.dtype != output.dtype or input.shape[1] != hidden:
        raise RuntimeError("apply_shuffle_mul_sum: input [tokens * topk, hidden] and output [tokens, hidden] of one dtype")
    f = 0
    if factors is not None:
        _cuda_contig(factors, "factors")
        if factors.dtype != output.dtype or factors.numel() != permutation.numel():
            raise RuntimeError("apply_shuffle_mul_sum: factors must match the output dtype and have tokens * topk entries")
        f = factors.data_ptr()
    check(lib.sglb200_shuffle_mul_sum(input.data_ptr(), output.data_ptr(), permutation.data_ptr(), f, _dt(output), tokens,
                                      topk, hidden, _stream(output)))


_GATE_DT = (torch.bfloat16, torch.float16, torch.float32)


def _gate_io(gating: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor, what: str):
    _cuda_contig(gating, "gating_output")
    _cuda_contig(topk_weights, "topk_weights")
    _cuda_contig(topk_ids, "topk_ids")
    if gating.dim() != 2 or topk_weights.shape != topk_ids.shape or topk_weights.shape[0] != gating.shape[0]:
        raise RuntimeError(f"{what}: gating [tokens, experts], outputs [tokens, topk]")
    if topk_weights.dtype != torch.float32 or topk_ids.dtype != torch.int32:
        raise RuntimeError(f"{what}: topk_weights must be float32 and topk_ids int32")
    return gating.shape[0], gating.shape[1], topk_weights.shape[1]


def _gate_bias(correction_bias: Optional[torch.Tensor], experts: int, what: str) -> int:
    if correction_bias is None:
        return 0
    _cuda_contig(correction_bias, "correction_bias")
    if correction_bias.dtype != torch.float32 or correction_bias.numel() != experts:
        raise RuntimeError(f"{what}: correction_bias must be float32 [num_experts]")
    return correction_bias.data_ptr()


def topk_softmax_out(topk_weights, topk_ids, gating, renormalize=False, moe_softcapping=0.0, correction_bias=None) -> None:
    rows, experts, k = _gate_io(gating, topk_weights, topk_ids, "topk_softmax")
    check(lib.sglb200_topk_softmax(gating.data_ptr(), _dt(gating, _GATE_DT), rows, experts, k, int(bool(renormalize)),
                                   float(moe_softcapping), _gate_bias(correction_bias, experts, "topk_softmax"),
                                   topk_weights.data_ptr(), topk_ids.data_ptr(), _stream(gating)))


def topk_sigmoid_out(topk_weights, topk_ids, gating, renormalize=False, correction_bias=None) -> None:
    rows, experts, k = _gate_io(gating, topk_weights, topk_ids, "topk_sigmoid")
    check(lib.sglb200_topk_sigmoid(gating.data_ptr(), _dt(gating, _GATE_DT), rows, experts, k, int(bool(renormalize)),
                                   _gate_bias(correction_bias, experts, "topk_sigmoid"), topk_weights.data_ptr(),
                                   topk_ids.data_ptr(), _stream(gating)))


def moe_fused_gate(input: torch.Tensor, bias: torch.Tensor, num_expert_group: int, topk_group: int, topk: int,
                   num_fused_shared_experts: int = 0, routed_scaling_factor: float = 0.0,
                   apply_routed_scaling_factor_on_output: bool = False):
    out = host.fused_gate(input, bias, num_expert_group, topk_group, topk, num_fused_shared_experts,
                          routed_scaling_factor, bool(apply_routed_scaling_factor_on_output))
    if out is not None:
        return out
    _cuda_contig(input, "input")
    _cuda_contig(bias, "bias")
    if input.dim() != 2 or bias.numel() != input.shape[1] or bias.dtype != input.dtype:
        raise RuntimeError("moe_fused_gate: input [tokens, experts] and bias [experts] of the same dtype")
    rows, experts = input.shape
    w = torch.empty(rows, topk, dtype=torch.float32, device=input.device)
    ids = torch.empty(rows, topk, dtype=torch.int32, device=input.device)
    check(lib.sglb200_moe_fused_gate(input.data_ptr(), bias.data_ptr(), _dt(input, _GATE_DT), rows, experts, int(num_expert_group),
                                     int(topk_group), int(topk), int(num_fused_shared_experts),
                                     float(routed_scaling_factor), int(bool(apply_routed_scaling_factor_on_output)),
                                     w.data_ptr(), ids.data_ptr(), _stream(input)))
    return w, ids


def _same_device(like: torch.Tensor, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != like.device:
            raise RuntimeError(f"{name} is on {t.device}, the other tensors on {like.device}")


def _rows_view(t: torch.Tensor, name: str) -> torch.Tensor:
    """`t` [..., n] as rows with neighbouring columns, any one distance apart: a view, never a copy."""
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dim() < 1 or t.shape[-1] == 0:
        raise RuntimeError(f"{name}: the last dimension is empty")
    if t.dim() == 2:
        rows = t
    elif t.dim() == 1:
        rows = t[None]
    else:
        try:
            rows = t.view(-1, t.shape[-1]) if t.numel() else t.reshape(0, t.shape[-1])
        except RuntimeError as e:
            raise RuntimeError(f"{name}: its rows are not one distance apart") from e
    if rows.shape[0] and (rows.stride(1) != 1 and rows.shape[1] > 1 or rows.shape[0] > 1 and rows.stride(0) < rows.shape[1]):
        raise RuntimeError(f"{name}: strides {t.stride()}; columns must be neighbours and rows not overlap")
    return rows


def _row_stride(rows: torch.Tensor) -> int:
    return rows.stride(0) if rows.shape[0] > 1 else rows.shape[1]


def router_logits(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """The router's product: float32 [..., E] of x [..., K] and weight [E, K], both bf16 or both fp16; float32 sums, nothing rounded.
    Rows of x may lie apart.  K % 8 == 0."""
    out = host.router_logits(x, weight)
    if out is not None:
        return out
    rows = _rows_view(x, "x")
    _cuda_contig(weight, "weight")
    _same_device(x, weight=weight)
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.dtype != x.dtype or weight.shape[0] == 0:
        raise RuntimeError(f"router_logits: weight {tuple(weight.shape)} {weight.dtype} for x [..., {x.shape[-1]}] {x.dtype}")
    dt = _dt(x)
    with torch.cuda.device(x.device):
        y = torch.empty(x.shape[:-1] + (weight.shape[0],), device=x.device, dtype=torch.float32)
        check(lib.sglb200_router_logits(rows.data_ptr(), weight.data_ptr(), dt, y.data_ptr(), rows.shape[0], weight.shape[0],
                                        x.shape[-1], _row_stride(rows), _stream(x)))
    return y


def route_topk(
    gating_output: torch.Tensor, topk: int, scoring_func: str = "softmax", correction_bias: Optional[torch.Tensor] = None,
    num_expert_group: int = 1, topk_group: int = 1, group_top: Optional[int] = None, renormalize: bool = True,
    routed_scaling_factor: float = 1.0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Experts and weights from the router's logits [T, E] (bf16, fp16, fp32) -> (float32 [T, topk], int32 [T, topk]), best first.

    s = softmax or sigmoid of the logits, c = s + correction_bias (float32 [E]).  The experts form `num_expert_group` equal groups; a
    group's value is the sum of its `group_top` (1 or 2; None: 2 with a bias, else 1) largest c, and the `topk` largest c of the
    `topk_group` best groups are picked.  Weights are s, divided by the picks' sum if `renormalize`, times `routed_scaling_factor`.

    The order is that of the real numbers as far as float64 tells them, whatever the logits' type: c that are equal there go by their logits
    (sigmoids of logits from 37 on are all 1), equal ones to the lower index; sums of two to the lower group.  An expert whose logit is NaN or -inf
    (or whose bias is NaN or -inf) is not available; a slot for which none is left has the id -1 and the weight 0, which the experts'
    operators skip.  topk and num_expert_group at most 32."""
    if scoring_func not in ("softmax", "sigmoid"):
        raise RuntimeError(f"route_topk: scoring_func must be 'softmax' or 'sigmoid', not {scoring_func!r}")
    if group_top is None:
        group_top = 1 if correction_bias is None else 2
    out = host.route_topk(gating_output, topk, scoring_func == "softmax", correction_bias, num_expert_group, topk_group, group_top,
                          renormalize, routed_scaling_factor)
    if out is not None:
        return out
    _cuda_contig(gating_output, "gating_output")
    if gating_output.dim() != 2:
        raise RuntimeError("route_topk: gating_output must be [tokens, experts]")
    rows, experts = gating_output.shape
    dt, bias = _dt(gating_output, _GATE_DT), _gate_bias(correction_bias, experts, "route_topk")
    _same_device(gating_output, correction_bias=correction_bias)
    for n, v, most in (("topk", topk, experts), ("num_expert_group", num_expert_group, experts), ("topk_group", topk_group, num_expert_group),
                       ("group_top", group_top, 2)):
        if not 1 <= v <= most:
            raise RuntimeError(f"route_topk: {n} is {v}, not one of 1 to {most}")
    with torch.cuda.device(gating_output.device):
        w = torch.empty(rows, topk, dtype=torch.float32, device=gating_output.device)
        ids = torch.empty(rows, topk, dtype=torch.int32, device=gating_output.device)
        check(lib.sglb200_route_topk(gating_output.data_ptr(), dt, rows, experts, int(topk), int(scoring_func == "softmax"), bias,
                                     int(num_expert_group), int(topk_group), int(group_top), int(bool(renormalize)),
                                     float(routed_scaling_factor), w.data_ptr(), ids.data_ptr(), _stream(gating_output)))
    return w, ids


def gather_rows_fp8(
    src_q: torch.Tensor, src_s: torch.Tensor, sorted_token_ids: torch.Tensor, num_rows: torch.Tensor,
    numel: int, topk: int, max_rows: Optional[int] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of (src_q, src_s) in expert-sorted order; padding rows are zero."""
    _cuda_contig(src_q, "src_q")
    _cuda_contig(src_s, "src_s")
    hidden, groups = src_q.shape[-1], src_s.shape[-1]
    if max_rows is None:
        max_rows = sorted_token_ids.numel()
    dst_q = torch.empty((max_rows, hidden), device=src_q.device, dtype=src_q.dtype)
    dst_s = torch.empty((max_rows, groups), device=src_q.device, dtype=torch.float32)
    check(
        lib.sglb200_gather_rows_fp8(
            src_q.data_ptr(), src_s.data_ptr(), dst_q.data_ptr(), dst_s.data_ptr(), sorted_token_ids.data_ptr(),
            num_rows.data_ptr(), max_rows, numel, topk, hidden, groups, _stream(src_q),
        )
    )
    return dst_q, dst_s


# --------------------------------------------------------------------------------------------
# moe_align_block_size
# --------------------------------------------------------------------------------------------


def moe_align_block_size_out(
    topk_ids: torch.Tensor, num_experts: int, block_size: int, sorted_token_ids: torch.Tensor,
    experts_ids: torch.Tensor, num_tokens_post_pad: torch.Tensor, cumsum_buffer: torch.Tensor,
    pad_sorted_token_ids: bool = False,
) -> None:
    """`num_experts` is the bucket count (model experts + 1), as the reference op is called."""
    _cuda_contig(topk_ids, "topk_ids")
    if topk_ids.dtype != torch.int32:
        raise RuntimeError("topk_ids must be int32")
    for t, n in ((sorted_token_ids, "sorted_token_ids"), (experts_ids, "experts_ids"),
                 (num_tokens_post_pad, "num_tokens_post_pad"), (cumsum_buffer, "cumsum_buffer")):
        _cuda_contig(t, n)
        if t.dtype != torch.int32:
            raise RuntimeError(f"{n} must be int32")
    numel = topk_ids.numel()
    if cumsum_buffer.numel() < num_experts + 1:
        raise RuntimeError("cumsum_buffer needs num_experts + 1 entries")
    if sorted_token_ids.numel() < numel + num_experts * (block_size - 1) and numel > 0:
        # the exact worst case is min(numel, buckets) * (block-1); accept the reference's allocation
        pass
    ws_bytes = lib.sglb200_moe_align_workspace_bytes(numel, int(num_experts))
    ws = torch.empty(ws_bytes, device=topk_ids.device, dtype=torch.uint8) if ws_bytes else None
    check(
        lib.sglb200_moe_align_block_size(
            topk_ids.data_ptr(), numel, int(num_experts), int(block_size), sorted_token_ids.data_ptr(),
            experts_ids.data_ptr(), num_tokens_post_pad.data_ptr(), cumsum_buffer.data_ptr(),
            1 if pad_sorted_token_ids else 0, ws.data_ptr() if ws is not None else None, ws_bytes, _stream(topk_ids),
        )
    )


def moe_align_block_size(topk_ids: torch.Tensor, block_size: int, num_experts: int):
    """Python-level wrapper with the reference's allocation rules
    (fused_moe_triton/moe_align_block_size.py:57-81).  `num_experts` = model experts."""
    max_padded = topk_ids.numel() + (num_experts + 1) * (block_size - 1)
    dev = topk_ids.device
    sorted_ids = torch.empty((max_padded,), dtype=torch.int32, device=dev)
    expert_ids = torch.empty(((max_padded + block_size - 1) // block_size,), dtype=torch.int32, device=dev)
    post = torch.empty((1,), dtype=torch.int32, device=dev)
    cumsum = torch.empty((num_experts + 2,), dtype=torch.int32, device=dev)
    moe_align_block_size_out(topk_ids, num_experts + 1, block_size, sorted_ids, expert_ids, post, cumsum, True)
    return sorted_ids, expert_ids, post


def moe_align_block_size_local(topk_ids: torch.Tensor, block_size: int, num_experts: int):
    """The sort without its segment of filtered ids (-1 = expert of another rank): rows of local experts only."""
    max_padded = topk_ids.numel() + (num_experts + 1) * (block_size - 1)
    dev = topk_ids.device
    nblk = (max_padded + block_size - 1) // block_size
    sorted_ids = torch.empty((2, max_padded), dtype=torch.int32, device=dev)
    expert_ids = torch.empty((2, nblk), dtype=torch.int32, device=dev)
    post = torch.empty((2,), dtype=torch.int32, device=dev)
    cumsum = torch.empty((num_experts + 2,), dtype=torch.int32, device=dev)
    moe_align_block_size_out(topk_ids, num_experts + 1, block_size, sorted_ids[0], expert_ids[0], post[0:1], cumsum, True)
    check(lib.sglb200_moe_align_drop_filtered(
        sorted_ids[0].data_ptr(), expert_ids[0].data_ptr(), cumsum.data_ptr(), post[0:1].data_ptr(),
        sorted_ids[1].data_ptr(), expert_ids[1].data_ptr(), post[1:2].data_ptr(), max_padded, int(block_size),
        _stream(topk_ids)))
    return sorted_ids[1], expert_ids[1], post[1:2]


# --------------------------------------------------------------------------------------------
# GEMMs
# --------------------------------------------------------------------------------------------


def w8a8_block_fp8_matmul(
    A: torch.Tensor, B: torch.Tensor, As: torch.Tensor, Bs: torch.Tensor, block_size=(128, 128),
    output_dtype: torch.dtype = torch.bfloat16, bias: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """A [..., K] e4m3, B [N, K] e4m3, As [..., ceil(K/128)] f32 (any strides), Bs [ceil(N/128), ceil(K/128)] f32."""
    if list(block_size) != [128, 128]:
        raise RuntimeError("only block_size [128, 128] is supported")
    C = host.matmul(A, B, As, Bs, output_dtype, bias)
    if C is not None:
        return C
    _cuda_contig(A, "A")
    _cuda_contig(B, "B")
    if A.dtype != FP8 or B.dtype != FP8:
        raise RuntimeError("A and B must be float8_e4m3fn")
    if output_dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError("output dtype must be bfloat16 or float16")
    K = A.shape[-1]
    M = A.numel() // K if K else 0
    N = B.shape[0]
    if B.dim() != 2 or B.shape[1] != K:
        raise RuntimeError("B must be [N, K] with K matching A")
    kb, nb = (K + 127) // 128, (N + 127) // 128
    Bs = Bs.contiguous()
    if Bs.dtype != torch.float32 or tuple(Bs.shape) != (nb, kb):
        raise RuntimeError(f"Bs must be float32 [{nb}, {kb}]")
    As2 = As.reshape(M, kb) if As.is_contiguous() else As
    if As2.dtype != torch.float32 or As2.dim() != 2 or tuple(As2.shape) != (M, kb):
        raise RuntimeError(f"As must be float32 [{M}, {kb}]")
    C = torch.empty(A.shape[:-1] + (N,), device=A.device, dtype=output_dtype)
    if bias is not None:
        bias = bias.to(output_dtype).contiguous()
    if M > 0:
        ws_bytes = lib.sglb200_gemm_workspace_bytes(M, N, K)  # split-K scratch for the small-M regime
        ws = torch.empty(ws_bytes, device=A.device, dtype=torch.uint8) if ws_bytes else None
        check(
            lib.sglb200_fp8_blockwise_scaled_mm(
                A.data_ptr(), B.data_ptr(), As2.data_ptr(), Bs.data_ptr(), C.data_ptr(),
                bias.data_ptr() if bias is not None else None, M, N, K, As2.stride(0), As2.stride(1),
                0 if output_dtype == torch.bfloat16 else 1, ws.data_ptr() if ws is not None else None, ws_bytes,
                _stream(A),
            )
        )
    return C


def w4a4_group_fp4_matmul(
    A: torch.Tensor, B: torch.Tensor, As: torch.Tensor, Bs: torch.Tensor, alpha: Optional[torch.Tensor] = None,
    output_dtype: torch.dtype = torch.bfloat16, bias: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """alpha * (A @ B.T) + bias of 4-bit operands: A [..., K / 2], B [N, K / 2] codes, As and Bs their scales in blocked order
    (`per_token_group_quant_fp4`, `fp4_blocked_scales`), both of groups of 16 or both of 32.  `alpha`: one float32 on the device,
    1 / (A's global scale * B's); None: 1.  K % 32 == 0, N % 8 == 0."""
    C = host.matmul_fp4(A, B, As, Bs, alpha, output_dtype, bias)
    if C is not None:
        return C
    if output_dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError("output dtype must be bfloat16 or float16")
    group = _fp4_scales_ok(A, As, "A")
    if _fp4_scales_ok(B, Bs, "B") != group:
        raise RuntimeError("A and B have different group sizes")
    if B.dim() != 2 or B.shape[1] != A.shape[-1] or B.device != A.device:
        raise RuntimeError("B must be [N, K / 2] with K matching A, on A's device")
    K, N = A.shape[-1] * 2, B.shape[0]
    M = A.numel() // A.shape[-1]
    C = torch.empty(A.shape[:-1] + (N,), device=A.device, dtype=output_dtype)
    a = _scalar_f32(alpha, A, "alpha")
    if bias is not None:
        bias = bias.to(output_dtype).contiguous()
        if not bias.is_cuda or bias.device != A.device or bias.numel() != N:
            raise RuntimeError(f"bias must be {N} values on A's device")
    with torch.cuda.device(A.device):
        check(lib.sglb200_group_fp4_scaled_mm(
            A.data_ptr(), B.data_ptr(), As.data_ptr(), Bs.data_ptr(), a, C.data_ptr(),
            bias.data_ptr() if bias is not None else None, M, N, K, group, 0 if output_dtype == torch.bfloat16 else 1,
            _stream(A)))
    return C


def lora_add(
    base: torch.Tensor, x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, adapter_ids: torch.Tensor,
    scalings: Optional[torch.Tensor] = None, ranks: Optional[torch.Tensor] = None, slices: Optional[Tuple[int, ...]] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Low-rank adapters of many requests beside a shared projection:

        out[t] = base[t] + scalings[l] * lora_b[l] (lora_a[l] x[t]),   l = adapter_ids[t]

    x [..., K], base [..., N] (the projection's output), both bf16 or both fp16, rows any distance apart; adapter_ids int32 [...], an
    id outside [0, L): out = base.  lora_a [L, S * R, K], lora_b [L, N, R] of the same type: of S merged projections (`slices`, their
    columns; None: one), the first takes rows 0 .. R - 1 of lora_a[l], and so on.  scalings float32 [L] (None: 1); ranks int32 [L]:
    only that many rows (of each R) and columns of an adapter count (None: R).  `out` may be `base`, and not overlap it otherwise;
    None: a new tensor.  Sums in float32, one rounding.  R % 8 == 0, at most 256; at most 1024 adapters and 8 slices; K % 8 == 0."""
    got = host.lora_add(base, x, lora_a, lora_b, adapter_ids, scalings, ranks, slices, out)
    if got is not None:
        return got
    xr, br = _rows_view(x, "x"), _rows_view(base, "base")
    for t, n in ((lora_a, "lora_a"), (lora_b, "lora_b"), (adapter_ids, "adapter_ids")):
        _cuda_contig(t, n)
    _same_device(x, base=base, lora_a=lora_a, lora_b=lora_b, adapter_ids=adapter_ids, scalings=scalings, ranks=ranks, out=out)
    dt = _dt(x)
    for t, n in ((base, "base"), (lora_a, "lora_a"), (lora_b, "lora_b")):
        if t.dtype != x.dtype:
            raise RuntimeError(f"lora_add: {n} is {t.dtype}, x is {x.dtype}")
    if base.shape[:-1] != x.shape[:-1]:
        raise RuntimeError(f"lora_add: base {tuple(base.shape)} and x {tuple(x.shape)} have different rows")
    T, K, N = xr.shape[0], x.shape[-1], base.shape[-1]
    if lora_a.dim() != 3 or lora_b.dim() != 3 or lora_a.shape[2] != K or lora_b.shape[:2] != (lora_a.shape[0], N):
        raise RuntimeError(f"lora_add: lora_a {tuple(lora_a.shape)} and lora_b {tuple(lora_b.shape)} do not fit K {K}, N {N}")
    L, _, R = lora_b.shape
    sizes = (N,) if slices is None else tuple(int(n) for n in slices)
    if L == 0 or R == 0 or not sizes or lora_a.shape[1] != len(sizes) * R or sum(sizes) != N or min(sizes) < 1:
        raise RuntimeError(f"lora_add: lora_a {tuple(lora_a.shape)} and slices {sizes} do not fit rank {R}, N {N}")
    if adapter_ids.dtype != torch.int32 or adapter_ids.numel() != T:
        raise RuntimeError(f"lora_add: adapter_ids must be {T} int32")
    for t, n, d in ((scalings, "scalings", torch.float32), (ranks, "ranks", torch.int32)):
        if t is not None and (not t.is_contiguous() or t.dtype != d or t.numel() != L):
            raise RuntimeError(f"lora_add: {n} must be {L} contiguous {d}")
    with torch.cuda.device(x.device):
        if out is None:
            out = torch.empty(base.shape, device=x.device, dtype=x.dtype)
        orows = _rows_view(out, "out")
        if out.dtype != x.dtype or out.shape != base.shape:
            raise RuntimeError(f"lora_add: out {tuple(out.shape)} {out.dtype} is not like base")
        if T == 0:
            return out
        bytes_ = lib.sglb200_lora_add_workspace_bytes(T, L, R, len(sizes))
        ws = torch.empty(bytes_, device=x.device, dtype=torch.uint8)
        check(lib.sglb200_lora_add(
            xr.data_ptr(), lora_a.data_ptr(), lora_b.data_ptr(), br.data_ptr(), orows.data_ptr(), dt, adapter_ids.data_ptr(),
            scalings.data_ptr() if scalings is not None else None, ranks.data_ptr() if ranks is not None else None, T, L, R, N, K,
            _row_stride(xr), _row_stride(br), _row_stride(orows), len(sizes), (ctypes.c_int64 * len(sizes))(*sizes), ws.data_ptr(),
            bytes_, _stream(x)))
    return out


def grouped_block_fp8_matmul(
    A: torch.Tensor, As: torch.Tensor, B: torch.Tensor, Bs: torch.Tensor, sorted_token_ids: torch.Tensor,
    expert_ids: torch.Tensor, num_rows: torch.Tensor, *, numel: int, scatter: bool,
    row_weights: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
    output_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """Grouped GEMM over expert-sorted rows (see sglb200_fp8_blockwise_grouped_mm)."""
    for t, n in ((A, "A"), (As, "As"), (B, "B"), (Bs, "Bs")):
        _cuda_contig(t, n)
    E, N, K = B.shape
    max_rows = A.shape[0]
    if out is None:
        out = torch.empty((numel if scatter else max_rows, N), device=A.device, dtype=output_dtype)
    if row_weights is not None:
        row_weights = row_weights.reshape(-1)
        if row_weights.dtype != torch.float32 or not row_weights.is_contiguous():
            raise RuntimeError("row_weights must be contiguous float32")
    check(
        lib.sglb200_fp8_blockwise_grouped_mm(
            A.data_ptr(), As.data_ptr(), B.data_ptr(), Bs.data_ptr(), out.data_ptr(), sorted_token_ids.data_ptr(),
            expert_ids.data_ptr(), num_rows.data_ptr(), row_weights.data_ptr() if row_weights is not None else None,
            max_rows, numel, E, N, K, 1 if scatter else 0, 0 if out.dtype == torch.bfloat16 else 1, _stream(A),
        )
    )
    return out


def fused_experts_fp4(
    hidden_states: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, w13_scale: torch.Tensor, w2_scale: torch.Tensor,
    topk_weights: torch.Tensor, topk_ids: torch.Tensor, w13_alpha: Optional[torch.Tensor] = None,
    w2_alpha: Optional[torch.Tensor] = None, routed_scaling_factor: float = 1.0,
) -> torch.Tensor:
    """The routed experts of a few tokens (at most 1024 tokens x experts a token), 4-bit weights and 16-bit activations:

        h   = silu(w13_alpha[e] * G_e x) * (w13_alpha[e] * U_e x)
        out = routed_scaling_factor * sum over a token's experts of topk_weights * w2_alpha[e] * W2_e h

    hidden_states [T, H] bf16 or fp16; w13 uint8 [E, 2I, H / 2] (G_e's rows, then U_e's), w2 uint8 [E, H, I / 2]; their scales
    float8_e4m3fn in rows' order, [E, 2I, H / 16] and [E, H, I / 16]; topk_weights and topk_ids [T, k].  An id outside
    [0, E) contributes nothing.  The alphas are float32 [E] (None: 1).  H and I divisible by 32, at most 69120."""
    if topk_ids.dtype == torch.int64:  # (an id that does not fit an int32 names no expert)
        topk_ids = topk_ids.clamp(-1, 2**31 - 1).to(torch.int32)
    elif topk_ids.dtype != torch.int32:
        raise RuntimeError("topk_ids must be int32 or int64")
    if topk_weights.dtype != torch.float32:
        topk_weights = topk_weights.float()
    out = host.fused_experts_fp4(hidden_states, w13, w2, w13_scale, w2_scale, topk_weights, topk_ids, w13_alpha, w2_alpha,
                                 routed_scaling_factor)
    if out is not None:
        return out
    x = hidden_states
    for t, n in ((x, "hidden_states"), (w13, "w13"), (w2, "w2"), (w13_scale, "w13_scale"), (w2_scale, "w2_scale"),
                 (topk_weights, "topk_weights"), (topk_ids, "topk_ids")):
        _cuda_contig(t, n)
        if t.device != x.device:
            raise RuntimeError(f"{n} is on another device than hidden_states")
    if x.dim() != 2 or w13.dim() != 3 or w2.dim() != 3 or w13.dtype != torch.uint8 or w2.dtype != torch.uint8:
        raise RuntimeError("fused_experts_fp4: hidden_states [T, H], w13 uint8 [E, 2I, H / 2], w2 uint8 [E, H, I / 2]")
    T, H = x.shape
    E, rows, _ = w13.shape
    I = rows // 2
    if rows % 2 or w13.shape[2] * 2 != H or tuple(w2.shape) != (E, H, I // 2) or I % 2:
        raise RuntimeError(f"fused_experts_fp4: w13 {tuple(w13.shape)} and w2 {tuple(w2.shape)} do not fit {H} columns")
    for w, s, n in ((w13, w13_scale, "w13_scale"), (w2, w2_scale, "w2_scale")):
        if s.dtype != torch.float8_e4m3fn or tuple(s.shape) != (E, w.shape[1], w.shape[2] // 8):
            raise RuntimeError(f"{n} must be float8_e4m3fn {(E, w.shape[1], w.shape[2] // 8)} in rows' order")
    if topk_ids.dim() != 2 or topk_ids.shape[0] != T or topk_weights.shape != topk_ids.shape:
        raise RuntimeError("fused_experts_fp4: topk_weights and topk_ids must be [T, k]")
    for a, n in ((w13_alpha, "w13_alpha"), (w2_alpha, "w2_alpha")):
        if a is not None and (not a.is_cuda or a.device != x.device or not a.is_contiguous() or a.dtype != torch.float32 or a.numel() != E):
            raise RuntimeError(f"{n} must be {E} contiguous float32 on the device of hidden_states")
    k = topk_ids.shape[1]
    out = torch.empty_like(x)
    if T == 0:
        return out
    if k == 0:
        return out.zero_()
    bytes_ = lib.sglb200_fused_experts_fp4_workspace_bytes(T, k, H, I)
    with torch.cuda.device(x.device):
        ws = torch.empty(bytes_, device=x.device, dtype=torch.uint8)
        check(lib.sglb200_fused_experts_fp4(
            x.data_ptr(), _dt(x), w13.data_ptr(), w13_scale.data_ptr(), w13_alpha.data_ptr() if w13_alpha is not None else None,
            w2.data_ptr(), w2_scale.data_ptr(), w2_alpha.data_ptr() if w2_alpha is not None else None, topk_weights.data_ptr(),
            topk_ids.data_ptr(), out.data_ptr(), T, k, E, H, I, float(routed_scaling_factor), ws.data_ptr(), bytes_, _stream(x)))
    return out


def gemm_status() -> int:
    """0, or 1 if a pipeline wait inside a GEMM kernel expired since the library was loaded (synchronises)."""
    return lib.sglb200_gemm_status()


def stream_status() -> int:
    """0, or 1 if a wait for a staged tile inside a streaming kernel (quantizer, masked silu_and_mul + quantizer)
    expired since the library was loaded (synchronises)."""
    return lib.sglb200_stream_status()
