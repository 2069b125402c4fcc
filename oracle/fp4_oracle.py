"""The 4-bit format and its operators in float64 (numpy): the definition that the fp4 kernels are tested against.

A value is an e2m1 code, two to a byte, the even column in the low half; a group of 16 columns shares an e4m3 scale beside one
float32 scale of the tensor, a group of 32 columns a power of two.  Every rounding is decided by comparing exact products (a
24-bit number times a 24-bit number fits a float64), never a rounded quotient.
"""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([m * 2.0**-9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1])
NAN_CODE = {16: 0x7F, 32: 0xFF}


def nearest(num, den, grid):
    """Index of the value of `grid` nearest to num / den (num >= 0, den > 0), ties to the even index, saturating."""
    code = np.zeros(np.broadcast(num, den).shape, dtype=np.int64)
    for c in range(len(grid) - 1):
        border = (grid[c] + grid[c + 1]) / 2 * den
        code += (num > border) | ((num == border) & (c % 2 == 1))
    return code


def group_scales(x, g, group):
    """x [rows, hidden] -> (scale codes uint8 [rows, groups], scale values, NaN where a group is not finite)."""
    a = np.abs(x.reshape(x.shape[0], -1, group).astype(np.float64))
    fine = np.isfinite(a).all(-1)
    amax = np.where(fine, np.where(np.isfinite(a), a, 0).max(-1), 0.0)
    if group == 32:
        e = np.where(amax > 0, np.frexp(amax)[1] - 3, -127)
        code = np.clip(e, -127, 127) + 127
        value = np.exp2(code - 127.0)
    else:
        mids = 6 * (E4M3[:-1] + E4M3[1:]) / 2  # amax * g against 6 * border
        num = amax * np.float64(g)
        low, high = np.searchsorted(mids, num, side="left"), np.searchsorted(mids, num, side="right")
        code = np.where(low == high, low, low + low % 2)
        value = E4M3[code]
    return np.where(fine, code, NAN_CODE[group]).astype(np.uint8), np.where(fine, value, np.nan)


def quantize(x, g, group):
    """x [rows, hidden] -> (codes uint8 [rows, hidden / 2], scale codes uint8 [rows, groups])."""
    x = np.asarray(x, dtype=np.float64)
    scode, s = group_scales(x, g, group)
    return pack(value_codes(x, s, g, group)), scode


def value_codes(x, s, g, group):
    v = x.reshape(x.shape[0], -1, group)
    live = (s > 0)[..., None]  # (not NaN, not zero)
    num = np.where(live, np.abs(v) * np.float64(1.0 if group == 32 else g), 0.0)
    code = nearest(num, np.where(live, s[..., None], 1.0), E2M1) + 8 * np.signbit(v)
    return np.where(live, code, 0).reshape(x.shape)


def pack(codes):
    return (codes[..., 0::2] + 16 * codes[..., 1::2]).astype(np.uint8)


def unpack(codes):
    """uint8 [.., k / 2] -> e2m1 codes [.., k]."""
    return np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1)


def scale_values(scode, group):
    if group == 32:
        return np.where(scode == 255, np.nan, np.exp2(scode.astype(np.float64) - 127))
    return np.where(scode == 0x7F, np.nan, E4M3[np.minimum(scode, 126)])


def dequantize(codes, scode, group):
    """codes [.., k / 2], scale codes [.., groups] -> code * s [.., k]."""
    c = unpack(codes)
    v = np.where(c >= 8, -E2M1[c % 8], E2M1[c % 8])
    return v * np.repeat(scale_values(scode, group), group, -1)


def blocked(scode, fill=0):
    """Scale codes [rows, groups] -> blocked order [whole blocks of 128 rows, whole blocks of 4 groups]."""
    rows, groups = scode.shape
    mb, gb = -(-rows // 128), -(-groups // 4)
    out = np.full(mb * gb * 512, fill, dtype=np.uint8)
    r, c = np.meshgrid(np.arange(rows), np.arange(groups), indexing="ij")
    out[((r // 128) * gb + c // 4) * 512 + r % 32 * 16 + r // 32 % 4 * 4 + c % 4] = scode
    return out.reshape(mb * 128, gb * 4)


def unblocked(b, rows, groups):
    """The scale codes [rows, groups] of a tensor in blocked order."""
    gb = b.shape[1] // 4
    r, c = np.meshgrid(np.arange(rows), np.arange(groups), indexing="ij")
    return b.reshape(-1)[((r // 128) * gb + c // 4) * 512 + r % 32 * 16 + r // 32 % 4 * 4 + c % 4]


def silu_and_mul(x):
    d = x.shape[-1] // 2
    gate, up = x[..., :d].astype(np.float64), x[..., d:].astype(np.float64)
    with np.errstate(over="ignore"):
        return gate / (1 + np.exp(-gate)) * up
