// The 4-bit format and its conversions, shared by the fp4 kernels.
//
// A value is an e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, the even column in the low half.  A
// group of a row's columns shares a scale: 16 columns an e4m3 one (beside one float32 scale of the whole tensor), or 32 columns a
// power of two (e8m0).  Scales of the products' operands lie in blocked order, the order in which tensor memory takes them: blocks
// of 128 rows x 4 groups, 512 bytes each, a block's rows r, r + 32, r + 64 and r + 96 side by side.
#pragma once
#include "common.cuh"

namespace sglb200 {
namespace fp4 {

constexpr int kUnit = 16;         // columns that a thread of the elementwise kernels takes
constexpr int kBlockBytes = 512;  // 128 rows x 4 groups of scales
constexpr uint32_t kNanE4m3 = 0x7f, kNanE8m0 = 0xff;

// Where the scale of (row, group) lies, with `group_blocks` blocks in a row.
__host__ __device__ __forceinline__ int64_t scale_at(int64_t row, int group, int group_blocks) {
  return ((row >> 7) * group_blocks + (group >> 2)) * kBlockBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (group & 3);
}

// n / d for n < 2^31 by a multiplication (d >= 1): the reciprocal rounded up, with one bit more than a word (Granlund and Montgomery, 1994).
struct FastDiv {
  uint32_t d, mul, shift;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div), mul(0), shift(0) {
    while ((1ull << shift) < div) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - div)) / div + 1);
  }
  __device__ __forceinline__ uint32_t quot(uint32_t n) const { return (__umulhi(mul, n) + n) >> shift; }
};

// (lo, hi) -> two codes, lo in bits 0-3; to nearest, ties to even, saturating.
__device__ __forceinline__ uint32_t cvt_e2m1x2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 b;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\n\t"
      "cvt.u32.u8 %0, b;\n\t}"
      : "=r"(r)
      : "f"(lo), "f"(hi));
  return r;
}

// Eight float32 -> eight codes.
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Eight codes -> four pairs of fp16 (exact), even columns in the low halves.
__device__ __forceinline__ void cvt_f16x2_e2m1x8(uint32_t codes, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
}

// Two e4m3 codes (bits 0-7, 8-15) -> a pair of fp16 (exact; NaN stays NaN).
__device__ __forceinline__ uint32_t cvt_f16x2_e4m3x2(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 t;\n\t"
      "cvt.u16.u32 t, %1;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, t;\n\t}"
      : "=r"(r)
      : "r"(two));
  return r;
}
__device__ __forceinline__ float2 f16x2_to_f32(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

// e8m0 code -> float32 (255 is NaN).
__device__ __forceinline__ float e8m0_to_f32(uint32_t code) {
  return __uint_as_float(code == kNanE8m0 ? 0x7fc00000u : code == 0 ? 0x00400000u : code << 23);
}

// The smallest e2m1 magnitude above each border between two neighbours is decided by the border itself: twice the border
// between codes c and c + 1 (a multiple of 1/2 that float32 holds exactly), c in 0..6.
__device__ __forceinline__ float e2m1_border(uint32_t c) {
  const uint32_t quarters = c < 4 ? 2 * c + 1 : c == 4 ? 10 : c == 5 ? 14 : 20;  // 0.25 0.75 1.25 1.75 2.5 3.5 5
  return 0.25f * (float)quarters;
}

// The scale of a group of 16: the e4m3 value nearest to amax * g / 6 (ties to even, saturating), decided on the exact product.
// float32 alone would round amax * g / 6 onto a border it is only near to, which happens whenever g is a short number: the
// quotient is therefore taken a little too small and a little too large, and where that matters the sign of the exact
// amax * g - 6 * border, one fused multiply-add, decides.
__device__ __forceinline__ uint32_t group_scale_e4m3(float amax, float g) {
  const float v = amax * g * 0.16666667f;
  const uint32_t two = cvt_e4m3x2(v * (1.0f - 0x1p-20f), v * (1.0f + 0x1p-20f));
  uint32_t lo = two & 0xff;
  const uint32_t hi = two >> 8;
  if (lo != hi) {
    const float2 f = f16x2_to_f32(cvt_f16x2_e4m3x2(two));
    const float over = fmaf(amax, g, -3.0f * (f.x + f.y));
    if (over > 0.f || (over == 0.f && (lo & 1))) lo = hi;
  }
  return lo;
}

// silu(gate) * up in float32.  Below kSiluTail 1 + e^-gate and its reciprocal come to the ends of float32's range, while silu = gate e^gate,
// times a large `up`, need not be small: e^(gate / 2) is taken twice there, with `up` in between.
constexpr float kSiluTail = -87.0f;
__device__ __forceinline__ float silu_mul(float gate, float up) {
  if (gate < kSiluTail) {
    const float e = expf(0.5f * gate);
    return gate * e * up * e;
  }
  return gate / (1.f + expf(-gate)) * up;
}
// (a, b) times r, both products in one instruction.
__device__ __forceinline__ void mul2(float& a, float& b, float x, float y, float r) {
  asm("{\n\t.reg .b64 v, f, q;\n\t"
      "mov.b64 v, {%2, %3};\n\t"
      "mov.b64 f, {%4, %4};\n\t"
      "mul.rn.f32x2 q, v, f;\n\t"
      "mov.b64 {%0, %1}, q;\n\t}"
      : "=f"(a), "=f"(b)
      : "f"(x), "f"(y), "f"(r));
}

// x[i] of eight registers.
__device__ __forceinline__ float pick(const float (&x)[8], uint32_t i) {
  const bool b0 = i & 1, b1 = i & 2, b2 = i & 4;
  const float a = b0 ? x[1] : x[0], b = b0 ? x[3] : x[2], c = b0 ? x[5] : x[4], d = b0 ? x[7] : x[6];
  const float e = b1 ? b : a, f = b1 ? d : c;
  return b2 ? f : e;
}

// Codes of eight values x under a factor a little too small and one a little too large; `differ`: where the two are not the same.
__device__ __forceinline__ uint32_t codes_between(const float (&x)[8], float r_lo, float r_hi, uint32_t& differ) {
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) mul2(a[i], a[i + 1], x[i], x[i + 1], r_lo), mul2(b[i], b[i + 1], x[i], x[i + 1], r_hi);
  const uint32_t lo = cvt_e2m1x8(a);
  differ = lo ^ cvt_e2m1x8(b);
  return lo;
}

// Codes of eight values x under scale s (not 0) and the tensor's scale g: e2m1 nearest to x * g / s, decided likewise.
// `r_lo`, `r_hi`: g / s a little too small and too large.  Where the two codes of a value differ the exact product decides, one value
// after the other: g of few bits, or quotients of such as calibration gives, puts some value of a warp next to a border more often
// than not, though seldom two of a thread (all eight unrolled: 8192 x 18432 in 117 us).
__device__ __forceinline__ uint32_t codes_x8(const float (&x)[8], float r_lo, float r_hi, float s, float g) {
  uint32_t differ, lo = codes_between(x, r_lo, r_hi, differ);
  while (differ != 0) {
    const uint32_t at = (__ffs(differ) - 1) & ~3u, c = lo >> at & 7;
    const float over = fmaf(fabsf(pick(x, at >> 2)), g, -e2m1_border(c) * s);
    if (over > 0.f || (over == 0.f && (c & 1))) lo += 1u << at;
    differ &= ~(15u << at);
  }
  return lo;
}

}  // namespace fp4
}  // namespace sglb200
