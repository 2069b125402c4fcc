// Quantizers to e2m1 codes with a scale per group of a row (fp4_math.cuh has the format), and the way back:
//
//   groups of 16:  s = e4m3(amax * g / 6),  code = e2m1(x * g / s),  value = code * s / g   (g: the tensor's float32 scale)
//   groups of 32:  s = 2^(floor(log2 amax) - 2),  code = e2m1(x / s),  value = code * s
//
// Every rounding is to nearest with ties to even and decided on exact numbers; a group whose scale is zero has zero codes, and one
// that holds a NaN or an infinity has the scale NaN, so that no product hides it.
//
// All of them are bound by HBM: 2 bytes an element in and 0.5625 out (bf16, groups of 16).  A thread takes 16 columns of one row,
// so a group of 16 needs no exchange and one of 32 a shuffle with the neighbour.
#include <algorithm>
#include <type_traits>

#include "fp4_math.cuh"
#include "ptx_sm100.cuh"

namespace sglb200 {
namespace fp4 {

constexpr int kThreads = 256;
constexpr int64_t kMaxUnits = 1ll << 31;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 16 consecutive elements as float32.
template <typename T>
__device__ __forceinline__ void load16(const T* src, float (&v)[16]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 q = ld_nc_16(src + 4 * j);
      v[4 * j] = __uint_as_float(q.x), v[4 * j + 1] = __uint_as_float(q.y);
      v[4 * j + 2] = __uint_as_float(q.z), v[4 * j + 3] = __uint_as_float(q.w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint4 q = ld_nc_16(src + 8 * j);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
          const float2 f = f16x2_to_f32(w[i]);
          v[8 * j + 2 * i] = f.x, v[8 * j + 2 * i + 1] = f.y;
        } else {
          v[8 * j + 2 * i] = __uint_as_float(w[i] << 16), v[8 * j + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
    }
  }
}

// Quantises this thread's 16 values and stores codes and scale.  All lanes of the warp take part where the group is 32.
template <int kGroup>
__device__ __forceinline__ void quantize16(const float (&v)[16], float g, uint2* codes, uint8_t* scales, int64_t row, int unit,
                                           int units, int group_blocks, bool live) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) amax = max_nan(amax, fabsf(v[i]));
  const float(&x0)[8] = *reinterpret_cast<const float(*)[8]>(&v[0]);
  const float(&x1)[8] = *reinterpret_cast<const float(*)[8]>(&v[8]);
  uint2 out = make_uint2(0u, 0u);
  uint32_t code;
  if constexpr (kGroup == 32) {
    amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    const bool fine = amax < __int_as_float(0x7f800000);
    const int e = max((int)(__float_as_uint(amax) >> 23) - 2, 0);
    code = fine ? (uint32_t)e : kNanE8m0;
    const float r = __uint_as_float((uint32_t)(254 - e) << 23);
    if (fine) {
      float a[8], b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = x0[i] * r, b[i] = x1[i] * r;
      out = make_uint2(cvt_e2m1x8(a), cvt_e2m1x8(b));
    }
  } else {
    const bool fine = amax < __int_as_float(0x7f800000);
    code = fine ? group_scale_e4m3(amax, g) : kNanE4m3;
    if (fine && code != 0) {
      const float s = f16x2_to_f32(cvt_f16x2_e4m3x2(code)).x;
      const float r = g * __frcp_rn(s), r_lo = r * (1.0f - 0x1p-20f), r_hi = r * (1.0f + 0x1p-20f);
      out = make_uint2(codes_x8(x0, r_lo, r_hi, s, g), codes_x8(x1, r_lo, r_hi, s, g));
    }
  }
  if (!live) return;
  *codes = out;
  constexpr int kPer = kGroup / kUnit;
  if (unit % kPer == 0) {
    const int group = unit / kPer;
    uint8_t* at = scales + scale_at(row, group, group_blocks);
    *at = (uint8_t)code;
    if (unit + kPer == units)  // the block's columns past the last group
      for (int c = group + 1; c < 4 * group_blocks; ++c) at[c - group] = 0;
  }
}

template <typename T, int kGroup, bool kSilu>
__global__ void __launch_bounds__(kThreads)
    quant_fp4_kernel(const T* __restrict__ x, uint2* __restrict__ codes, uint8_t* __restrict__ scales,
                     const float* __restrict__ global_scale, uint32_t total, FastDiv units, int64_t first_row, int group_blocks) {
  ptx::grid_dependency_wait();
  const uint32_t n = blockIdx.x * kThreads + threadIdx.x;
  const bool live = n < total;
  const uint32_t at = live ? n : total - 1;  // (total is even where a group takes two threads)
  const uint32_t row = units.quot(at), unit = at - row * units.d;
  const float g = global_scale ? *global_scale : 1.0f;
  float v[16];
  if constexpr (kSilu) {
    const T* src = x + (int64_t)row * units.d * (2 * kUnit) + unit * kUnit;
    float up[16];
    load16(src, v);
    load16(src + (int64_t)units.d * kUnit, up);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = v[i] / (1.0f + expf(-v[i])) * up[i];
  } else {
    load16(x + (int64_t)at * kUnit, v);
  }
  quantize16<kGroup>(v, g, codes + at, scales, first_row + row, (int)unit, (int)units.d, group_blocks, live);
}

template <typename T, int kGroup>
__global__ void __launch_bounds__(kThreads)
    dequant_fp4_kernel(const uint2* __restrict__ codes, const uint8_t* __restrict__ scales, const float* __restrict__ global_scale,
                       T* __restrict__ out, uint32_t total, FastDiv units, int64_t first_row, int group_blocks) {
  ptx::grid_dependency_wait();
  const uint32_t n = blockIdx.x * kThreads + threadIdx.x;
  if (n >= total) return;
  const uint32_t row = units.quot(n), unit = n - row * units.d;
  const uint2 c = __ldg(codes + n);
  const uint32_t code = __ldg(scales + scale_at(first_row + row, (int)unit / (kGroup / kUnit), group_blocks));
  float s = kGroup == 32 ? e8m0_to_f32(code) : f16x2_to_f32(cvt_f16x2_e4m3x2(code)).x;
  if (global_scale) s = s / *global_scale;
  uint32_t h[8];
  cvt_f16x2_e2m1x8(c.x, *reinterpret_cast<uint32_t(*)[4]>(&h[0]));
  cvt_f16x2_e2m1x8(c.y, *reinterpret_cast<uint32_t(*)[4]>(&h[4]));
  T* dst = out + (int64_t)n * kUnit;
  float v[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = f16x2_to_f32(h[i]);
    v[2 * i] = f.x * s, v[2 * i + 1] = f.y * s;
  }
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      reinterpret_cast<float4*>(dst)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  } else {
    union {
      T t[16];
      uint4 q[2];
    } o;
#pragma unroll
    for (int i = 0; i < 16; ++i) o.t[i] = ElemTraits<T>::from_f32(v[i]);
    reinterpret_cast<uint4*>(dst)[0] = o.q[0];
    reinterpret_cast<uint4*>(dst)[1] = o.q[1];
  }
}

// Rows per launch: their units are counted in 31 bits, and a launch starts at a block of 128 rows.
static int64_t rows_per_launch(int64_t units) { return std::max<int64_t>(128, kMaxUnits / 2 / units / 128 * 128); }

template <typename T, int kGroup, bool kSilu>
static int launch_quant(const void* x, void* codes, void* scales, const float* g, int64_t rows, int64_t hidden, cudaStream_t st) {
  const int64_t units = hidden / kUnit, step = rows_per_launch(units);
  const int group_blocks = (int)((hidden / kGroup + 3) / 4);
  for (int64_t r = 0; r < rows; r += step) {
    const int64_t total = std::min(step, rows - r) * units;
    SGLB_CUDA(launch_pdl(quant_fp4_kernel<T, kGroup, kSilu>, (unsigned)((total + kThreads - 1) / kThreads), kThreads, 0, st,
                         static_cast<const T*>(x) + r * hidden * (kSilu ? 2 : 1), static_cast<uint2*>(codes) + r * units,
                         static_cast<uint8_t*>(scales), g, (uint32_t)total, FastDiv((uint32_t)units), r, group_blocks));
  }
  return SGLB200_OK;
}

template <typename T, int kGroup>
static int launch_dequant(const void* codes, const void* scales, const float* g, void* out, int64_t rows, int64_t hidden,
                          cudaStream_t st) {
  const int64_t units = hidden / kUnit, step = rows_per_launch(units);
  const int group_blocks = (int)((hidden / kGroup + 3) / 4);
  for (int64_t r = 0; r < rows; r += step) {
    const int64_t total = std::min(step, rows - r) * units;
    SGLB_CUDA(launch_pdl(dequant_fp4_kernel<T, kGroup>, (unsigned)((total + kThreads - 1) / kThreads), kThreads, 0, st,
                         static_cast<const uint2*>(codes) + r * units, static_cast<const uint8_t*>(scales), g,
                         static_cast<T*>(out) + r * hidden, (uint32_t)total, FastDiv((uint32_t)units), r, group_blocks));
  }
  return SGLB200_OK;
}

// What the three entry points refuse alike.
static int check_shape(const char* what, int64_t rows, int64_t hidden, int group, const float* g) {
  if (group != 16 && group != 32) return fail(SGLB200_E_UNSUPPORTED, "%s: group_size %d is neither 16 nor 32", what, group);
  SGLB_REQUIRE(rows >= 0 && hidden > 0, "%s: %lld rows of %lld columns", what, (long long)rows, (long long)hidden);
  SGLB_REQUIRE(hidden % group == 0, "%s: hidden size %lld is not divisible by group_size %d", what, (long long)hidden, group);
  SGLB_REQUIRE(hidden <= 1 << 20, "%s: hidden size %lld exceeds 2^20", what, (long long)hidden);
  SGLB_REQUIRE(group == 16 || g == nullptr, "%s: groups of 32 have power-of-two scales and take no global scale", what);
  SGLB_REQUIRE(((uintptr_t)g & 3) == 0, "%s: the global scale is not aligned to 4 bytes", what);
  return SGLB200_OK;
}

}  // namespace fp4
}  // namespace sglb200

using namespace sglb200;

extern "C" {

int sglb200_per_token_group_quant_fp4(const void* input, int in_dtype, void* output_q, void* output_s, const float* global_scale,
                                      int64_t num_tokens, int64_t hidden, int group_size, void* stream) {
  const int rc = fp4::check_shape("per_token_group_quant_fp4", num_tokens, hidden, group_size, global_scale);
  if (rc) return rc;
  if (in_dtype < 0 || in_dtype > 2) return fail(SGLB200_E_UNSUPPORTED, "per_token_group_quant_fp4: unsupported input dtype %d", in_dtype);
  if (num_tokens == 0) return SGLB200_OK;
  SGLB_REQUIRE(input && output_q && output_s, "per_token_group_quant_fp4: null pointer");
  SGLB_REQUIRE(aligned16(input) && aligned16(output_q) && aligned16(output_s), "per_token_group_quant_fp4: pointers must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define GO(T, G) return fp4::launch_quant<T, G, false>(input, output_q, output_s, global_scale, num_tokens, hidden, st)
  if (group_size == 16) {
    if (in_dtype == 0) GO(__nv_bfloat16, 16);
    if (in_dtype == 1) GO(__half, 16);
    GO(float, 16);
  }
  if (in_dtype == 0) GO(__nv_bfloat16, 32);
  if (in_dtype == 1) GO(__half, 32);
  GO(float, 32);
#undef GO
}

int sglb200_silu_and_mul_quant_fp4(const void* input, int dtype, void* output_q, void* output_s, const float* global_scale,
                                   int64_t rows, int64_t d, int group_size, void* stream) {
  const int rc = fp4::check_shape("silu_and_mul_quant_fp4", rows, d, group_size, global_scale);
  if (rc) return rc;
  if (dtype != 0 && dtype != 1) return fail(SGLB200_E_UNSUPPORTED, "silu_and_mul_quant_fp4: unsupported input dtype %d", dtype);
  if (rows == 0) return SGLB200_OK;
  SGLB_REQUIRE(input && output_q && output_s, "silu_and_mul_quant_fp4: null pointer");
  SGLB_REQUIRE(aligned16(input) && aligned16(output_q) && aligned16(output_s), "silu_and_mul_quant_fp4: pointers must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define GO(T, G) return fp4::launch_quant<T, G, true>(input, output_q, output_s, global_scale, rows, d, st)
  if (group_size == 16) {
    if (dtype == 0) GO(__nv_bfloat16, 16);
    GO(__half, 16);
  }
  if (dtype == 0) GO(__nv_bfloat16, 32);
  GO(__half, 32);
#undef GO
}

int sglb200_per_token_group_dequant_fp4(const void* input_q, const void* input_s, const float* global_scale, void* output,
                                        int out_dtype, int64_t num_tokens, int64_t hidden, int group_size, void* stream) {
  const int rc = fp4::check_shape("per_token_group_dequant_fp4", num_tokens, hidden, group_size, global_scale);
  if (rc) return rc;
  if (out_dtype < 0 || out_dtype > 2) return fail(SGLB200_E_UNSUPPORTED, "per_token_group_dequant_fp4: unsupported output dtype %d", out_dtype);
  if (num_tokens == 0) return SGLB200_OK;
  SGLB_REQUIRE(input_q && input_s && output, "per_token_group_dequant_fp4: null pointer");
  SGLB_REQUIRE(aligned16(input_q) && aligned16(input_s) && aligned16(output), "per_token_group_dequant_fp4: pointers must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define GO(T, G) return fp4::launch_dequant<T, G>(input_q, input_s, global_scale, output, num_tokens, hidden, st)
  if (group_size == 16) {
    if (out_dtype == 0) GO(__nv_bfloat16, 16);
    if (out_dtype == 1) GO(__half, 16);
    GO(float, 16);
  }
  if (out_dtype == 0) GO(__nv_bfloat16, 32);
  if (out_dtype == 1) GO(__half, 32);
  GO(float, 32);
#undef GO
}

}  // extern "C"
