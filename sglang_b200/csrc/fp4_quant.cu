// Quantizers to e2m1 codes with a scale per group of a row (fp4_math.cuh has the format), and the way back:
//
//   groups of 16:  s = e4m3(amax * g / 6),  code = e2m1(x * g / s),  value = code * s / g   (g: the tensor's float32 scale)
//   groups of 32:  s = 2^(floor(log2 amax) - 2),  code = e2m1(x / s),  value = code * s
//
// Every rounding is to nearest with ties to even and decided on exact numbers; a group whose scale is zero has zero codes, and one
// that holds a NaN or an infinity has the scale NaN, so that no product hides it.  silu(gate) * up is taken in float32, and once more in
// float64 where a rounding of it could matter.
//
// All of them are bound by HBM: 2 bytes an element in and 0.5625 out (bf16, groups of 16).  A thread takes 16 columns of a row, so a
// group of 16 needs no exchange and one of 32 a shuffle with the neighbour.  A warp takes the 64 columns of a scale block in the
// eight rows whose scales fill one 32-byte sector of it (rows r, r + 1 and those 32, 64 and 96 further), so that every sector it
// touches, of values, codes and scales, is whole; with 32 columns a group it is 128 columns of four rows.
#include <algorithm>
#include <type_traits>

#include "fp4_math.cuh"
#include "ptx_sm100.cuh"

namespace sglb200 {
namespace fp4 {

constexpr int kThreads = 256;
constexpr int64_t kMostScales = 1ll << 30;  // of a launch, in bytes (a block of 512 is at most 32 tasks)

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 32 bytes at once.
__device__ __forceinline__ void ld_32(const void* p, uint32_t (&v)[8]) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p));
}
__device__ __forceinline__ void st_32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// 16 elements as they lie in memory.  kWide: they begin on 32 bytes.
template <typename T>
struct Raw {
  uint32_t w[sizeof(T) * 4];
  template <bool kWide>
  __device__ __forceinline__ void load(const T* src) {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) {
      uint32_t v[8];
      if constexpr (kWide) {
        ld_32(reinterpret_cast<const uint8_t*>(src) + 32 * j, v);
      } else {
        const uint4 a = ld_nc_16(reinterpret_cast<const uint8_t*>(src) + 32 * j), b = ld_nc_16(reinterpret_cast<const uint8_t*>(src) + 32 * j + 16);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) w[8 * j + i] = v[i];
    }
  }
  __device__ __forceinline__ void to_f32(float (&v)[16]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[2 * i] = __uint_as_float(w[2 * i]), v[2 * i + 1] = __uint_as_float(w[2 * i + 1]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = f16x2_to_f32(w[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
};

// Where a lane works: 16 columns of a row.  A warp's task is a block of scales (64 or 128 columns) in the rows of its block of 128
// whose scales are neighbours.
template <int kGroup>
struct Place {
  static constexpr int kUnits = 4 * kGroup / kUnit;  // of a block in a row
  static constexpr int kRows = 32 / kUnits;          // of a task: 8 or 4
  static constexpr int kTasks = 128 / kRows;         // of a block of 128 rows and a block of scales
  int64_t unit;                                      // of the tensor; the first one where this lane has none
  uint32_t scale;                                    // where its scale lies, from the first of this launch
  uint32_t column;                                   // of the row, in units
  bool row_live, live;                               // whether there is such a row, and such columns in it
  Place() = default;
  // `rows`: of this launch.
  __device__ __forceinline__ Place(uint32_t task, const FastDiv& blocks, uint32_t units, int rows, uint32_t lane = threadIdx.x & 31) {
    const uint32_t u = lane % kUnits, r = lane / kUnits;
    const uint32_t set = blocks.quot(task), block = task - set * blocks.d;  // set: (block of rows, rows of it)
    const uint32_t low = set % kTasks * (kRows / 4) + r / 4, quarter = r % 4, row = set / kTasks * 128 + quarter * 32 + low;
    column = block * kUnits + u;
    row_live = (int)row < rows, live = row_live && column < units;
    unit = live ? (int64_t)((uint64_t)row * units + column) : 0;
    scale = (set / kTasks * blocks.d + block) * kBlockBytes + low * 16 + quarter * 4 + u / (kGroup / kUnit);
  }
};

// Quantises this thread's 16 values; the code of the scale.  The lanes of a warp whose group takes two of them go together.
// kInexact: the values are rounded, off by at most 2^-21, and a rounded number cannot tell on which side of a border that it is next to
// the exact one lies.  `near`: the scale or a code is so near, and whoever has the exact values has to decide.
template <int kGroup, bool kInexact>
__device__ __forceinline__ uint32_t quantize16(const float (&v)[16], float g, uint2& out, bool& near) {
  constexpr float kLess = 1.0f - 0x1p-19f, kMore = 1.0f + 0x1p-19f;  // (where kInexact: what the values, g and its quotient are off by, twice)
  float amax = max_nan(fabsf(v[0]), fabsf(v[1]));
#pragma unroll
  for (int i = 2; i < 16; i += 2) amax = max3_nan(amax, fabsf(v[i]), fabsf(v[i + 1]));
  const float(&x0)[8] = *reinterpret_cast<const float(*)[8]>(&v[0]);
  const float(&x1)[8] = *reinterpret_cast<const float(*)[8]>(&v[8]);
  out = make_uint2(0u, 0u);
  uint32_t code;
  if constexpr (kGroup == 32) {
    amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    const bool fine = amax < __int_as_float(0x7f800000);
    const int e = max((int)(__float_as_uint(amax) >> 23) - 2, 0);
    code = fine ? (uint32_t)e : kNanE8m0;
    const float r = __uint_as_float((uint32_t)(254 - e) << 23);
    if constexpr (kInexact) {
      if (fine) {
        uint32_t differ[2];
        out.x = codes_between(x0, r * kLess, r * kMore, differ[0]), out.y = codes_between(x1, r * kLess, r * kMore, differ[1]);
        near = (__float_as_uint(amax * kLess) ^ __float_as_uint(amax * kMore)) >> 23 != 0 || (differ[0] | differ[1]) != 0;
      }
    } else if (fine) {
      float a[8], b[8];
#pragma unroll
      for (int i = 0; i < 8; i += 2) mul2(a[i], a[i + 1], x0[i], x0[i + 1], r), mul2(b[i], b[i + 1], x1[i], x1[i + 1], r);
      out = make_uint2(cvt_e2m1x8(a), cvt_e2m1x8(b));
    }
  } else {
    const bool fine = amax < __int_as_float(0x7f800000);
    if constexpr (kInexact) {
      const float scaled = amax * g * 0.16666667f;
      const uint32_t two = cvt_e4m3x2(scaled * kLess, scaled * kMore);
      code = fine ? two & 0xff : kNanE4m3;
      near = fine && (two & 0xff) != two >> 8;
      if (fine && code != 0) {
        const float r = g * __frcp_rn(f16x2_to_f32(cvt_f16x2_e4m3x2(code)).x);
        uint32_t differ[2];
        out.x = codes_between(x0, r * kLess, r * kMore, differ[0]), out.y = codes_between(x1, r * kLess, r * kMore, differ[1]);
        near = near || (differ[0] | differ[1]) != 0;
      }
      return code;
    }
    code = fine ? group_scale_e4m3(amax, g) : kNanE4m3;
    if (fine && code != 0) {
      const float s = f16x2_to_f32(cvt_f16x2_e4m3x2(code)).x;
      const float r = g * __frcp_rn(s), r_lo = r * (1.0f - 0x1p-20f), r_hi = r * (1.0f + 0x1p-20f);
      out = make_uint2(codes_x8(x0, r_lo, r_hi, s, g), codes_x8(x1, r_lo, r_hi, s, g));
    }
  }
  return code;
}

// Quantises a group of silu(gate) * up once more in float64, where float32 does not do: next to a border (a few in 10^5 groups) and
// below kSiluTail.  A warp, one value a lane (by one thread, a value after the other, it took 10 us).  `gate`, `up`: the group's first values;
// `codes`: where its codes go.
template <typename T, int kGroup>
__device__ __noinline__ void quantize_silu_f64(const T* gate, const T* up, float g, uint32_t* codes, uint8_t* scale) {
  const int lane = threadIdx.x & 31, i = lane % kGroup;
  const double x = (double)ElemTraits<T>::to_f32(gate[i]), h = x / (1.0 + exp(-x)) * (double)ElemTraits<T>::to_f32(up[i]);
  const bool fine = __all_sync(0xffffffffu, fabsf((float)h) < __int_as_float(0x7f800000));
  double amax = fabs(h);
#pragma unroll
  for (int o = kGroup / 2; o > 0; o >>= 1) amax = fmax(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  constexpr float kLess = 1.0f - 0x1p-20f, kMore = 1.0f + 0x1p-20f;
  const double factor = kGroup == 32 ? 1.0 : (double)g;
  uint32_t code;
  double s;
  if constexpr (kGroup == 32) {
    const int e = amax > 0.0 ? max(ilogb(amax) - 2, -127) : -127;
    code = (uint32_t)(e + 127), s = ldexp(1.0, e);
  } else {
    const float v = (float)(amax * factor / 6.0);
    const uint32_t two = cvt_e4m3x2(v * kLess, v * kMore);
    const float2 f = f16x2_to_f32(cvt_f16x2_e4m3x2(two));
    const double border = 3.0 * ((double)f.x + (double)f.y), num = amax * factor;
    const bool higher = (two & 0xff) != two >> 8 && (num > border || (num == border && (two & 1)));
    code = higher ? two >> 8 : two & 0xff, s = higher ? f.y : f.x;
  }
  if (!fine) code = kGroup == 32 ? kNanE8m0 : kNanE4m3;
  uint32_t word = 0;
  if (fine && s > 0.0) {
    const double num = fabs(h) * factor;
    const float q = (float)fmin(num / s, 8.0);
    const uint32_t two = cvt_e2m1x2(q * kLess, q * kMore), c = two & 15;
    const double border = (double)e2m1_border(c) * s;
    const bool higher = c != two >> 4 && (num > border || (num == border && (c & 1)));
    word = (c + (higher ? 1u : 0u) | (signbit(h) ? 8u : 0u)) << 4 * (i & 7);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
  if (lane < kGroup && lane % 8 == 0) codes[lane / 8] = word;
  if (lane == 0) *scale = (uint8_t)code;
}

// A warp takes kAhead tasks, whose values are all asked for before the first is quantised.
template <typename T, int kGroup, bool kSilu, bool kWide, int kAhead>
__global__ void __launch_bounds__(kThreads)
    quant_fp4_kernel(const T* __restrict__ x, uint2* __restrict__ codes, uint8_t* __restrict__ scales,
                     const float* __restrict__ global_scale, uint32_t tasks, FastDiv blocks, uint32_t units, int rows) {
  ptx::grid_dependency_wait();
  const uint32_t task0 = blockIdx.x * (kThreads / 32 * kAhead) + threadIdx.x / 32;
  if (task0 >= tasks) return;
  Place<kGroup> at[kAhead];
  Raw<T> raw[kAhead][kSilu ? 2 : 1];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    at[k] = Place<kGroup>(min(task0 + k * (kThreads / 32), tasks - 1), blocks, units, rows);  // (the last one again rather than none)
    const T* src = x + at[k].unit * kUnit;
    if constexpr (kSilu) src += at[k].live ? (at[k].unit - at[k].column) * kUnit : 0;  // (rows of twice the columns)
    raw[k][0].template load<kWide>(src);
    if constexpr (kSilu) raw[k][1].template load<kWide>(src + (int64_t)units * kUnit);
  }
  const float g = global_scale ? __ldcg(global_scale) : 1.0f;
  uint32_t again = 0;  // tasks that float32 does not do for
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    if (task0 + k * (kThreads / 32) >= tasks) break;
    float v[16];
    raw[k][0].to_f32(v);
    if constexpr (kSilu) {
      float up[16];
      raw[k][1].to_f32(up);
      float least = fminf(v[0], v[1]);
#pragma unroll
      for (int i = 2; i < 16; ++i) least = fminf(least, v[i]);
      if (least < kSiluTail) again |= 1u << k;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        // The quotient by a reciprocal and one correction (Markstein's): half a unit in the last place, and the instructions of a division
        // are half of the kernel's.  Not below kSiluTail.
        const float d = 1.0f + expf(-v[i]);
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
        const float q = v[i] * r;
        v[i] = fmaf(fmaf(-q, d, v[i]), r, q) * up[i];
      }
    }
    uint2 c;
    bool near = false;
    const uint32_t code = quantize16<kGroup, kSilu>(v, g, c, near);
    if (near) again |= 1u << k;
    if (at[k].live) codes[at[k].unit] = c;
    // (zeros for groups past the last)
    if (at[k].row_live && at[k].column % (kGroup / kUnit) == 0) scales[at[k].scale] = at[k].live ? (uint8_t)code : 0;
  }
  if constexpr (kSilu) {
    if (__ballot_sync(0xffffffffu, again != 0) == 0) return;
    __syncwarp();  // (what one lane has stored another may store again)
#pragma unroll 1
    for (int k = 0; k < kAhead; ++k) {
      uint32_t left = __ballot_sync(0xffffffffu, again >> k & 1);
      if constexpr (kGroup == 32) left = (left | left >> 1) & 0x55555555u;  // (a group's first lane)
      for (; left != 0; left &= left - 1) {
        const Place<kGroup> place(min(task0 + k * (kThreads / 32), tasks - 1), blocks, units, rows, __ffs(left) - 1);
        if (!place.live) continue;
        const T* gate = x + (2 * place.unit - place.column) * kUnit;  // (rows of twice the columns)
        quantize_silu_f64<T, kGroup>(gate, gate + (int64_t)units * kUnit, g, reinterpret_cast<uint32_t*>(codes + place.unit), scales + place.scale);
      }
    }
  }
}

template <typename T, int kGroup, bool kWide, int kAhead>
__global__ void __launch_bounds__(kThreads)
    dequant_fp4_kernel(const uint2* __restrict__ codes, const uint8_t* __restrict__ scales, const float* __restrict__ global_scale,
                       T* __restrict__ out, uint32_t tasks, FastDiv blocks, uint32_t units, int rows) {
  ptx::grid_dependency_wait();
  const uint32_t task0 = blockIdx.x * (kThreads / 32 * kAhead) + threadIdx.x / 32;
  if (task0 >= tasks) return;
  Place<kGroup> at[kAhead];
  uint2 c[kAhead];
  uint32_t code[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    at[k] = Place<kGroup>(min(task0 + k * (kThreads / 32), tasks - 1), blocks, units, rows);
    c[k] = __ldg(codes + at[k].unit);
    code[k] = at[k].live ? __ldg(scales + at[k].scale) : 0u;
  }
  const float g = global_scale ? __ldcg(global_scale) : 1.0f;
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    if (task0 + k * (kThreads / 32) >= tasks) break;
    if (!at[k].live) continue;
    float s = kGroup == 32 ? e8m0_to_f32(code[k]) : f16x2_to_f32(cvt_f16x2_e4m3x2(code[k])).x;
    if (global_scale) s = s / g;
    uint32_t h[8];
    cvt_f16x2_e2m1x8(c[k].x, *reinterpret_cast<uint32_t(*)[4]>(&h[0]));
    cvt_f16x2_e2m1x8(c[k].y, *reinterpret_cast<uint32_t(*)[4]>(&h[4]));
    T* dst = out + at[k].unit * kUnit;
    uint32_t o[sizeof(T) * 4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = f16x2_to_f32(h[i]);
      if constexpr (sizeof(T) == 4) {
        o[2 * i] = __float_as_uint(f.x * s), o[2 * i + 1] = __float_as_uint(f.y * s);
      } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 p = __floats2half2_rn(f.x * s, f.y * s);
        o[i] = *reinterpret_cast<const uint32_t*>(&p);
      } else {
        const __nv_bfloat162 p = __floats2bfloat162_rn(f.x * s, f.y * s);
        o[i] = *reinterpret_cast<const uint32_t*>(&p);
      }
    }
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) {
      const uint32_t(&part)[8] = *reinterpret_cast<const uint32_t(*)[8]>(&o[8 * j]);
      if constexpr (kWide) {
        st_32(reinterpret_cast<uint8_t*>(dst) + 32 * j, part);
      } else {
        reinterpret_cast<uint4*>(dst)[2 * j] = make_uint4(part[0], part[1], part[2], part[3]);
        reinterpret_cast<uint4*>(dst)[2 * j + 1] = make_uint4(part[4], part[5], part[6], part[7]);
      }
    }
  }
}

// Tasks and scales are counted in 31 bits; a launch starts at a block of 128 rows.  launch(tasks, blocks, first row, its rows, its
// first scale).
template <int kGroup, class Launch>
static int over_rows(int64_t rows, int64_t hidden, Launch&& launch) {
  const int64_t blocks = (hidden / kGroup + 3) / 4;
  const int64_t step = std::max<int64_t>(1, kMostScales / (blocks * kBlockBytes)) * 128;
  for (int64_t r = 0; r < rows; r += step) {
    const int64_t left = std::min(step, rows - r), row_blocks = (left + 127) / 128;
    // of a block with few rows, only the tasks that have one of them
    const int64_t tail = std::min<int64_t>(left - (row_blocks - 1) * 128, 32);
    const int64_t sets = (row_blocks - 1) * Place<kGroup>::kTasks + (tail + Place<kGroup>::kRows / 4 - 1) / (Place<kGroup>::kRows / 4);
    SGLB_CUDA(launch((uint32_t)(sets * blocks), FastDiv((uint32_t)blocks), r, (int)left, r / 128 * blocks * kBlockBytes));
  }
  return SGLB200_OK;
}

// Tasks a warp takes: two where that still fills the SMs.
constexpr int kAheadMany = 2;
static bool many(uint32_t tasks) { return tasks >= (uint32_t)sm_count() * 64 * kAheadMany; }
static unsigned grid_of(uint32_t tasks, int ahead) { return (tasks + kThreads / 32 * ahead - 1) / (kThreads / 32 * ahead); }

template <typename T, int kGroup, bool kSilu>
static int launch_quant(const void* x, void* codes, void* scales, const float* g, int64_t rows, int64_t hidden, cudaStream_t st) {
  const int units = (int)(hidden / kUnit);
  return over_rows<kGroup>(rows, hidden, [&](uint32_t tasks, FastDiv blocks, int64_t r, int count, int64_t scale) {
    const auto go = [&](auto kern, int ahead) {
      return launch_pdl(kern, grid_of(tasks, ahead), kThreads, 0, st, static_cast<const T*>(x) + r * hidden * (kSilu ? 2 : 1),
                        static_cast<uint2*>(codes) + r * units, static_cast<uint8_t*>(scales) + scale, g, tasks, blocks, (uint32_t)units, count);
    };
    if (reinterpret_cast<uintptr_t>(x) % 32) return go(quant_fp4_kernel<T, kGroup, kSilu, false, 1>, 1);
    return many(tasks) ? go(quant_fp4_kernel<T, kGroup, kSilu, true, kAheadMany>, kAheadMany) : go(quant_fp4_kernel<T, kGroup, kSilu, true, 1>, 1);
  });
}

template <typename T, int kGroup>
static int launch_dequant(const void* codes, const void* scales, const float* g, void* out, int64_t rows, int64_t hidden,
                          cudaStream_t st) {
  const int units = (int)(hidden / kUnit);
  return over_rows<kGroup>(rows, hidden, [&](uint32_t tasks, FastDiv blocks, int64_t r, int count, int64_t scale) {
    const auto go = [&](auto kern, int ahead) {
      return launch_pdl(kern, grid_of(tasks, ahead), kThreads, 0, st, static_cast<const uint2*>(codes) + r * units,
                        static_cast<const uint8_t*>(scales) + scale, g, static_cast<T*>(out) + r * hidden, tasks, blocks, (uint32_t)units, count);
    };
    if (reinterpret_cast<uintptr_t>(out) % 32) return go(dequant_fp4_kernel<T, kGroup, false, 1>, 1);
    return many(tasks) ? go(dequant_fp4_kernel<T, kGroup, true, kAheadMany>, kAheadMany) : go(dequant_fp4_kernel<T, kGroup, true, 1>, 1);
  });
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
