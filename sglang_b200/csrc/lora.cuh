// What the adapters' second-product kernels share (lora.cu, lora_tile.cu).
#pragma once
#include <type_traits>

#include "common.cuh"
#include "narrow.cuh"
#include "narrow_rule.h"

namespace sglb200 {
namespace lora {

constexpr int kMaxAdapters = 1024;
constexpr int kMaxSlices = 8;
constexpr int kMaxRank = 256;

struct Params {
  const void* b;     // [L, N, R]
  const void* base;  // [T, N], rows ld_base apart
  void* out;         // rows ld_out apart; may be base
  const float* h;    // [T, S R]
  const float* scalings;  // or nullptr
  const int32_t* ranks;   // or nullptr
  narrow::Blocks blocks;
  int64_t N, ld_base, ld_out;
  int R, S, max_blocks, vec, in_place;
  int sub, subs;     // a block is taken `sub` rows at a time, in `subs` parts
  int64_t col0[kMaxSlices + 1];  // first column of every merged projection, and the end
  int chunk0[kMaxSlices + 1];    // the first unit of columns, and the end
  uint32_t wait_probes;
  int* status;  // 1 where a pipeline wait has run out
};

// This CTA's even share of `all` (below 2^31) units.  (A division in 64 bits takes a fifth of a microsecond, and a kernel's start was two of them.)
__device__ __forceinline__ void share(int all, int& begin, int& end) {
  const uint32_t each = (uint32_t)all / gridDim.x, more = (uint32_t)all - each * gridDim.x, i = blockIdx.x;
  begin = (int)(each * i + min(i, more)), end = begin + (int)(each + (i < more ? 1 : 0));
}

template <typename T>
__device__ __forceinline__ uint16_t bits(T v) {
  return *reinterpret_cast<const uint16_t*>(&v);
}

// Two neighbouring 16-bit values as floats, and back, rounded to nearest.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// A row of h times `scaling`, value j * 32 + lane in v[j] -> two terms of a 16-bit type, times a power of two, whose inverse is returned;
// put(r, high, low) for r below `width`.  One warp.
//
// The power of two brings the row's largest to [1, 2) for bfloat16, whose two terms hold 16 bits of values of any size, and to [2^14, 2^15) for
// float16, whose smallest step is 2^-24: 22 bits of values down to 2^-16 of the largest, and a bit less for every power of two below.
template <typename T, int kV, class Put>
__device__ __forceinline__ float split_row(const float (&v)[kV], int width, int lane, Put put) {
  float most = 0.f;
#pragma unroll
  for (int j = 0; j < kV; ++j) most = fmaxf(most, fabsf(v[j]));
  const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
  constexpr uint32_t kUp = std::is_same<T, __half>::value ? 14 : 0;
  const bool plain = top < 0x00800000u || top >= 0x7f800000u;  // nothing to bring anywhere
  const uint32_t e = min(max(top >> 23, kUp + 1), 253u);       // (float16's outputs end far above 2^-112)
  const float f = plain ? 1.f : __uint_as_float((254u + kUp - e) << 23);
#pragma unroll
  for (int j = 0; j < kV; ++j) {
    const int r = j * 32 + lane;
    if (r >= width) break;
    const float s = v[j] * f;
    const T a = ElemTraits<T>::from_f32(s);
    const float rest = s - ElemTraits<T>::to_f32(a);
    put(r, bits(a), bits(ElemTraits<T>::from_f32(fabsf(s) < INFINITY ? rest : 0.f)));
  }
  return plain ? 1.f : __uint_as_float((e - kUp) << 23);
}

// lora_tile.cu: the second product for blocks of 128 rows; rank at most kTileRank, p.vec.
constexpr int kTileRank = narrow::kMostTileRank;
int expand_tile(Params& p, int dtype, cudaStream_t st);

}  // namespace lora
}  // namespace sglb200
