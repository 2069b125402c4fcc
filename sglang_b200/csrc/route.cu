// Routing to experts:  s = softmax(x) or sigmoid(x);  c = s + bias;  a group's value = the sum of its one or two largest c;  the
// `topk` largest c of the `topk_group` best groups are picked, and their s are the weights, as they are or divided by their sum, times a
// factor.  Ties go to the lower expert or group.  An expert whose logit is NaN or -inf, or whose c is, is not available; a slot for which
// none is left gets the id -1 and the weight 0.
//
// The order is that of the real numbers.  Without a bias it is the order of the logits.  Where scores decide it is taken in float32, which
// tells two c apart that differ by more than `margin` (below); a row in which two neighbours of the order are closer than that, and are not
// the same logit with the same bias, is decided once more in float64 by its warp.  With 256 experts that is one row in a few hundred.
//
// One warp a row, the row in registers: lane l has consecutive experts of one group, so that a group's best come from its lanes' registers.
// The picks are arg-maxima over the lanes' own best: one reduction over order-preserving bit patterns and one vote; a lane holds lower
// experts than the next, so the lowest lane of equals has the lowest expert.
#include <cfloat>

#include "common.cuh"
#include "ptx_sm100.cuh"

namespace sglb200 {
namespace route {

constexpr int kWarps = 8;       // rows per CTA
constexpr int kMaxPerLane = 32;
constexpr int kMaxTopk = 32;
constexpr int kMaxGroups = 32;
constexpr float kNone = -INFINITY;
constexpr uint32_t kAll = 0xffffffffu;

struct Params {
  const float* bias;  // or nullptr
  float* out_w;
  int32_t* out_i;
  int64_t rows;
  int E, k, groups, kept, top;
  int group_size, group_lanes, per_lane;  // lanes of a group, experts of a lane
  int softmax, renorm;
  float factor;
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, m));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(kAll, v, m);
  return v;
}
// Bit patterns that compare as unsigned integers like the floats they come from (-0 as +0), and the way back.
__device__ __forceinline__ uint32_t to_ordered(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }

// How far apart two c have to be for float32 to have their order right.  A sigmoid is off by at most s (1 - s) (2^-22 + 2^-24) of the
// exponential (two units, and the sum beside it) and 2^-24 s of the quotient: below 2^-23.  A softmax by up to 2^-20 (the sum of up to
// 1024 terms, the difference to the row's largest logit, the exponential, the quotient's two roundings).  Two of them, and a rounding of
// each sum with the bias; a group's value is two c and one more rounding.
__device__ __forceinline__ float margin(const Params& p, float a, float b) {
  const float each = p.softmax ? 0x1p-20f : 0x1p-23f;
  return (float)(2 * p.top) * (each + 0x1p-23f * fmaxf(fabsf(a), fabsf(b)));
}

__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v = fmax(v, __shfl_xor_sync(kAll, v, m));
  return v;
}

// Which group lane l's experts belong to, its first expert and how many it has.
struct Place {
  int group, first, count;
};
__device__ __forceinline__ Place place(const Params& p, int lane) {
  Place a;
  a.group = lane / p.group_lanes;
  const int at = (lane - a.group * p.group_lanes) * p.per_lane;
  a.first = a.group * p.group_size + at;
  a.count = a.group < p.groups ? max(0, min(p.per_lane, p.group_size - at)) : 0;
  return a;
}

// The kept groups, one bit each, by value and index.
template <typename V>
__device__ __forceinline__ uint32_t keep_groups(const Params& p, V mine, int lane, V none) {
  int beaten_by = 0;
  for (int g = 0; g < p.groups; ++g) {
    const V other = __shfl_sync(kAll, mine, g);
    beaten_by += other > mine || (other == mine && g < lane);
  }
  return __ballot_sync(kAll, lane < p.groups && beaten_by < p.kept);
}

// The sum of a group's `top` largest values (of those that are there), in each of its lanes.
template <int kPer, typename V>
__device__ __forceinline__ V group_value(const Params& p, const V (&c)[kPer], V none) {
  V m1 = none, m2 = none;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (c[j] > m1) {
      m2 = m1, m1 = c[j];
    } else if (c[j] > m2) {
      m2 = c[j];
    }
  }
  for (int off = 1; off < p.group_lanes; off <<= 1) {
    const V o1 = __shfl_xor_sync(kAll, m1, off), o2 = __shfl_xor_sync(kAll, m2, off);
    const V low = m1 < o1 ? m1 : o1;
    m1 = m1 < o1 ? o1 : m1;
    m2 = m2 < o2 ? o2 : m2;
    m2 = m2 < low ? low : m2;
  }
  return p.top == 2 && m2 > none ? m1 + m2 : m1;
}

// The row's picks in float64: lane i < k gets the i-th.  `kept_x`: the row's logits in shared memory.
template <int kPer>
__device__ __noinline__ int pick_exact(const Params& p, const float* kept_x, int lane) {
  const Place at = place(p, lane);
  const double none = -INFINITY;
  double c[kPer];
  double mx = none, sum = 0.0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    c[j] = j < at.count ? (double)kept_x[at.first + j] : none;
    mx = fmax(mx, c[j]);
  }
  if (p.softmax) {
    mx = warp_max(mx);
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum += c[j] > none ? exp(c[j] - mx) : 0.0;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(kAll, sum, m);
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (!(c[j] > none)) continue;
    const double s = p.softmax ? exp(c[j] - mx) / sum : 1.0 / (1.0 + exp(-c[j]));
    const double v = s + (p.bias != nullptr ? (double)p.bias[at.first + j] : 0.0);
    c[j] = v > none ? v : none;
  }
  if (p.groups > 1) {
    const double value = group_value<kPer>(p, c, none);
    const double mine = __shfl_sync(kAll, value, (lane * p.group_lanes) & 31);
    const uint32_t keep = keep_groups<double>(p, lane < p.groups ? mine : none, lane, none);
    if (!(keep >> at.group & 1u))
#pragma unroll
      for (int j = 0; j < kPer; ++j) c[j] = none;
  }
  if (p.bias == nullptr) {  // (a score grows with its logit)
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (c[j] > none) c[j] = (double)kept_x[at.first + j];
  }
  int picked = -1;
  for (int i = 0; i < p.k; ++i) {
    double best = none;
    int best_j = -1;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (c[j] > best) best = c[j], best_j = j;
    const double top = warp_max(best);
    if (!(top > none)) break;
    const int winner = __ffs(__ballot_sync(kAll, best == top)) - 1;
    const int e = __shfl_sync(kAll, at.first + best_j, winner);
    if (lane == winner)
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (j == best_j) c[j] = none;
    if (lane == i) picked = e;
  }
  return picked;
}

// A lane's `count` consecutive values at `at` of the row (the rest none), 16 bytes at a time where they lie so.
template <typename T, int kPer>
__device__ __forceinline__ void load_run(const T* at, int count, float (&v)[kPer]) {
  constexpr int kVec = 16 / (int)sizeof(T);
  if (kPer % kVec == 0 && (count == kPer || count == 0) && (reinterpret_cast<uintptr_t>(at) & 15u) == 0) {
    uint4 raw[kPer % kVec == 0 ? kPer / kVec : 1];
#pragma unroll
    for (int c = 0; c < kPer / kVec; ++c) raw[c] = count ? __ldg(reinterpret_cast<const uint4*>(at) + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = ElemTraits<T>::to_f32(reinterpret_cast<const T*>(raw)[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = j < count ? ElemTraits<T>::to_f32(at[j]) : 0.f;
  }
}

template <typename T, int kPer>
__global__ void __launch_bounds__(kWarps * 32) route_kernel(const T* __restrict__ logits, const Params p) {
  extern __shared__ float smem[];  // per warp: the row's logits
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* kept_x = smem + warp * p.E;
  const int64_t row = (int64_t)blockIdx.x * kWarps + warp;
  ptx::launch_dependents();
  ptx::grid_dependency_wait();
  if (row >= p.rows) return;
  const Place at = place(p, lane);
  float x[kPer], c[kPer];
  load_run<T, kPer>(logits + row * p.E + at.first, at.count, x);
  const bool scored = p.bias != nullptr || p.top == 2;  // float32 decides, and may have to hand over to float64
  float mx = kNone;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const bool live = j < at.count && x[j] > kNone;  // (false for a NaN)
    x[j] = live ? fminf(x[j], FLT_MAX) : kNone;
    if (j < at.count) kept_x[at.first + j] = x[j];
    mx = fmaxf(mx, x[j]);
  }
  float inv = 0.f;
  if (p.softmax && (scored || !p.renorm)) {
    mx = warp_max(mx);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      c[j] = x[j] > kNone ? expf(x[j] - mx) : 0.f;
      sum += c[j];
    }
    sum = warp_sum(sum);
    inv = sum > 0.f ? 1.f / sum : 0.f;
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (!scored) {
      c[j] = x[j];
    } else {
      const float s = p.softmax ? c[j] * inv : 1.f / (1.f + expf(-x[j]));
      const float v = s + (p.bias != nullptr && j < at.count ? p.bias[at.first + j] : 0.f);
      c[j] = x[j] > kNone && v > kNone ? v : kNone;
    }
  }
  bool close = false;
  if (p.groups > 1) {
    const float value = group_value<kPer>(p, c, kNone);
    float mine = __shfl_sync(kAll, value, (lane * p.group_lanes) & 31);
    if (lane >= p.groups) mine = kNone;
    const uint32_t keep = keep_groups<float>(p, mine, lane, kNone);
    if (scored) {
      const bool in = keep >> lane & 1u;
      const float low = from_ordered(__reduce_min_sync(kAll, in ? to_ordered(mine) : kAll));
      const float high = from_ordered(__reduce_max_sync(kAll, in ? 0u : to_ordered(mine)));
      close = keep != kAll && high > kNone && !(low - high > margin(p, low, high));
    }
    if (!(keep >> at.group & 1u))
#pragma unroll
      for (int j = 0; j < kPer; ++j) c[j] = kNone;
  }
  if (p.bias == nullptr && p.top == 2) {  // the groups' values were sums of scores; the logits order the experts
#pragma unroll
    for (int j = 0; j < kPer; ++j) c[j] = c[j] > kNone ? x[j] : kNone;
  }
  __syncwarp();

  float best;
  int best_j;
  auto look = [&]() {
    best = kNone, best_j = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (c[j] > best) best = c[j], best_j = j;
  };
  look();
  int picked = -1, last_e = 0;
  float last = 0.f;
  const int looks = p.bias != nullptr ? p.k + 1 : p.k;  // (the first that is not picked has to be told apart as well)
  for (int i = 0; i < looks; ++i) {
    const uint32_t key = to_ordered(best), top = __reduce_max_sync(kAll, key);
    const float v = from_ordered(top);
    if (!(v > kNone)) break;
    const int winner = __ffs(__ballot_sync(kAll, key == top)) - 1;
    const int e = __shfl_sync(kAll, at.first + best_j, winner);
    if (p.bias != nullptr) {
      if (i > 0 && !(last - v > margin(p, last, v)))
        close = close || !(kept_x[last_e] == kept_x[e] && p.bias[last_e] == p.bias[e]);
      last = v, last_e = e;
    }
    if (i == p.k) break;
    if (lane == i) picked = e;
    if (lane == winner) {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (j == best_j) c[j] = kNone;
      look();
    }
  }
  if (close) picked = pick_exact<kPer>(p, kept_x, lane);

  // Weights: the score, or its share of the picks' scores, for which the largest pick takes the place of the row's largest logit (softmax) or
  // of 0 (sigmoid = e^min(x, 0) / (1 + e^-|x|)): scores that are too small for float32 have shares all the same.
  const bool there = picked >= 0;
  const float px = there ? kept_x[picked] : 0.f;
  float w;
  if (p.renorm) {
    const float num = p.softmax ? px : fminf(px, 0.f);
    const float shift = warp_max(there ? num : kNone);
    w = there ? expf(num - shift) : 0.f;
    if (!p.softmax) w /= 1.f + expf(-fabsf(px));
    const float sum = warp_sum(w);
    w = there ? w / sum * p.factor : 0.f;
  } else {
    w = p.softmax ? expf(px - mx) * inv : 1.f / (1.f + expf(-px));
    w = there ? w * p.factor : 0.f;
  }
  if (lane < p.k) {
    p.out_w[row * p.k + lane] = w;
    p.out_i[row * p.k + lane] = picked;
  }
}

template <typename T>
static int launch(const void* logits, const Params& p, cudaStream_t st) {
  const unsigned grid = (unsigned)((p.rows + kWarps - 1) / kWarps);
  const size_t smem = (size_t)kWarps * p.E * sizeof(float);
  const T* x = static_cast<const T*>(logits);
#define SGLB_ROUTE_CASE(P)                                                                    \
  if (p.per_lane <= P) {                                                                      \
    SGLB_CUDA(launch_pdl(route_kernel<T, P>, grid, kWarps * 32, smem, st, x, p));             \
    return SGLB200_OK;                                                                        \
  }
  SGLB_ROUTE_CASE(1) SGLB_ROUTE_CASE(2) SGLB_ROUTE_CASE(4) SGLB_ROUTE_CASE(8) SGLB_ROUTE_CASE(16) SGLB_ROUTE_CASE(32)
#undef SGLB_ROUTE_CASE
  return fail(SGLB200_E_UNSUPPORTED, "route_topk: %d groups of %d experts", p.groups, p.group_size);
}

}  // namespace route
}  // namespace sglb200

using namespace sglb200;

extern "C" int sglb200_route_topk(const void* logits, int dtype, int64_t rows, int num_experts, int topk, int softmax,
                                  const float* correction_bias, int num_expert_group, int topk_group, int group_top, int renormalize,
                                  float routed_scaling_factor, float* topk_weights, int32_t* topk_ids, void* stream) {
  SGLB_REQUIRE(rows >= 0 && rows < (1ll << 33) && num_experts >= 1 && topk >= 1 && topk <= num_experts,
               "route_topk: rows=%lld experts=%d topk=%d", (long long)rows, num_experts, topk);
  SGLB_REQUIRE(dtype >= 0 && dtype <= 2, "route_topk: dtype %d (0 bf16, 1 fp16, 2 fp32)", dtype);
  SGLB_REQUIRE(num_expert_group >= 1 && num_experts % num_expert_group == 0, "route_topk: %d groups for %d experts (groups of equal size)",
               num_expert_group, num_experts);
  SGLB_REQUIRE(topk_group >= 1 && topk_group <= num_expert_group, "route_topk: topk_group %d of %d groups", topk_group, num_expert_group);
  SGLB_REQUIRE((int64_t)topk_group * (num_experts / num_expert_group) >= topk, "route_topk: topk %d exceeds the experts of %d kept groups",
               topk, topk_group);
  SGLB_REQUIRE(group_top == 1 || group_top == 2, "route_topk: group_top %d is neither 1 nor 2", group_top);
  if (topk > route::kMaxTopk || num_expert_group > route::kMaxGroups)
    return fail(SGLB200_E_UNSUPPORTED, "route_topk: topk %d, %d groups (at most %d and %d)", topk, num_expert_group, route::kMaxTopk,
                route::kMaxGroups);
  route::Params p{};
  p.group_size = num_experts / num_expert_group;
  int lanes = 32;
  while (lanes * num_expert_group > 32) lanes >>= 1;
  p.group_lanes = lanes, p.per_lane = (p.group_size + lanes - 1) / lanes;
  if (p.per_lane > route::kMaxPerLane)
    return fail(SGLB200_E_UNSUPPORTED, "route_topk: %d groups of %d experts (at most %d experts a group)", num_expert_group, p.group_size,
                route::kMaxPerLane * lanes);
  if (rows == 0) return SGLB200_OK;
  SGLB_REQUIRE(logits && topk_weights && topk_ids, "route_topk: null pointer");
  p.bias = correction_bias, p.out_w = topk_weights, p.out_i = topk_ids, p.rows = rows, p.E = num_experts, p.k = topk;
  p.groups = num_expert_group, p.kept = topk_group, p.top = num_expert_group > 1 ? group_top : 1;
  p.softmax = softmax != 0, p.renorm = renormalize != 0, p.factor = routed_scaling_factor;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == 0) return route::launch<__nv_bfloat16>(logits, p, st);
  if (dtype == 1) return route::launch<__half>(logits, p, st);
  return route::launch<float>(logits, p, st);
}
