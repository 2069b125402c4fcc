// Routing to experts:  s = softmax(x) or sigmoid(x);  c = s + bias;  a group's value = the sum of its one or two largest c;  the
// `topk` largest c of the `topk_group` best groups are picked, and their s are the weights, as they are or divided by their sum, times a
// factor.  Ties go to the lower expert or group.  An expert whose logit is NaN or -inf, or whose c is, is not available; a slot for which
// none is left gets the id -1 and the weight 0.
//
// The order is that of the real numbers.  Without a bias it is the order of the logits.  Where scores decide it is taken in float32, which
// tells two c apart that differ by more than `margin` (below); a row in which two neighbours of the order are closer than that, and are not
// the same logit with the same bias, is decided once more in float64 by its warp: the picks' order (order_exact) of one row in forty with 256
// experts, a whole row (pick_exact) of a few thousand.  c that float64 does not tell apart either (sigmoids of logits from 37 on are all 1) go
// by their logits (pick_by_logit), which is right wherever their biases are equal; a group's sum of two is what float64 makes it.
//
// One warp a row, the row in registers: lane l has consecutive experts of one group.  It is bound by issue slots.  A lane sorts its
// experts once, as integers: an order-preserving bit pattern of c, whose lowest bits give way to the expert's number in the lane and, for the
// picks, to the lane's (which the margins allow for; 16-bit logits lose nothing).  A pick is then one reduction over the lanes' best and a
// shift of the winner's list.  16384 rows of 256 experts, best 8 in 4 of 8 groups: 841 instructions a row and 21 us; with the lanes' best looked for
// after every pick and scores by division 1657 and 33.  The three that decide anew are functions of their own: they run in cold
// instructions, and registers that they need would be the loop's.
#include <algorithm>
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
  int group_size, group_lanes, group_shift, per_lane;  // lanes of a group (2^group_shift), experts of a lane
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
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
constexpr uint32_t kLeast = 0x00800000u;  // of the pattern of a finite number; -inf is below
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }

// How far apart two c have to be for float32 to have their order right.  A sigmoid is off by at most s (1 - s) of the exponential's relative
// error (2^-22, and |x| 2^-24 from its argument, of which s (1 - s) |x| is below 1/4) and 2^-23 s of the reciprocal: below 2^-22.  A softmax
// by up to 2^-19 (the sum of up to 1024 terms, the difference to the row's largest logit, the exponential, the quotient).  Scores of
// logits whose lowest bits gave way: 2^-19 as well (up to 32 units of x, times s (1 - s)).  A rounding of the sum with the bias, and what the
// number in the lane takes: `units` of 2^-23.  A group's value is up to two c, one more rounding and the group's number.
__device__ __forceinline__ float margin(float each, int units, float a, float b) {
  return 2.f * each + (float)(2 * units + 2) * 0x1p-23f * fmaxf(fabsf(a), fabsf(b));
}

// 2^x and 1 / x as the hardware gives them (2 units and 1 unit).
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.44269504f;

// Descending, by Batcher's odd-even merges.
template <int N>
__device__ __forceinline__ void sort_keys(uint32_t (&v)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const uint32_t a = v[i + j], b = v[i + j + k];
            v[i + j] = max(a, b), v[i + j + k] = min(a, b);
          }
}

// Which group lane l's experts belong to, its first expert and how many it has.
struct Place {
  int group, first, count;
};
__device__ __forceinline__ Place place(const Params& p, int lane) {
  Place a;
  a.group = lane >> p.group_shift;
  const int at = (lane & (p.group_lanes - 1)) * p.per_lane;
  a.first = a.group * p.group_size + at;
  a.count = a.group < p.groups ? max(0, min(p.per_lane, p.group_size - at)) : 0;
  return a;
}

// The kept groups, one bit each, by value (lane g has group g's) and index.
template <typename V>
__device__ __forceinline__ uint32_t keep_groups(const Params& p, V mine, int lane) {
  int beaten_by = 0;
  for (int g = 0; g < p.groups; ++g) {
    const V other = __shfl_sync(kAll, mine, g);
    beaten_by += other > mine || (other == mine && g < lane);
  }
  return __ballot_sync(kAll, lane < p.groups && beaten_by < p.kept);
}

// A logit as the order takes it: NaN is -inf, the largest is float32's.
template <typename T>
__device__ __forceinline__ float clean(T v) {
  const float x = ElemTraits<T>::to_f32(v);
  return x > kNone ? fminf(x, FLT_MAX) : kNone;
}

// 64-bit patterns that compare like the doubles they come from; 0 is below them all.
__device__ __forceinline__ uint64_t to_ordered64(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double from_ordered64(uint64_t u) { return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u)); }
__device__ __forceinline__ uint64_t warp_max64(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(kAll, (uint32_t)(v >> 32));
  return (uint64_t)hi << 32 | __reduce_max_sync(kAll, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
}

// c in float64, given the largest logit and the sum of a softmax.
__device__ __forceinline__ double exact_c(const Params& p, float x, int e, double mx, double sum) {
  const double s = p.softmax ? exp((double)x - mx) / sum : 1.0 / (1.0 + exp(-(double)x));
  return p.bias != nullptr ? s + (double)p.bias[e] : s;
}
// The softmax's sum over the row.
template <typename T>
__device__ __forceinline__ double exact_sum(const Params& p, const T* x, double mx, int lane) {
  double sum = 0.0;
  for (int e = lane; e < p.E; e += 32) {
    const float v = clean(x[e]);
    if (v > kNone) sum += exp((double)v - mx);
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(kAll, sum, m);
  return sum;
}

// A pair that goes by its first and, where that is the same, by its second.
struct Ranked {
  uint64_t c;  // (0: none)
  float x;
};
__device__ __forceinline__ bool above(Ranked a, Ranked b) { return a.c > b.c || (a.c == b.c && a.x > b.x); }

// The row's picks by c in float64, then by logit, then by index, for a row with a bias: lane i < k gets the i-th.  Each is looked for anew
// below the one before it, which is slow and small: few rows of few programs come here.
template <typename T>
__device__ __noinline__ int pick_by_logit(const Params& p, const T* x, int lane) {
  const Place at = place(p, lane);
  float mx = kNone;
  for (int j = 0; j < at.count; ++j) mx = fmaxf(mx, clean(x[at.first + j]));
  const double top = (double)warp_max(mx), sum = p.softmax ? exact_sum(p, x, top, lane) : 0.0;
  auto ranked = [&](int e) {
    Ranked r{0, clean(x[e])};
    if (r.x > kNone) {
      const double c = exact_c(p, r.x, e, top, sum);
      if (c > -INFINITY) r.c = to_ordered64(c);
    }
    return r;
  };
  bool in = true;
  if (p.groups > 1) {
    Ranked m1{0, kNone};
    uint64_t m2 = 0;
    for (int j = 0; j < at.count; ++j) {
      const Ranked r = ranked(at.first + j);
      m2 = max(m2, min(m1.c, r.c));
      if (above(r, m1)) m1 = r;
    }
    for (int off = 1; off < p.group_lanes; off <<= 1) {
      const Ranked o{__shfl_xor_sync(kAll, m1.c, off), __shfl_xor_sync(kAll, m1.x, off)};
      m2 = max(max(m2, __shfl_xor_sync(kAll, m2, off)), min(m1.c, o.c));
      if (above(o, m1)) m1 = o;
    }
    if (p.top == 2) {  // (a sum is by itself)
      if (m1.c != 0) m1.c = to_ordered64(from_ordered64(m1.c) + (m2 != 0 ? from_ordered64(m2) : 0.0));
      m1.x = 0.f;
    }
    int beaten_by = 0;
    for (int g = 0; g < p.groups; ++g) {
      const Ranked o{__shfl_sync(kAll, m1.c, g * p.group_lanes), __shfl_sync(kAll, m1.x, g * p.group_lanes)};
      beaten_by += above(o, m1) || (!above(m1, o) && g < at.group);
    }
    in = beaten_by < p.kept;
  }
  Ranked last{~0ull, INFINITY};
  int last_e = -1, picked = -1;
  for (int i = 0; i < p.k; ++i) {
    Ranked best{0, kNone};
    int e_best = -1;
    for (int j = 0; j < at.count && in; ++j) {
      const int e = at.first + j;
      const Ranked r = ranked(e);
      const bool left = above(last, r) || (!above(r, last) && e > last_e);
      if (left && r.c != 0 && above(r, best)) best = r, e_best = e;
    }
    last.c = warp_max64(best.c);
    if (last.c == 0) break;
    const uint32_t by_logit = best.c == last.c ? to_ordered(best.x) : 0u, largest = __reduce_max_sync(kAll, by_logit);
    const int winner = __ffs(__ballot_sync(kAll, by_logit == largest)) - 1;
    last.x = __shfl_sync(kAll, best.x, winner), last_e = __shfl_sync(kAll, e_best, winner);
    if (lane == i) picked = last_e;
  }
  return picked;
}

// The row's picks in float64: lane i < k gets the i-th.
template <typename T, int kPer>
__device__ __noinline__ int pick_exact(const Params& p, const T* x, int lane) {
  const Place at = place(p, lane);
  float v[kPer], mx = kNone;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    v[j] = j < at.count ? clean(x[at.first + j]) : kNone;
    mx = fmaxf(mx, v[j]);
  }
  const bool biased = p.bias != nullptr, scored = biased || p.top == 2;
  const double top = (double)warp_max(mx), sum = p.softmax && scored ? exact_sum(p, x, top, lane) : 0.0;
  uint64_t c[kPer];  // (without a bias the logits' order: a score grows with its logit)
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const double s = !(v[j] > kNone) ? -INFINITY : biased ? exact_c(p, v[j], at.first + j, top, sum) : (double)v[j];
    c[j] = s > -INFINITY ? to_ordered64(s) : 0;
  }
  bool by_logit = false;
  if (p.groups > 1) {
    uint64_t m1 = 0, m2 = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) m2 = max(m2, min(m1, c[j])), m1 = max(m1, c[j]);
    for (int off = 1; off < p.group_lanes; off <<= 1) {
      const uint64_t o1 = __shfl_xor_sync(kAll, m1, off), o2 = __shfl_xor_sync(kAll, m2, off);
      m2 = max(max(m2, o2), min(m1, o1)), m1 = max(m1, o1);
    }
    uint64_t value = m1;
    if (p.top == 2 && m1 != 0) {
      double v1 = from_ordered64(m1), v2 = m2 != 0 ? from_ordered64(m2) : 0.0;
      if (!biased) v1 = exact_c(p, (float)v1, 0, top, sum), v2 = m2 != 0 ? exact_c(p, (float)v2, 0, top, sum) : 0.0;
      value = to_ordered64(v1 + v2);
    }
    uint64_t mine = __shfl_sync(kAll, value, (lane * p.group_lanes) & 31);
    if (lane >= p.groups) mine = 0;
    const uint32_t keep = keep_groups<uint64_t>(p, mine, lane);
    if (!(keep >> at.group & 1u))
#pragma unroll
      for (int j = 0; j < kPer; ++j) c[j] = 0;
    if (biased && p.top == 1) {  // does a group that goes have the value of one that stays?
      const uint64_t most = warp_max64(keep >> lane & 1u ? 0 : mine);
      by_logit = __any_sync(kAll, (keep >> lane & 1u) && mine == most && most != 0);
    }
  }
  int picked = -1, e = -1;
  uint64_t last = 0;
  for (int i = 0; i < p.k; ++i) {
    uint64_t best = 0;
    int best_j = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (c[j] > best) best = c[j], best_j = j;
    const uint64_t winning = warp_max64(best);
    if (winning == 0) break;
    const int winner = __ffs(__ballot_sync(kAll, best == winning)) - 1, before = e;
    e = __shfl_sync(kAll, at.first + best_j, winner);
    if (lane == winner)
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (j == best_j) c[j] = 0;
    if (lane == i) picked = e;
    if (winning == last && biased) by_logit = by_logit || clean(x[e]) > clean(x[before]);
    last = winning;
  }
  if (biased && last != 0) {  // is a larger logit left of the last one's c?
    bool left = false;
#pragma unroll
    for (int j = 0; j < kPer; ++j) left = left || c[j] == last;
    if (__any_sync(kAll, left)) {
      bool larger = false;
      for (int j = 0; j < at.count && left; ++j) {
        const float other = clean(x[at.first + j]);
        larger = larger || (other > clean(x[e]) && to_ordered64(exact_c(p, other, at.first + j, top, sum)) == last);
      }
      by_logit = by_logit || __any_sync(kAll, larger);
    }
  }
  return by_logit ? pick_by_logit<T>(p, x, lane) : picked;
}

// The `count` picks of the lanes (none left of those beyond in question) put in order in the same way, through `room`: lane i gets the i-th.
template <typename T>
__device__ __noinline__ int order_exact(const Params& p, const T* x, float mx, int picked, int count, int lane, uint32_t* room) {
  const double sum = p.softmax && p.bias != nullptr ? exact_sum(p, x, (double)mx, lane) : 0.0;
  uint64_t c = 0;
  float v = kNone;
  if (lane < count) {
    v = clean(x[picked]);
    c = to_ordered64(p.bias != nullptr ? exact_c(p, v, picked, (double)mx, sum) : (double)v);
  }
  int rank = 0, same = 0;
  for (int i = 0; i < count; ++i) {
    const uint64_t other = __shfl_sync(kAll, c, i);
    rank += other > c, same += other == c;
  }
  if (__any_sync(kAll, lane < count && same > 1))
    for (int i = 0; i < count; ++i) {
      const uint64_t other = __shfl_sync(kAll, c, i);
      const float other_v = __shfl_sync(kAll, v, i);
      const int e = __shfl_sync(kAll, picked, i);
      rank += other == c && (other_v > v || (other_v == v && e < picked));
    }
  __syncwarp();
  if (lane < count) room[rank] = (uint32_t)picked;
  __syncwarp();
  return lane < count ? (int)room[lane] : -1;
}

// A lane's `count` consecutive values at `at` of the row (the rest -inf), 16 bytes at a time where they lie so.
template <typename T, int kPer>
__device__ __forceinline__ void load_run(const T* at, int count, float (&v)[kPer]) {
  constexpr int kVec = 16 / (int)sizeof(T);
  if (kPer % kVec == 0 && count == kPer && (reinterpret_cast<uintptr_t>(at) & 15u) == 0) {
    uint4 raw[kPer % kVec == 0 ? kPer / kVec : 1];
#pragma unroll
    for (int c = 0; c < kPer / kVec; ++c) raw[c] = __ldg(reinterpret_cast<const uint4*>(at) + c);
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = ElemTraits<T>::to_f32(reinterpret_cast<const T*>(raw)[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = j < count ? ElemTraits<T>::to_f32(at[j]) : kNone;
  }
}

// kSoftmax: else sigmoid.
template <typename T, int kPer, bool kSoftmax>
__global__ void __launch_bounds__(kWarps * 32, kPer <= 8 ? 4 : 1) route_kernel(const T* __restrict__ logits, const __grid_constant__ Params p) {
  constexpr uint32_t kIndex = kPer - 1;  // the bits of a key that hold the expert's number in the lane, the lowest on top
  constexpr uint32_t kUnits = 32 * kPer;  // and the lane
  __shared__ uint32_t picks[kWarps][kMaxTopk];
  const int lane = threadIdx.x & 31, warp = ptx::warp_index();
  ptx::launch_dependents();
  const Place at = place(p, lane);
  const bool biased = p.bias != nullptr;
  ptx::grid_dependency_wait();
  float add[kPer];
  if (biased) load_run<float, kPer>(p.bias + at.first, at.count, add);
  int64_t row = (int64_t)blockIdx.x * kWarps + warp;
  const int64_t step = (int64_t)gridDim.x * kWarps;
  for (; row < p.rows; row += step) {
    const T* logits_row = logits + row * p.E;
    float x[kPer];
    load_run<T, kPer>(logits_row + at.first, at.count, x);
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[j] = fminf(fmaxf(x[j], kNone), FLT_MAX);  // (the larger of a NaN and -inf is -inf)
    float mx = kNone, inv = 0.f;
    if (kSoftmax && (biased || p.top == 2 || !p.renorm)) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) mx = fmaxf(mx, x[j]);
      mx = warp_max(mx);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < kPer; ++j) sum += x[j] > kNone ? fast_exp2((x[j] - mx) * kLog2e) : 0.f;
      sum = warp_sum(sum);
      inv = sum > 0.f ? 1.f / sum : 0.f;
    }
    auto score = [&](float v) { return kSoftmax ? fast_exp2((v - mx) * kLog2e) * inv : fast_rcp(1.f + fast_exp2(v * -kLog2e)); };
    uint32_t key[kPer];  // descending; below kLeast: not available
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      float c = x[j];
      if (biased) c = c > kNone ? fmaxf(score(c) + add[j], kNone) : kNone;
      key[j] = (to_ordered(c) & ~kIndex) | (kIndex - j);
    }
    sort_keys<kPer>(key);

    constexpr float kEach = kSoftmax ? 0x1p-19f : 0x1p-22f;
    bool redo = false;  // the row is decided in float64 from its groups on
    if (p.groups > 1) {
      // the group's two largest, in each of its lanes
      uint32_t m1 = key[0], m2 = kPer > 1 ? key[kPer > 1 ? 1 : 0] : 0u;
      for (int off = 1; off < p.group_lanes; off <<= 1) {
        const uint32_t o1 = __shfl_xor_sync(kAll, m1, off), o2 = __shfl_xor_sync(kAll, m2, off);
        m2 = max(max(m2, o2), min(m1, o1)), m1 = max(m1, o1);
      }
      m1 = __shfl_sync(kAll, m1, (lane * p.group_lanes) & 31), m2 = __shfl_sync(kAll, m2, (lane * p.group_lanes) & 31);
      // lane g < groups: group g's value
      float v1 = from_ordered(m1 & ~kIndex), v2 = from_ordered(m2 & ~kIndex);
      // (the largest of what is added: a sum may be smaller than what it is off by)
      const float reach = __uint_as_float(__reduce_max_sync(
          kAll, lane < p.groups && m1 >= kLeast ? __float_as_uint(fmaxf(fabsf(v1), m2 >= kLeast && p.top == 2 ? fabsf(v2) : 0.f)) : 0u));
      if (p.top == 2) {
        if (!biased) v1 = score(v1), v2 = score(v2);
        v1 = m2 >= kLeast ? v1 + v2 : v1;
      }
      const uint32_t value = lane < p.groups && m1 >= kLeast ? to_ordered(v1) : 0u;
      const uint32_t keep = keep_groups<uint32_t>(p, value, lane);
      // the last that stays and the first that goes have to be told apart
      const bool in = keep >> lane & 1u;
      const uint32_t low = __reduce_min_sync(kAll, in ? value : kAll), high = __reduce_max_sync(kAll, in ? 0u : value);
      if (p.kept < p.groups && high != 0u) {
        const float a = from_ordered(low), b = from_ordered(high);
        if (biased) {
          redo = !(a - b > (float)p.top * margin(kEach, kPer + 2, reach, 0.f));
        } else if (p.top == 2) {  // (scores of logits whose lowest bits gave way)
          redo = !(a - b > 2.f * margin(0x1p-19f + (kSoftmax ? 0x1p-18f * reach : 0.f), kPer + 2, 1.f, 0.f));
        } else if (sizeof(T) == 4) {
          redo = !(a - b > margin(0.f, kPer, a, b));
        }  // (16-bit logits lose nothing)
      }
      if (!(keep >> at.group & 1u))
#pragma unroll
        for (int j = 0; j < kPer; ++j) key[j] = 0u;
    }

    // The picks, best first, through shared memory to lane i.  With the lane in its lowest bits as well, the lower on top, a key is the row's
    // only one of its kind, and a pick is a reduction and a comparison.
    const bool inexact = biased || sizeof(T) == 4;  // neighbours have to be told apart, two beyond the last as well
    const int looks = min(inexact ? p.k + 2 : p.k, 32);
#pragma unroll
    for (int j = 0; j < kPer; ++j) key[j] = (key[j] & ~(kUnits - kPer)) | (uint32_t)(31 - lane) * kPer;
    int count = 0;
    for (; count < looks; ++count) {
      const uint32_t top = __reduce_max_sync(kAll, key[0]);
      if (top < kLeast) break;
      if (lane == 0) picks[warp][count] = top;
      if (key[0] == top) {
#pragma unroll
        for (int j = 0; j + 1 < kPer; ++j) key[j] = key[j + 1];
        key[kPer - 1] = 0u;
      }
    }
    __syncwarp();
    const uint32_t pick = picks[warp][lane], mine = pick & ~(kUnits - 1);
    int picked = __shfl_sync(kAll, at.first, 31 - (int)(pick / kPer % 32)) + (int)(kIndex - (pick & kIndex));
    if (lane >= count) picked = -1;
    if (inexact) {
      const uint32_t after = __shfl_down_sync(kAll, mine, 1);
      const float a = from_ordered(mine), b = from_ordered(after);
      bool tell = lane + 1 < count && lane < p.k + 1 && !(a - b > margin(biased ? kEach : 0.f, kUnits, a, b));
      const uint32_t close = __ballot_sync(kAll, tell);
      uint32_t telling = close;
      if (close != 0u) {  // equal logits with equal biases are in order
        const int after_e = __shfl_down_sync(kAll, picked, 1);
        if (tell) tell = !(clean(logits_row[picked]) == clean(logits_row[after_e]) && (!biased || p.bias[picked] == p.bias[after_e]));
        telling = __ballot_sync(kAll, tell);
      }
      // Neighbours among the picks and the first that goes are put in order.  Where that one is close to the last pick and to the next as well,
      // the run of close ones may go on behind what was looked at: the row is decided anew, unless all of the run are equal.  From 31 picks on the
      // next cannot be looked at.
      const uint32_t among = p.k >= 32 ? kAll : (1u << p.k) - 1;
      if (p.k > 30) {
        redo = redo || count == 32;
      } else if ((close >> (p.k - 1) & 3u) == 3u) {
        const int from = 32 - __clz(~close & among);  // where the run begins
        bool differs = (telling & ((2u << p.k) - 1)) >> from != 0u;
        if (!differs) {  // a lane's experts that are left, in descending order
          const int tied = __shfl_sync(kAll, picked, p.k);
          const float c = __shfl_sync(kAll, a, p.k);
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const float left = from_ordered(key[j] & ~(kUnits - 1));
            if (key[j] < kLeast || c - left > margin(biased ? kEach : 0.f, kUnits, c, left)) continue;
            const int e = at.first + (int)(kIndex - (key[j] & kIndex));
            if (!(clean(logits_row[e]) == clean(logits_row[tied]) && (!biased || p.bias[e] == p.bias[tied]))) differs = true;
          }
          differs = __any_sync(kAll, differs);
        }
        redo = redo || differs;
      }
      if ((telling & among) != 0u && !redo) picked = order_exact<T>(p, logits_row, mx, picked, min(count, p.k + 1), lane, picks[warp]);
    }
    if (redo) picked = pick_exact<T, kPer>(p, logits_row, lane);
    if (lane >= p.k) picked = -1;

    // Weights: the score, or its share of the picks' scores, for which the largest pick takes the place of the row's largest logit (softmax)
    // or of 0 (sigmoid = e^min(x, 0) / (1 + e^-|x|)): scores that are too small for float32 have shares all the same.
    const bool there = picked >= 0;
    const float px = there ? clean(logits_row[picked]) : 0.f;
    float w;
    if (p.renorm) {
      const float num = kSoftmax ? px : fminf(px, 0.f);
      const float shift = warp_max(there ? num : kNone);
      w = there ? expf(num - shift) : 0.f;
      if (!kSoftmax) w = __fdividef(w, 1.f + expf(-fabsf(px)));
      const float sum = warp_sum(w);
      w = there ? __fdividef(w, sum) * p.factor : 0.f;
    } else {
      w = kSoftmax ? expf(px - mx) * inv : 1.f / (1.f + expf(-px));
      w = there ? w * p.factor : 0.f;
    }
    if (lane < p.k) {
      p.out_w[row * p.k + lane] = w;
      p.out_i[row * p.k + lane] = picked;
    }
    __syncwarp();
  }
}

template <typename T, bool kSoftmax>
static int launch(const void* logits, const Params& p, cudaStream_t st) {
  // (rows in rounds: the next row is asked for under this one)
  const unsigned grid = (unsigned)std::min<int64_t>((p.rows + kWarps - 1) / kWarps, 4 * sm_count());
  const T* x = static_cast<const T*>(logits);
#define SGLB_ROUTE_CASE(P)                                                                              \
  if (p.per_lane <= P) {                                                                                \
    SGLB_CUDA(launch_pdl(route_kernel<T, P, kSoftmax>, grid, kWarps * 32, (size_t)0, st, x, p));        \
    return SGLB200_OK;                                                                                  \
  }
  SGLB_ROUTE_CASE(1) SGLB_ROUTE_CASE(2) SGLB_ROUTE_CASE(4) SGLB_ROUTE_CASE(8) SGLB_ROUTE_CASE(16) SGLB_ROUTE_CASE(32)
#undef SGLB_ROUTE_CASE
  return fail(SGLB200_E_UNSUPPORTED, "route_topk: %d groups of %d experts", p.groups, p.group_size);
}
template <typename T>
static int launch(const void* logits, const Params& p, cudaStream_t st) {
  return p.softmax ? launch<T, true>(logits, p, st) : launch<T, false>(logits, p, st);
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
  p.group_lanes = lanes, p.group_shift = 0;
  while (1 << p.group_shift < lanes) ++p.group_shift;
  p.per_lane = (p.group_size + lanes - 1) / lanes;
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
