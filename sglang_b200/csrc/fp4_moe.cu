// The routed experts of a few tokens, 4-bit weights (e2m1, groups of 16 with e4m3 scales in rows' order, a factor per expert) and
// 16-bit activations, in two launches:
//
//   h[s, i]   = silu(a13_e * sum_k G_e[i, k] x[t, k]) * (a13_e * sum_k U_e[i, k] x[t, k])     for slot s = (t, j), e = ids[s]
//   out[t, n] = factor * sum_j weights[s] * a2_e * sum_i W2_e[n, i] h[s, i]
//
// Few tokens name many experts once or twice each, so a layer is one read of those experts' weights: 0.5625 bytes a weight, and
// the weights come in faster (12 T/s) than they could be expanded for anything but the matrix instructions.  A weight times its group's
// scale has six significant bits and lies within fp16, so it goes into mma.m16n8k16 exactly; the weights are the 16-row side, read
// straight from their rows in the order in which the instruction's lanes hold them (the order of k within a sum is free), and eight
// activation rows are the other; with more rows of an expert, 16 or 32 of them share what was expanded.  bf16 activations become fp16
// under a power of two per row: 2^6 where the row's largest magnitude lies in [2^-5, 2^9), else what brings that to 2^14.  So they are
// exact down to 2^-18 of that magnitude and off by at most 2^-26 of it below.  h is kept in float32 and enters the second product
// under such a power of two as the sum of two fp16 terms, hi + 2^-11 lo, a column each: 23 bits, off by at most 2^-23 of a value or 2^-37 of
// the row's largest.  (hi alone, 11 bits, moved one bf16 output in fifty by a step.)
//
// A CTA's item is a pass (an expert and at most 32 of its slots) and a few 16-row tiles; its 16 warps split the tiles and K.
// Passes of one expert go to CTAs of their own, which read its weights from the L2 (64 tokens, 4 of 8 experts of 4096 x 1024: 106
// us, against 148 where a CTA took all passes of its tiles in turn; 82 with passes of eight rows instead of four; 93 since a row of
// h has two columns).  One more warp keeps a ring of 36 KB stages (codes and scales of 256 columns of all 16 tiles, one TMA load
// each) full across items, so that the memory streams while rows are staged and sums are taken.  Partial sums meet in shared memory
// in a fixed order.  The second launch writes every slot's product to a scratch, and whichever CTA is the last of a set of columns
// adds the slots of a token in their order, so results do not depend on the order of CTAs.
//
// 16 tokens, 8 of 256 experts of 7168 x 2048 (101 named, 2.5 GB): 483 to 550 us with the weights of three layers in turn, 0.70 to
// 0.79 of the measured copy rate; the first product streams at 0.96 of it, the second's items are shorter: a third of its time is
// their ends.  What bounds both is the expansion, 1500 clocks a stage against 1530 that the memory takes for it.  Small layers are
// bound by latency: two launches without weights to speak of take 13 us (of which staging the rows 2 to 3 a launch, finding the
// experts 0.7, the count of items and the last sums 2), one token through eighths of experts (25 MB) 21.  Not kept: weights
// straight into registers (16 warps, three steps deep: 570 us), two tiles a warp (620; the ring is then two stages deep), two CTAs
// of eight warps an SM (520), a warp of its own that counts items (500).
#include <algorithm>
#include <type_traits>

#include "fp4_math.cuh"
#include "fp4_rules.h"
#include "gemm_common.cuh"
#include "ptx_sm100.cuh"

namespace sglb200 {
namespace fp4 {

constexpr int kMoeConsumers = kMoeWarps * 32;  // threads that multiply
constexpr int kScaleWarps = 3;                // that fetch scales where K is not whole steps
// One more warp fetches codes, and scales where K is whole steps.
template <bool kWhole>
constexpr int kMoeThreads = kMoeConsumers + 32 + (kWhole ? 0 : kScaleWarps * 32);
constexpr int kMoeMaxExperts = 1024, kMoeMaxSlots = 1024;
constexpr int kMoeRows = 32;                  // activation rows per pass, at most: four times the eight columns of an instruction
// Columns of an instruction that an activation row takes: a float32 row has two, its terms.
template <typename T>
constexpr int kTerms = std::is_same<T, float>::value ? 2 : 1;
constexpr float kLoTerm = 0x1p-11f;           // the second term's unit in the first one's
constexpr uint32_t kTileBytes = 16 * kStep / 2;                  // of a tile and step
constexpr uint32_t kCodeBytes = kMoeWarps * kTileBytes;    // of a stage: 32 KB, and 4 or 5 KB of scales
// Scales of a row and step in a stage: 16 bytes, or the five words that hold them where rows begin on two bytes.
template <bool kWhole>
constexpr uint32_t kScalePitch = kWhole ? 16 : 20;
template <bool kWhole>
constexpr uint32_t kStageBytes = kCodeBytes + kMoeWarps * 16 * kScalePitch<kWhole>;
constexpr int kUsualShift = 6;                // rows whose largest magnitude lies in [2^-5, 2^9) are staged under 2^6

__device__ int g_fp4_moe_status = 0;  // 0 ok, 1 = a wait for weights expired

struct MoeParams {
  const void* x;            // up: [tokens, K] 16-bit; down: h [slots, K] float32
  const uint8_t* ws;        // [experts, rows, K / 16]
  const float* alpha;       // [experts] or nullptr
  const int32_t* ids;       // [slots]
  const float* weights;     // [slots] (down)
  float* h;                 // up: [slots, rows / 2]; down: products [slots, rows]
  void* out;                // down: [tokens, rows]
  int32_t* done;            // a counter per set of columns (zeroed by the up launch)
  int done_count;
  int64_t K, rows;          // rows of w: 2 I or H
  int slots, topk, experts, tokens;
  int steps;                // of K
  int warps_k;              // warps that split K; the others split tiles
  int sets;                 // items per pass
  int pass_rows;            // activation rows per pass
  int cols;                 // columns of an instruction that they take
  int stages;
  float factor;
  uint32_t wait_probes;
};

struct MoeCtl {
  uint64_t full[kMoeMaxStages], empty[kMoeMaxStages];
  uint16_t count[kMoeMaxExperts];   // slots of an expert, then where they begin
  uint16_t live[kMoeMaxSlots];      // passes: their expert, and where their slots begin (at most pass_rows of them each)
  uint16_t begin[kMoeMaxSlots + 1];
  uint16_t slot[kMoeMaxSlots];      // slots in experts' order
  int warp_sum[8];
  int amax[2][kMoeRows];            // largest magnitudes of the staged rows, as float bits; used in turn
  float factor[kMoeRows];           // of the staged rows: alpha (times the routing weight)
  int num_live, complete[2], abort_flag;  // num_live: passes
};

static_assert(sizeof(MoeCtl) == kMoeCtlBytes && kStageBytes<false> == kMoeStageBytes);

__device__ __forceinline__ int ld_fresh(const int32_t* at) {  // (past the first-level cache)
  int v;
  asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(at));
  return v;
}

// Which experts are named and by which slots, in passes of at most p.pass_rows slots; ids outside the experts are skipped.  All threads.
// (The order of the slots of an expert with one pass can depend on the order of atomics; it decides only which column of an instruction
// a slot takes, and columns do not mix.)
__device__ __forceinline__ void route(const MoeParams& p, MoeCtl* ctl) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (p.slots <= 32) {  // a slot a lane: its expert's slots are those lanes whose id is the same
    if (warp == 0) {
      const int id = lane < p.slots ? ld_fresh(p.ids + lane) : -1;
      const bool in = (uint32_t)id < (uint32_t)p.experts;
      const uint32_t same = __match_any_sync(0xffffffffu, in ? id : -1 - lane), before = (1u << lane) - 1;
      const bool first = in && (same & before) == 0;
      const int count = __popc(same), alone = first ? ((count + p.pass_rows - 1) / p.pass_rows << 16) + count : 0;  // (passes, slots)
      int incl = alone;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const int begin = __shfl_sync(0xffffffffu, incl - alone, in ? __ffs(same) - 1 : lane), rank = __popc(same & before);
      if (in) {
        const int at = (begin & 0xffff) + rank;
        ctl->slot[at] = (uint16_t)lane;
        if (rank % p.pass_rows == 0) {
          const int j = (begin >> 16) + rank / p.pass_rows;
          ctl->live[j] = (uint16_t)id;
          ctl->begin[j] = (uint16_t)at;
        }
      }
      if (lane == 31) {
        ctl->num_live = incl >> 16;
        ctl->begin[incl >> 16] = (uint16_t)(incl & 0xffff);
      }
    }
    __syncthreads();
    return;
  }
  constexpr int kRouters = 256, kIds = kMoeMaxSlots / kRouters, kExperts = kMoeMaxExperts / kRouters;
  uint32_t* count32 = reinterpret_cast<uint32_t*>(ctl->count);
  int place[kIds], id[kIds];
  if (tid < kRouters) {
#pragma unroll
    for (int j = 0; j < kIds; ++j) id[j] = tid + j * kRouters < p.slots ? ld_fresh(p.ids + tid + j * kRouters) : -1;
    for (int i = tid; i < kMoeMaxExperts / 2; i += kRouters) count32[i] = 0;
  }
  __syncthreads();
  if (tid < kRouters) {
#pragma unroll
    for (int j = 0; j < kIds; ++j) {
      if ((uint32_t)id[j] < (uint32_t)p.experts) {
        const uint32_t shift = (id[j] & 1) * 16;
        place[j] = (int)(atomicAdd(&count32[id[j] >> 1], 1u << shift) >> shift & 0xffffu);
      } else {
        id[j] = -1;
      }
    }
  }
  __syncthreads();
  // exclusive scan over the experts, four a thread: (passes, slots) packed
  int mine = 0, c[kExperts], incl = 0;
  if (tid < kRouters) {
#pragma unroll
    for (int k = 0; k < kExperts; ++k) {
      c[k] = ctl->count[tid * kExperts + k];
      mine += ((c[k] + p.pass_rows - 1) / p.pass_rows << 16) + c[k];
    }
    incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) ctl->warp_sum[warp] = incl;
  }
  __syncthreads();
  if (tid < kRouters) {
    int before = incl - mine;
    for (int w = 0; w < warp; ++w) before += ctl->warp_sum[w];
#pragma unroll
    for (int k = 0; k < kExperts; ++k) {
      ctl->count[tid * kExperts + k] = (uint16_t)(before & 0xffff);
      for (int r = 0; r < c[k]; r += p.pass_rows) {
        ctl->live[before >> 16] = (uint16_t)(tid * kExperts + k);
        ctl->begin[before >> 16] = (uint16_t)(before & 0xffff);
        before += (1 << 16) + min(c[k] - r, p.pass_rows);
      }
    }
    if (tid == kRouters - 1) {
      ctl->num_live = before >> 16;
      ctl->begin[before >> 16] = (uint16_t)(before & 0xffff);
    }
  }
  __syncthreads();
  bool split = false;  // a slot of this thread is of an expert of several passes
  int first[kIds], end[kIds];
  if (tid < kRouters) {
#pragma unroll
    for (int j = 0; j < kIds; ++j) {
      if (id[j] < 0) continue;
      first[j] = ctl->count[id[j]], end[j] = id[j] + 1 < kMoeMaxExperts ? ctl->count[id[j] + 1] : ctl->begin[ctl->num_live];
      ctl->slot[first[j] + place[j]] = (uint16_t)(tid + j * kRouters);
      split |= end[j] - first[j] > p.pass_rows;
    }
  }
  if (!__syncthreads_or(split)) return;
  // CTAs have to agree on the slots of such an expert's passes: those are put into ascending order.
  if (tid < kRouters) {
#pragma unroll
    for (int j = 0; j < kIds; ++j) {
      if (id[j] < 0 || end[j] - first[j] <= p.pass_rows) continue;
      place[j] = 0;
      for (int i = first[j]; i < end[j]; ++i) place[j] += ctl->slot[i] < tid + j * kRouters;
    }
  }
  __syncthreads();
  if (tid < kRouters) {
#pragma unroll
    for (int j = 0; j < kIds; ++j)
      if (id[j] >= 0) ctl->slot[first[j] + place[j]] = (uint16_t)(tid + j * kRouters);
  }
  __syncthreads();
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2, int c3, int c4) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
               : "memory");
}

// Barrier of the warps that multiply.
__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kMoeConsumers) : "memory"); }

__device__ __forceinline__ uint32_t lds_32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Where a slot's activations are: the token's row, or the slot's row of h.
template <typename T>
__device__ __forceinline__ const T* act_row(const MoeParams& p, int slot) {
  const int row = std::is_same<T, float>::value ? slot : slot / p.topk;
  return static_cast<const T*>(p.x) + (int64_t)row * p.K;
}

// Eight activations as they lie in memory, as float32, and the largest of their magnitudes' bits (NaN above infinity).
template <typename T>
struct Piece {
  uint32_t w[std::is_same<T, float>::value ? 8 : 4];
  __device__ __forceinline__ void load(const T* src) {
    const uint4 a = __ldcg(reinterpret_cast<const uint4*>(src));
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    if constexpr (std::is_same<T, float>::value) {
      const uint4 b = __ldcg(reinterpret_cast<const uint4*>(src) + 1);
      w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (uint32_t& v : w) v = 0;
  }
  __device__ __forceinline__ float2 pair(int i) const {  // values 2 i, 2 i + 1
    if constexpr (std::is_same<T, float>::value) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    if constexpr (std::is_same<T, __half>::value) return f16x2_to_f32(w[i]);
    return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  // two 16-bit maxima for bf16, one for float32
  __device__ __forceinline__ uint32_t most(uint32_t m) const {
#pragma unroll
    for (uint32_t v : w) m = std::is_same<T, float>::value ? max(m, v & 0x7fffffffu) : __vmaxu2(m, v & 0x7fff7fffu);
    return m;
  }
};

__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }
// The power of two under which a row with this largest magnitude is staged: the usual one, or the one that brings it into [2^14,
// 2^15); 1 where it is not finite.  fp16 rows are taken as they are.
template <typename T>
__device__ __forceinline__ int row_shift(int amax_bits) {
  if constexpr (std::is_same<T, __half>::value) return 0;
  const int e = min(amax_bits >> 23, 0xff);
  if (amax_bits == 0 || (e >= 127 - 5 && e < 127 + 9)) return kUsualShift;
  return e == 0xff ? 0 : min(max(14 + 127 - e, -126), 126);
}

// A piece as fp16 under the factor f.
template <typename T>
__device__ __forceinline__ uint4 to_f16(const Piece<T>& x, float f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value) {
      w[i] = x.w[i];
    } else {
      const float2 v = x.pair(i);
      const __half2 h = __floats2half2_rn(v.x * f, v.y * f);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// What that rounding left over, in units of kLoTerm: at most 2^14, as the first term is below 2^15.
template <typename T>
__device__ __forceinline__ uint4 rest_f16(const Piece<T>& x, float f, const uint4& first) {
  const uint32_t had[4] = {first.x, first.y, first.z, first.w};
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = x.pair(i), h = f16x2_to_f32(had[i]);
    const __half2 r = __floats2half2_rn(fmaf(v.x, f, -h.x) * (1.f / kLoTerm), fmaf(v.y, f, -h.y) * (1.f / kLoTerm));
    w[i] = *reinterpret_cast<const uint32_t*>(&r);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The first term of a row that is not finite, whose second one is zero: its finite values stay finite.
template <typename T>
__device__ __forceinline__ uint4 to_f16_clamped(const Piece<T>& x) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 v = x.pair(i);
    if (fabsf(v.x) < __int_as_float(0x7f800000)) v.x = fminf(fmaxf(v.x, -65504.f), 65504.f);
    if (fabsf(v.y) < __int_as_float(0x7f800000)) v.y = fminf(fmaxf(v.y, -65504.f), 65504.f);
    const __half2 h = __floats2half2_rn(v.x, v.y);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows [first, first + n) of the slots, as fp16 in the order in which lanes take them: 16-byte pieces of 8 columns of K, piece
// (step, jj, column, t) = columns step * 256 + t * 64 + jj * 8 ..; what is past K is zeros.  A row of two terms has them in neighbouring columns,
// or, where only one fits (`term` 0 or 1, else -1), that one in the row's column.  The multiplying warps, which share out the
// rows, several to a row where there are few; ends with a barrier.
template <typename T>
__device__ __noinline__ void stage_rows(const MoeParams& p, MoeCtl* ctl, int expert, int first, int n, int turn, int term, uint4* xs) {
  constexpr bool kTwo = kTerms<T> == 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int pieces = p.steps * 32, K = (int)p.K, pitch = p.cols * 4, row_pitch = kTwo && term < 0 ? 8 : 4;
  int* amax = ctl->amax[turn & 1];
  if (turn > 0) consumer_sync();  // the rows before these have been used
  if (tid < kMoeRows) ctl->amax[(turn + 1) & 1][tid] = 0;
  if (tid < n) {
    const float alpha = p.alpha ? __ldcg(p.alpha + expert) : 1.f;
    ctl->factor[tid] = std::is_same<T, float>::value ? alpha * __ldcg(p.weights + ctl->slot[first + tid]) : alpha;
  }
  const auto put = [&](int r, int q, const Piece<T>& x, float f, bool fine) {
    uint4* at = xs + ((q >> 5) * 8 + (q & 7)) * pitch + r * row_pitch + ((q >> 3) & 3);
    const uint4 hi = fine ? to_f16(x, f) : to_f16_clamped(x);
    if constexpr (kTwo) {
      const uint4 lo = fine ? rest_f16(x, f, hi) : make_uint4(0, 0, 0, 0);
      if (term < 0) at[4] = lo;
      *at = term == 1 ? lo : hi;
    } else {
      *at = hi;
    }
  };
  const int share = n > 8 ? 0 : n > 4 ? 1 : n > 2 ? 2 : n > 1 ? 3 : 4;  // 2^share warps to a row
  // (Four lanes take pieces that lie side by side in shared memory and eight lanes those of two jj, which fall on the same banks twice
  // at most; in the order of the columns it would be eight times.  1 to 3 % of a layer whose experts have many rows.)
  constexpr int kAhead = 2;  // pieces that are asked for before the first is converted (four: 2 us more a layer, for the instructions)
  for (int r = warp >> share; r < n; r += kMoeWarps >> share) {
    const T* src = act_row<T>(p, ctl->slot[first + r]);
    uint32_t most = 0;
#pragma unroll 1
    for (int q0 = (warp & ((1 << share) - 1)) * 32 + (lane & 3) * 8 + (lane >> 2); q0 < pieces; q0 += (kAhead * 32) << share) {
      Piece<T> x[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int q = q0 + ((k * 32) << share);
        if (q * 8 < K) x[k].load(src + q * 8); else x[k].zero();
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int q = q0 + ((k * 32) << share);
        if constexpr (!std::is_same<T, __half>::value) most = x[k].most(most);
        if (q < pieces) put(r, q, x[k], pow2(kUsualShift), true);
      }
    }
    if constexpr (!std::is_same<T, __half>::value) {
      if constexpr (!std::is_same<T, float>::value) most = max(most << 16, most & 0xffff0000u);
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0) atomicMax(&amax[r], (int)most);
    }
  }
  consumer_sync();
  if constexpr (!std::is_same<T, __half>::value) {
    bool again = false;
#pragma unroll 1
    for (int r = 0; r < n; ++r) {
      const int bits = amax[r], shift = row_shift<T>(bits);
      if (shift == kUsualShift) continue;
      again = true;
      const T* src = act_row<T>(p, ctl->slot[first + r]);
#pragma unroll 1
      for (int q = tid; q * 8 < K; q += kMoeConsumers) {
        Piece<T> x;
        x.load(src + q * 8);
        put(r, q, x, pow2(shift), bits < 0x7f800000);
      }
    }
    if (again) consumer_sync();  // (the same for all threads)
  }
}

// The tokens' slots of the columns [col0, col0 + cols), added in their order, by the CTA whose item was the last of those columns.
template <typename OutT>
__device__ __noinline__ void sum_slots(const MoeParams& p, int col0, int cols) {
  __threadfence();
  for (int j = threadIdx.x * 4; j < p.tokens * cols; j += kMoeConsumers * 4) {  // four columns a thread
    const int token = j / cols, col = col0 + j - token * cols;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < p.topk; k0 += 8) {  // eight slots are asked for before the first is added
      float4 v[8];
      int id[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int s = token * p.topk + min(k0 + k, p.topk - 1);
        v[k] = __ldcg(reinterpret_cast<const float4*>(p.h + (int64_t)s * p.rows + col)), id[k] = __ldcg(p.ids + s);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)  // (a slot of no expert has not been written)
        if (k0 + k < p.topk && (uint32_t)id[k] < (uint32_t)p.experts)
          sum[0] += v[k].x, sum[1] += v[k].y, sum[2] += v[k].z, sum[3] += v[k].w;
    }
    OutT o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = ElemTraits<OutT>::from_f32(sum[k] * p.factor);
    *reinterpret_cast<uint2*>(static_cast<OutT*>(p.out) + (int64_t)token * p.rows + col) = *reinterpret_cast<const uint2*>(o);
  }
}

// acc += weights of a step times the staged rows, 8 NT of them (`b`: this lane's pieces, `stride` apart).  185 instructions with the loads from
// shared memory, 64 of them conversions and 64 scalings, for 16 x 256 weights: an SM that does nothing else takes 8 TB/s of weights so
// (two tiles a warp, which share the pieces of x: 9, but half as many stages fit).
// A step's sums start from zero and are added in float32: the instructions cut off what does not fit their sum, and carried over all of 28
// steps that moved one bf16 output in 350 by a step (16 tokens, 8 of 256 of 7168 x 2048); now one in 4400, as float32 sums do.  It costs nothing
// with 8 columns, 1 to 2 % with 16 and 3 to 5 % with 32.
template <int NT>
__device__ __forceinline__ void multiply(float (&acc)[NT][4], const uint4 (&code)[2][2], const uint32_t (&scale)[2], const uint4* b, int stride) {
  float sum[NT][4];
#pragma unroll
  for (int q = 0; q < NT; ++q) sum[q][0] = sum[q][1] = sum[q][2] = sum[q][3] = 0.f;
  uint32_t s2[2][2];
#pragma unroll
  for (int u = 0; u < 2; ++u) s2[u][0] = cvt_f16x2_e4m3x2(scale[u]), s2[u][1] = cvt_f16x2_e4m3x2(scale[u] >> 16);
#pragma unroll
  for (int jj = 0; jj < 8; ++jj) {
    uint32_t a[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t s = __byte_perm(s2[u][jj >> 2], 0, (jj >> 1) & 1 ? 0x3232 : 0x1010);
      const uint4 c = code[u][jj >> 2];
      cvt_f16x2_e2m1x8((jj & 3) == 0 ? c.x : (jj & 3) == 1 ? c.y : (jj & 3) == 2 ? c.z : c.w, a[u]);
#pragma unroll
      for (int i = 0; i < 4; ++i) a[u][i] = hmul2(a[u][i], s);
    }
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      const uint4 x = b[jj * stride + q * 32];
      mma_f16(sum[q], a[0][0], a[1][0], a[0][1], a[1][1], x.x, x.y);
      mma_f16(sum[q], a[0][2], a[1][2], a[0][3], a[1][3], x.z, x.w);
    }
  }
#pragma unroll
  for (int q = 0; q < NT; ++q)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[q][j] += sum[q][j];
}

// kWhole: K is a multiple of a step.  kUp: T is the activations' type and a tile is 8 gate and the 8 matching up rows; else T is float
// (h) and OutT the output's type.  kTwice: both terms of a row of h do not fit, so an item takes K twice, first with the lesser ones.
template <typename T, typename OutT, bool kUp, bool kWhole, int NT, bool kTwice>
__global__ void __launch_bounds__(kMoeThreads<kWhole>, 1)
    fp4_experts_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_s,
                       const __grid_constant__ MoeParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint4* xs = reinterpret_cast<uint4*>(ring + p.stages * kStageBytes<kWhole>);
  float* red = reinterpret_cast<float*>(xs + p.steps * 32 * p.cols);  // [warp][values of a lane][32]
  MoeCtl* ctl = reinterpret_cast<MoeCtl*>(red + kMoeWarps * NT * 128);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t bar_full = ptx::smem_u32(ctl->full), bar_empty = ptx::smem_u32(ctl->empty);
  const int S = p.stages;

  if (tid == kMoeConsumers) {
    ptx::tma_prefetch_desc(&map_w);
    if constexpr (kWhole) ptx::tma_prefetch_desc(&map_s);
    for (int s = 0; s < S; ++s) ptx::mbar_init(bar_full + s * 8, kWhole ? 1 : 1 + kScaleWarps * 32), ptx::mbar_init(bar_empty + s * 8, kMoeWarps);
    ctl->abort_flag = 0;
    ptx::mbar_fence_init();
  }
  if (tid < kMoeRows) ctl->amax[0][tid] = 0;
  // The down launch may begin when every CTA of the up launch runs, which is after all that is in front of both: it finds its experts
  // and asks for its first weights, neither of which the up launch writes, before it waits for that.
  if constexpr (kUp) {
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
    if (blockIdx.x == 0)
      for (int i = tid; i < p.done_count; i += kMoeThreads<kWhole>) p.done[i] = 0;
  }
  route(p, ctl);

  const int warps_k = p.warps_k, warps_m = kMoeWarps / warps_k;
  const int tiles = (int)(p.rows / 16);  // of an expert (16 rows of w each)
  const int items = ctl->num_live * p.sets, turns = (p.steps + warps_k - 1) / warps_k, all_turns = kTwice ? 2 * turns : turns;
  // A CTA takes neighbouring items, which are mostly of one pass.
  const int each = (int)((uint32_t)items / gridDim.x), more = items - each * (int)gridDim.x;
  const int item0 = (int)blockIdx.x * each + min((int)blockIdx.x, more), item1 = item0 + each + ((int)blockIdx.x < more ? 1 : 0);

  if (warp == kMoeWarps) {
    // ------------------------------ weights ------------------------------
    if (ptx::elect_one()) {
      bool ok = true;
      int s = 0;                      // stage
      uint32_t ph = 1, part_bytes = warps_m * kTileBytes;  // (the first round of stages is free)
      for (int item = item0; item < item1 && ok; ++item) {
        const int live = item / p.sets, tile0 = (item - live * p.sets) * warps_m, expert = ctl->live[live];
        for (int i = 0, step0 = 0; i < all_turns; ++i) {
          ok = p.wait_probes != ptx::kProbesNone && ptx::mbar_wait_quiet(bar_empty + s * 8, ph);
          if (!ok) break;
          const uint32_t bar = bar_full + s * 8, at = ptx::smem_u32(ring) + s * kStageBytes<kWhole>;
          if constexpr (kWhole) {  // one load for the codes of all parts of K, one for their scales (a box is counted whole)
            ptx::mbar_arrive_expect_tx(bar, kStageBytes<kWhole>);
            if constexpr (kUp) {
              tma_load_5d(at, &map_w, bar, 0, tile0 * 8, 0, step0, expert);
              tma_load_5d(at + kCodeBytes, &map_s, bar, 0, tile0 * 8, 0, step0, expert);
            } else {
              tma_load_4d(at, &map_w, bar, 0, tile0 * 16, step0, expert);
              tma_load_4d(at + kCodeBytes, &map_s, bar, 0, tile0 * 16, step0, expert);
            }
          } else {
            const int parts = min(warps_k, p.steps - step0);
            ptx::mbar_arrive_expect_tx(bar, parts * part_bytes);
            for (int k = 0; k < parts; ++k) {
              if constexpr (kUp)
                tma_load_4d(at + k * part_bytes, &map_w, bar, (step0 + k) * (kStep / 2), tile0 * 8, 0, expert);
              else
                ptx::tma_load_3d(at + k * part_bytes, &map_w, bar, (step0 + k) * (kStep / 2), tile0 * 16, expert);
            }
          }
          step0 = kTwice && i + 1 == turns ? 0 : step0 + warps_k;
          if (++s == S) s = 0, ph ^= 1;
        }
      }
      if (!ok) ctl->abort_flag = 1;
    }
    __syncwarp();
    if constexpr (!kUp) ptx::grid_dependency_wait();
  } else if (!kWhole && warp > kMoeWarps) {
    // ------------------------------ scales, where their rows do not begin on 16 bytes ------------------------------
    // Words of four bytes by asynchronous copies, which arrive at the stage's barrier by themselves, so that they are as far ahead as the
    // codes are.  A row that begins on two bytes takes five words to a step.  Where such a warp has few issue slots beside those that multiply,
    // all that does not change from stage to stage is kept.  16 tokens, 8 of 256 experts of 7200 x 2080 take 660 us (whole steps, 7168 x
    // 2048: 475), 32 tokens, 8 of 128 of 2080 x 800 131 (91); when the warps that multiply loaded them, two steps ahead, 683 and 141; by
    // these through registers 840 and more.
    constexpr int kWords = kScalePitch<kWhole> / 4, kAll = kMoeWarps * 16 * kWords;
    constexpr int kTasks = (kAll + kScaleWarps * 32 - 1) / (kScaleWarps * 32);
    const int h = (warp - kMoeWarps - 1) * 32 + lane, scale_row = (int)(p.K / 16), half_rows = warps_m * 8;
    const int limit = kUp ? (int)(p.rows / 2) : (int)p.rows;  // rows of a half of w13, or of w2
    uint32_t from[kTasks];  // where a task's word lies, from the set's first row and the stage's first column
    int left_of[kTasks];    // bytes of the row from there on, for the first stage
    const auto row_of = [&](int j, int& k, int& u) {  // a task's row of the set, its part of K, its half
      const int r = (h + j * kScaleWarps * 32) / kWords, in = (k = r / (warps_m * 16), r - k * warps_m * 16);
      u = kUp ? in / half_rows : 0;
      return in - u * half_rows;
    };
#pragma unroll
    for (int j = 0; j < kTasks; ++j) {
      int k, u;
      const int row = row_of(j, k, u), word = (h + j * kScaleWarps * 32) % kWords, back = (row & 1) * (scale_row & 2);
      from[j] = (uint32_t)((row + u * limit) * scale_row + k * (kStep / 16) - back + word * 4);
      left_of[j] = scale_row - k * (kStep / 16) + back - word * 4;
    }
    bool ok = p.wait_probes != ptx::kProbesNone;
    int s = 0;
    uint32_t ph = 1;
    for (int item = item0; item < item1 && ok; ++item) {
      const int live = item / p.sets, tile_row = (item - live * p.sets) * warps_m * (kUp ? 8 : 16);
      const uint8_t* base = p.ws + ((int64_t)ctl->live[live] * p.rows + tile_row) * scale_row;
      uint32_t rows_there = 0;  // of the tasks' rows, those that the expert has
#pragma unroll
      for (int j = 0; j < kTasks; ++j) {
        int k, u;
        const int row = row_of(j, k, u);
        rows_there |= (h + j * kScaleWarps * 32 < kAll && tile_row + row < limit ? 1u : 0u) << j;
      }
      const bool all_there = tile_row + (kUp ? half_rows : warps_m * 16) <= limit;
      for (int i = 0, step0 = 0; i < all_turns; ++i) {
        ok = ok && (ptx::mbar_test(bar_empty + s * 8, ph) || ptx::mbar_wait_quiet(bar_empty + s * 8, ph));
        if (!ok) break;
        const uint32_t at = ptx::smem_u32(ring) + s * kStageBytes<kWhole> + kCodeBytes + h * 4;
        const uint8_t* src = base + step0 * (kStep / 16);
        const int used = step0 * (kStep / 16);
        if (all_there && used + warps_k * (kStep / 16) + 4 <= scale_row) {  // every word is whole
#pragma unroll
          for (int j = 0; j < kTasks; ++j)
            if (j < kAll / (kScaleWarps * 32) || h + j * kScaleWarps * 32 < kAll)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at + j * kScaleWarps * 128), "l"(src + from[j]) : "memory");
        } else {
#pragma unroll
          for (int j = 0; j < kTasks; ++j)
            if (h + j * kScaleWarps * 32 < kAll) {
              const int bytes = rows_there >> j & 1 ? min(max(left_of[j] - used, 0), 4) : 0;  // (the rest of a word is filled with zeros)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(at + j * kScaleWarps * 128),
                           "l"(bytes > 0 ? src + from[j] : p.ws), "r"(bytes)
                           : "memory");
            }
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar_full + s * 8) : "memory");
        step0 = kTwice && i + 1 == turns ? 0 : step0 + warps_k;
        if (++s == S) s = 0, ph ^= 1;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!ok) ctl->abort_flag = 1;
    if constexpr (!kUp) ptx::grid_dependency_wait();
  } else {
    // ------------------------------ products ------------------------------
    const int wk = warp % warps_k, wm = warp / warps_k;
    // this lane's codes in a stage: rows g and g + 8 of its tiles, pieces 2 t and 2 t + 1 of 128 swizzled bytes; a part of K has
    // its tiles' gate rows, then their up rows, or its tiles
    const uint32_t part = ptx::smem_u32(ring) + wk * warps_m * kTileBytes + g * 128;
    const uint32_t tile_step = kUp ? 8 * 128 : 16 * 128, row_step = kUp ? warps_m * 8 * 128 : 8 * 128;
    const uint32_t code_lo = part + wm * tile_step + ((uint32_t)(2 * t) ^ g) * 16;
    const uint32_t code_hi = part + wm * tile_step + ((uint32_t)(2 * t + 1) ^ g) * 16;
    const uint32_t row_a = (kUp ? wm * 8 : wm * 16) + g, row_b = row_a + (kUp ? warps_m * 8 : 8);
    const uint32_t scale_a = ptx::smem_u32(ring) + kCodeBytes + (wk * warps_m * 16 + row_a) * kScalePitch<kWhole> + t * 4;
    const uint32_t scale_b = scale_a + (row_b - row_a) * kScalePitch<kWhole>;
    const uint32_t halves = (g & 1) && p.K % 64 != 0 ? 0x5432 : 0x3210;  // of two words, where odd rows' scales begin in the middle of one
    const auto read_scales = [&](uint32_t at) {
      if constexpr (kWhole) return lds_32(at);
      return __byte_perm(lds_32(at), lds_32(at + 4), halves);
    };

    if constexpr (!kUp) ptx::grid_dependency_wait();
    const auto sum_set = [&](int set) {
      const int col0 = set * warps_m * 16;
      sum_slots<OutT>(p, col0, min(warps_m * 16, (int)p.rows - col0));
    };
    bool ok = p.wait_probes != ptx::kProbesNone;
    int staged = -1, stagings = 0, s = 0;
    uint32_t ph = 0;
    for (int item = item0; item < item1; ++item) {
      const int live = item / p.sets, set = item - live * p.sets;
      const int expert = ctl->live[live], first = ctl->begin[live], n = ctl->begin[live + 1] - first;
      const int my_tile = set * warps_m + wm;
      float acc[NT][4];
#pragma unroll
      for (int q = 0; q < NT; ++q) acc[q][0] = acc[q][1] = acc[q][2] = acc[q][3] = 0.f;
      const int stride = p.cols * 4, mine = (p.steps - wk + warps_k - 1) / warps_k;  // (the last turn may have no step for this warp)
      const auto take_all = [&](int term) {  // K of the staged rows, or of their one term
        if (kTwice || staged != live) {
          stage_rows<T>(p, ctl, expert, first, n, stagings, term, xs);
          ++stagings, staged = live;
        }
        // (columns without a row are not looked at: they read what lies there, or column 0 where less than eight fit)
        const uint4* b = xs + (wk * 8 * p.cols + (g < p.cols ? g : 0)) * 4 + t;
        const auto step = [&](bool mine) {
          if (ok && !ptx::mbar_test(bar_full + s * 8, ph)) ok = ptx::mbar_wait_quiet(bar_full + s * 8, ph);
          const uint32_t lo = code_lo + s * kStageBytes<kWhole>, hi = code_hi + s * kStageBytes<kWhole>;
          const uint4 code[2][2] = {{ptx::lds_128(lo), ptx::lds_128(hi)}, {ptx::lds_128(lo + row_step), ptx::lds_128(hi + row_step)}};
          const uint32_t scale[2] = {read_scales(scale_a + s * kStageBytes<kWhole>), read_scales(scale_b + s * kStageBytes<kWhole>)};
          __syncwarp();
          ptx::mbar_arrive_if(bar_empty + s * 8, lane == 0);
          if (++s == S) s = 0, ph ^= 1;
          if (mine) multiply<NT>(acc, code, scale, b, stride);
          b += warps_k * 8 * stride;
        };
        for (int i = 0; i < turns; i += 2) {
          step(i < mine);
          if (i + 1 < turns) step(i + 1 < mine);
        }
      };
      if constexpr (kTwice) {
        take_all(1);
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[q][j] *= kLoTerm;
        take_all(0);
      } else {
        take_all(-1);
      }
      // Lane (g, t) has rows g (acc 0, 1) and g + 8 (2, 3) of columns 2 t, 2 t + 1: of two activation rows, or both terms of one, which
      // are added here.  A warp of those that split K adds up kVals values of each of their lanes.
      constexpr bool kPairs = !kUp && !kTwice;
      constexpr int kVals = kPairs ? 1 : 2;  // activation rows of a lane and eight columns
      if constexpr (kPairs) {
#pragma unroll
        for (int q = 0; q < NT; ++q) acc[q][0] = fmaf(acc[q][1], kLoTerm, acc[q][0]), acc[q][1] = fmaf(acc[q][3], kLoTerm, acc[q][2]);
      }
      const auto finish = [&](int tile, int r, float lo, float hi) {
        if (tile >= tiles || r >= n) return;
        const float f = ctl->factor[r], unscale = pow2(-row_shift<T>(ctl->amax[(stagings - 1) & 1][r]));
        // The factor and the row's power of two together, which is exact, so that neither of them by itself takes a sum out of range; where
        // together they leave it, one after the other does not.
        const float both = f * unscale;
        const bool fits = fabsf(both) >= 0x1p-126f && fabsf(both) < __int_as_float(0x7f800000);
        const float a = fits ? both : f, b = fits ? 1.f : unscale;
        lo = lo * a * b, hi = hi * a * b;
        const int slot = ctl->slot[first + r];
        if constexpr (kUp) {
          p.h[(int64_t)slot * (p.rows / 2) + tile * 8 + g] = silu_mul(lo, hi);
        } else {
          float* at = p.h + (int64_t)slot * p.rows + tile * 16 + g;
          at[0] = lo, at[8] = hi;
        }
      };
      if (warps_k == 1) {
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
          for (int j = 0; j < kVals; ++j) finish(my_tile, kVals * (4 * q + t) + j, acc[q][j], acc[q][j + kVals]);
      } else {
        consumer_sync();  // (the sums before these have been read)
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
          for (int j = 0; j < 2 * kVals; ++j) red[((warp * NT + q) * 2 * kVals + j) * 32 + lane] = acc[q][j];
        consumer_sync();
        for (int i = tid; i < warps_m * NT * kVals * 32; i += kMoeConsumers) {
          const int j = (i >> 5) % kVals, q = (i >> 5) / kVals % NT, m = (i >> 5) / kVals / NT;  // (i % 32 == lane)
          float lo = 0.f, hi = 0.f;
          for (int k = 0; k < warps_k; ++k) {
            const float* at = red + (((m * warps_k + k) * NT + q) * 2 * kVals + j) * 32 + lane;
            lo += at[0], hi += at[kVals * 32];
          }
          finish(set * warps_m + m, kVals * (4 * q + t) + j, lo, hi);
        }
      }
      if constexpr (!kUp) {
        // One thread counts the item once everybody's products are on their way; what it learns is looked at behind the next
        // item's weights, so that nobody waits for it.
        consumer_sync();
        const bool sum = item > item0 && ctl->complete[(item - 1) & 1];
        if (tid == 0) {
          __threadfence();
          ctl->complete[item & 1] = atomicAdd(&p.done[set], 1) == ctl->num_live - 1;
        }
        if (sum) sum_set((item - 1) % p.sets);
      }
    }
    if constexpr (!kUp) {
      consumer_sync();
      if (item0 < item1 && ctl->complete[(item1 - 1) & 1]) sum_set((item1 - 1) % p.sets);
      if (items == 0)  // no expert is named: zeros
        for (int64_t i = (int64_t)blockIdx.x * kMoeConsumers + tid; i < (int64_t)p.tokens * p.rows; i += (int64_t)gridDim.x * kMoeConsumers)
          static_cast<OutT*>(p.out)[i] = ElemTraits<OutT>::from_f32(0.f);
    }
    if (!ok) ctl->abort_flag = 1;
  }
  __syncthreads();
  if (ctl->abort_flag != 0 && tid == 0) {
    atomicExch(&g_fp4_moe_status, 1);
    // give copies that may still be in flight time to land before the CTA's shared memory is released
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) {
    }
  }
}

static int plan_product(MoeParams& p, int64_t K, int64_t rows, bool up) {
  SGLB_REQUIRE(rows * (K / 16) < (1ll << 31), "fused_experts_fp4: %lld x %lld weights are too many for an expert", (long long)rows, (long long)K);
  const ExpertsPlan plan = plan_experts(p.slots, p.experts, K, rows, up, sm_count());
  SGLB_REQUIRE(plan.stages > 0, "fused_experts_fp4: %lld columns are too many", (long long)K);
  p.K = K, p.rows = rows, p.steps = plan.steps, p.cols = plan.cols, p.pass_rows = plan.pass_rows;
  p.warps_k = plan.warps_k, p.sets = plan.sets, p.stages = plan.stages;
  return SGLB200_OK;
}

template <typename T, typename OutT, bool kUp, bool kWhole, int NT, bool kTwice>
static int launch_experts(const CUtensorMap& map_w, const CUtensorMap& map_s, const MoeParams& p, cudaStream_t st) {
  auto kern = fp4_experts_kernel<T, OutT, kUp, kWhole, NT, kTwice>;
  static thread_local bool attr_set[64] = {false};  // the opt-in is per function and per device
  int dev = 0;
  SGLB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    SGLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMoeMostSmem));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t most = (int64_t)std::min(p.slots, p.experts + p.slots / p.pass_rows) * p.sets;
  const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, sm_count()));
  SGLB_CUDA(launch_pdl(kern, grid, kMoeThreads<kWhole>, (size_t)moe_smem(p.steps, p.cols, p.stages), st, map_w, map_s, p));
  return SGLB200_OK;
}

template <typename T, typename OutT, bool kUp>
static int launch_product(const void* w, const MoeParams& p, cudaStream_t st) {
  // Dimensions: bytes (of a step), rows, for w13 its two halves, steps where rows are whole ones, experts.
  const bool whole = p.K % kStep == 0;
  const uint64_t rows = (uint64_t)(kUp ? p.rows / 2 : p.rows);
  const uint32_t tile_rows = (uint32_t)((kUp ? 8 : 16) * (kMoeWarps / p.warps_k));
  const auto map_of = [&](const void* at, uint64_t row_bytes, uint32_t step_bytes, bool swizzled, CUtensorMap* out) {
    uint64_t dims[5] = {whole ? (uint64_t)step_bytes : row_bytes, rows}, strides[4] = {row_bytes};
    uint32_t box[5] = {step_bytes, tile_rows}, rank = 2;
    const auto add = [&](uint64_t n, uint64_t stride, uint32_t b) { dims[rank] = n, strides[rank - 1] = stride, box[rank++] = b; };
    if (kUp) add(2, rows * row_bytes, 2);
    if (whole) add((uint64_t)p.steps, step_bytes, (uint32_t)p.warps_k);
    add((uint64_t)p.experts, (uint64_t)p.rows * row_bytes, 1);
    return get_tile_map(at, rank, dims, strides, box, swizzled, out);
  };
  CUtensorMap map_w, map_s;
  int rc = map_of(w, (uint64_t)p.K / 2, kStep / 2, true, &map_w);
  if (rc) return rc;
  if (whole && (rc = map_of(p.ws, (uint64_t)p.K / 16, kStep / 16, false, &map_s)) != SGLB200_OK) return rc;
#define GO(NT, TWICE) return whole ? launch_experts<T, OutT, kUp, true, NT, TWICE>(map_w, map_s, p, st) \
                                   : launch_experts<T, OutT, kUp, false, NT, TWICE>(map_w, map_w, p, st)
  if constexpr (!kUp) {
    if (p.cols == 1) GO(1, true);
  }
  if (p.cols <= 8) GO(1, false);
  if (p.cols <= 16) GO(2, false);
  GO(4, false);
#undef GO
}

}  // namespace fp4

int fp4_moe_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, fp4::g_fp4_moe_status, sizeof(int)) != cudaSuccess) return -1;
  return v;
}
int fp4_moe_status_clear() {
  const int zero = 0;
  SGLB_CUDA(cudaMemcpyToSymbol(fp4::g_fp4_moe_status, &zero, sizeof(int)));
  return SGLB200_OK;
}

}  // namespace sglb200

using namespace sglb200;

extern "C" {

int64_t sglb200_fused_experts_fp4_workspace_bytes(int64_t tokens, int64_t topk, int64_t hidden, int64_t intermediate) {
  if (tokens <= 0 || topk <= 0 || hidden <= 0 || intermediate <= 0) return 0;
  const int64_t slots = tokens * topk;
  return (slots * intermediate + slots * hidden) * 4 + (hidden / 16 * 4 + 15) / 16 * 16;  // h, products, counters
}

int sglb200_fused_experts_fp4(const void* x, int dtype, const void* w13, const void* w13_scale, const float* w13_alpha, const void* w2,
                              const void* w2_scale, const float* w2_alpha, const float* topk_weights, const int32_t* topk_ids, void* out,
                              int64_t tokens, int64_t topk, int num_experts, int64_t hidden, int64_t intermediate, float factor,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype != 0 && dtype != 1) return fail(SGLB200_E_UNSUPPORTED, "fused_experts_fp4: activations must be bfloat16 or float16");
  SGLB_REQUIRE(tokens >= 0 && topk > 0 && hidden > 0 && intermediate > 0, "fused_experts_fp4: %lld tokens, topk %lld, hidden %lld, intermediate %lld",
               (long long)tokens, (long long)topk, (long long)hidden, (long long)intermediate);
  SGLB_REQUIRE(num_experts > 0 && num_experts <= fp4::kMoeMaxExperts, "fused_experts_fp4: %d experts (at most %d)", num_experts, fp4::kMoeMaxExperts);
  SGLB_REQUIRE(hidden % 32 == 0 && intermediate % 32 == 0, "fused_experts_fp4: hidden (%lld) and intermediate (%lld) must be divisible by 32",
               (long long)hidden, (long long)intermediate);
  SGLB_REQUIRE(tokens <= fp4::kMoeMaxSlots && topk <= fp4::kMoeMaxSlots && tokens * topk <= fp4::kMoeMaxSlots,
               "fused_experts_fp4: %lld tokens with %lld experts each: it is for at most %d of both together", (long long)tokens,
               (long long)topk, fp4::kMoeMaxSlots);
  if (tokens == 0) return SGLB200_OK;
  SGLB_REQUIRE(x && w13 && w13_scale && w2 && w2_scale && topk_weights && topk_ids && out, "fused_experts_fp4: null pointer");
  SGLB_REQUIRE(aligned16(x) && aligned16(w13) && aligned16(w13_scale) && aligned16(w2) && aligned16(w2_scale) && aligned16(out),
               "fused_experts_fp4: pointers must be 16-byte aligned");
  const int64_t need = sglb200_fused_experts_fp4_workspace_bytes(tokens, topk, hidden, intermediate);
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need)
    return fail(SGLB200_E_WORKSPACE, "fused_experts_fp4: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t slots = tokens * topk;
  float* h = static_cast<float*>(workspace);
  float* y = h + slots * intermediate;
  fp4::MoeParams p{};
  p.ids = topk_ids, p.weights = topk_weights;
  p.slots = (int)slots, p.topk = (int)topk, p.experts = num_experts, p.tokens = (int)tokens;
  p.done = reinterpret_cast<int32_t*>(y + slots * hidden), p.done_count = (int)(hidden / 16);
  p.factor = factor;
  p.wait_probes = g_gemm_wait_probes;
  p.x = x, p.ws = static_cast<const uint8_t*>(w13_scale), p.alpha = w13_alpha, p.h = h;
  int rc = fp4::plan_product(p, hidden, 2 * intermediate, true);
  fp4::MoeParams q = p;
  q.x = h, q.ws = static_cast<const uint8_t*>(w2_scale), q.alpha = w2_alpha, q.h = y, q.out = out;
  if (rc == SGLB200_OK) rc = fp4::plan_product(q, intermediate, hidden, false);
  if (rc != SGLB200_OK) return rc;
  rc = dtype == 0 ? fp4::launch_product<__nv_bfloat16, __nv_bfloat16, true>(w13, p, st) : fp4::launch_product<__half, __half, true>(w13, p, st);
  if (rc != SGLB200_OK) return rc;
  return dtype == 0 ? fp4::launch_product<float, __nv_bfloat16, false>(w2, q, st) : fp4::launch_product<float, __half, false>(w2, q, st);
}

}  // extern "C"
