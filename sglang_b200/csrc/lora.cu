// Low-rank adapters of many requests beside a shared projection:
//   out[t, n] = rnd( base[t, n] + scaling[l] * sum_{r < rank[l]} B[l, n, r] h[t, s(n) R + r] ),   h[t, j] = sum_k x[t, k] A[l, j, k],
// l the adapter that token t names (none: out = base) and s(n) the merged projection that column n belongs to.
//
// Up to three launches with programmatic serialization.  plan_kernel sorts the tokens by adapter into blocks (narrow.cuh); up to 64 tokens
// need none.  The narrow product gives h in float32.  expand_kernel adds the second product.
//
// h keeps 16 bits and more in the second product: the row's values times a power of two (float16 would overflow or lose small ones without it)
// enter as two 16-bit terms, 16 bits of bfloat16 or 22 of float16, there of values down to 2^-16 of the row's largest (split_row); the weights
// are what they are.  A rounding to one term would be off by 2^-9 of h, as much as the rounding of the output.
#include <algorithm>

#include "gemm_common.cuh"
#include "lora.cuh"
#include "narrow_rule.h"
#include "ptx_sm100.cuh"

namespace sglb200 {
namespace lora {

// ---- plan -----------------------------------------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

// One CTA.  The tokens of an adapter stay in their order, so that those of a long request lie one after the other.  Warp w takes the w-th part
// of the tokens and counts them by adapter in a row of its own; neighbours mostly name the same adapter, so that it counts equal ids at once.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const int32_t* __restrict__ ids, const int32_t* __restrict__ ranks, int R, int T,
                                                            int L, int block, int32_t* order,
                                                            int4* blocks, int most, int32_t* count) {
  extern __shared__ int32_t counts[];  // [32 warps][L + 1], [L + 1] tokens and [L + 1] blocks before an adapter's
  const int tid = threadIdx.x, lane = tid & 31, warp = ptx::warp_index(), keys = L + 1;
  int32_t *mine = counts + warp * keys, *tokens_before = counts + 32 * keys, *blocks_before = tokens_before + keys;
  for (int i = tid; i < 32 * keys; i += kPlanThreads) counts[i] = 0;
  __syncthreads();
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int part = (T + kPlanThreads - 1) / kPlanThreads * 32, shift = __ffs(block) - 1, begin = min(warp * part, T), end = min(begin + part, T);
  auto key_of = [&](int t) {  // (past the end: nobody's)
    const int id = t < end ? ids[t] : 0;
    return t >= end ? keys : id >= 0 && id < L ? id : L;
  };
  for (int t = begin; t < end; t += 32) {
    const int key = key_of(t + lane);
    const uint32_t same = __match_any_sync(0xffffffffu, key);
    if (key < keys && __ffs(same) - 1 == lane) mine[key] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int l = tid; l < keys; l += kPlanThreads) {  // every warp's tokens of an adapter begin behind the earlier warps'
    int sum = 0;
    for (int w = 0; w < 32; ++w) {
      const int n = counts[w * keys + l];
      counts[w * keys + l] = sum;
      sum += n;
    }
    tokens_before[l] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    int tokens = 0, before = 0;
    for (int at = 0; at < keys; at += 32) {
      const int l = at + lane, n = l < keys ? tokens_before[l] : 0, b = (n + block - 1) >> shift;
      int sn = n, sb = b;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int un = __shfl_up_sync(0xffffffffu, sn, off), ub = __shfl_up_sync(0xffffffffu, sb, off);
        if (lane >= off) sn += un, sb += ub;
      }
      if (l < keys) tokens_before[l] = tokens + sn - n, blocks_before[l] = before + sb - b;
      tokens += __shfl_sync(0xffffffffu, sn, 31), before += __shfl_sync(0xffffffffu, sb, 31);
    }
    for (int i = before + lane; i < most; i += 32) blocks[i] = make_int4(0, 0, -1, 0);
    if (lane == 0) *count = before;
  }
  __syncthreads();
  for (int l = warp; l < keys; l += 32) {
    const int used = l == L ? 0 : ranks != nullptr ? min(max(ranks[l], 0), R) : R;
    const int first = tokens_before[l], n = (l + 1 < keys ? tokens_before[l + 1] : T) - first;
    for (int i = lane; i * block < n; i += 32) {
      blocks[blocks_before[l] + i] = make_int4(first + i * block, min(block, n - i * block), l < L ? l : -1, used);
    }
  }
  for (int t = begin; t < end; t += 32) {
    const int key = key_of(t + lane);
    const uint32_t same = __match_any_sync(0xffffffffu, key);
    const int before = key < keys ? mine[key] : 0;
    __syncwarp();
    if (key < keys && __ffs(same) - 1 == lane) mine[key] = before + __popc(same);
    if (key < keys) order[tokens_before[key] + before + __popc(same & ((1u << lane) - 1))] = t + lane;
    __syncwarp();
  }
}

// ---- second product -------------------------------------------------------------------------------------------------------------------
constexpr int kWarps = 8;

// The units of 8 warps' columns of all blocks, columns fastest, are cut evenly over as many CTAs as run at once; a run is what a CTA has of one
// block and one merged projection.  kPairs: 32 values of the rank at most, which are two instructions; kTiles: groups of 8 columns of a warp.
// As a sum does not mind the order of its terms, a lane's 16 consecutive bytes of a weight row (and of a row of h alike) are its part of both
// instructions.  A lane holds the same two kTiles neighbouring columns of a token in all groups, so that base and out go by 4 kTiles bytes.
//
// Weights and base bound this kernel, and with few tokens a run's start: 64 tokens of 16 adapters beside 36864 columns take about 12 us, where the 48 MB
// would take 7.5.  They come by asynchronous copies, each lane's to a place of its own, kDepth - 1 steps (16 tokens of a
// unit) ahead, and before h is there.
template <int kPairs, int kTiles>
struct ExpandCfg {
  static constexpr int kWeights = kPairs * kTiles * 16 * kWarps * 32, kBase = kTiles * 8 * kWarps * 32;  // bytes of a unit, of a step
  static constexpr int kDepth = kPairs == 1 ? 4 : kPairs == 2 && kTiles == 4 ? 3 : 2;
  static constexpr int kRing = kDepth * (kWeights + kBase), kCols = 8 * kTiles * kWarps;
  static constexpr int kPitch = kPairs * 128 + 64;  // of a token's two terms: two rows of 64 bytes are read without a bank conflict
  static constexpr int kMostRows = (227 * 1024 - 4096 - kRing) / kPitch >= 128 ? 128 : 64;
  static_assert(kRing + kMostRows * kPitch <= 227 * 1024 - 4096);
};

template <typename T, int kPairs, int kTiles>
__global__ void __launch_bounds__(kWarps * 32, kPairs == 1 ? 3 : 2) expand_kernel(const Params p) {
  using Cfg = ExpandCfg<kPairs, kTiles>;
  constexpr int kCols = 8 * kTiles, kMine = 2 * kTiles, kDepth = Cfg::kDepth;
  extern __shared__ __align__(16) uint8_t ring[];  // [kDepth] units' weights, [kDepth] steps' base, then [rows][kPitch]
  uint8_t* terms = ring + Cfg::kRing;              // a token's high terms, then its low terms, 32 kPairs each
  __shared__ float unscale[narrow::kTileBlock];
  __shared__ int32_t token[narrow::kTileBlock];
  __shared__ int found[4];
  const int tid = threadIdx.x, lane = tid & 31, warp = ptx::warp_index(), g = lane >> 2, q = lane & 3;
  const bool scan = p.blocks.ids != nullptr;
  const int per = p.chunk0[p.S];  // units of a block
  const uint8_t* base = static_cast<const uint8_t*>(p.base);
  uint8_t* out = static_cast<uint8_t*>(p.out);
  const uint32_t weights_at = ptx::smem_u32(ring) + tid * 16, base_at = ptx::smem_u32(ring) + kDepth * Cfg::kWeights + tid * (4 * kTiles);
  constexpr uint32_t kChunk = kWarps * 32 * 16;
  bool waited = false;

  // The launch in front let this one in after its own wait for all that came before it, so only h is not there yet.
  // This CTA's units, and its block's tokens, rows and adapter to shared memory.
  int block = -1, begin = 0, end = 0;
  auto cut = [&](int blocks) { share(blocks * p.subs * per, begin, end); };
  auto pick = [&](const narrow::Scan& s, int which) {
    int n = 0, a = -1;
    narrow::scan_pick(s, which, p.sub, lane, token, n, a);
    if (lane == 0) found[1] = n, found[2] = a, found[3] = a < 0 ? 0 : p.ranks != nullptr ? min(max(__ldg(p.ranks + a), 0), p.R) : p.R;
  };
  auto find = [&](int which) {
    if (scan) {
      if (warp == 0) pick(narrow::scan_ids(p.blocks, p.sub, lane), which);
    } else {
      const int4 at = __ldcg(p.blocks.at + which);
      if (tid < at.y) token[tid] = __ldcg(p.blocks.order + at.x + tid);
      if (tid == 0) found[1] = at.y, found[2] = at.z, found[3] = at.w;
    }
  };
  if (!scan) {
    cut(__ldcg(p.blocks.count));
  } else {
    if (warp == 0) {  // (one warp looks at the tokens once for both)
      const narrow::Scan s = narrow::scan_ids(p.blocks, p.sub, lane);
      cut(s.blocks());
      if (begin < end) pick(s, begin / per);
      if (lane == 0) found[0] = s.blocks();
    }
    block = -2;  // found already
    __syncthreads();
    cut(found[0]);
  }
  int all_rows = 0, adapter = -1, used = 0;
  for (int at = begin; at < end;) {
    const int piece = at / per, unit0 = at - piece * per, row0 = piece % p.subs * p.sub;
    int slice = 0;
    while (slice + 1 < p.S && unit0 >= p.chunk0[slice + 1]) ++slice;
    const int units = min(p.chunk0[slice + 1] - unit0, end - at);
    at += units;
    if (piece / p.subs != block) {
      if (block != -2) {  // (else it has been found)
        __syncthreads();  // (nobody is at the run before this one any more)
        find(piece / p.subs);
        __syncthreads();
      }
      block = piece / p.subs;
      all_rows = found[1], adapter = found[2], used = found[3];
    } else {
      __syncthreads();
    }
    if (row0 >= all_rows || (adapter < 0 && p.in_place)) continue;
    const int rows = min(all_rows - row0, p.sub), steps = units * ((rows + 15) / 16);
    const int64_t stop = p.col0[slice + 1];
    const int64_t c0 = p.col0[slice] + (int64_t)(unit0 - p.chunk0[slice]) * Cfg::kCols + warp * kCols;
    const int pairs = (used + 31) / 32;
    const uint8_t* weights = static_cast<const uint8_t*>(p.b) + (adapter < 0 ? 0 : (int64_t)adapter * p.N * p.R * 2);

    // What a lane copies and stores, as far as it is the same for all units: its part of a weight row, the rows of the first 16 tokens.
    uint32_t part[kPairs];  // bytes that count (beyond the rank anything may stand: zeros instead)
#pragma unroll
    for (int s = 0; s < kPairs; ++s) part[s] = (uint32_t)min(max((used - s * 32 - q * 8) * 2, 0), 16);
    const uint32_t row_bytes = (uint32_t)p.R * 2;
    const uint8_t* next_weights = weights + (c0 + (g >> 1) * kMine + (g & 1)) * row_bytes + q * 16;
    auto row_of = [&](int m, int i) { return (int64_t)token[row0 + min(m + i * 8 + g, rows - 1)]; };
    const int64_t mine0 = c0 + q * kMine;
    const uint8_t *next_base0 = base + (row_of(0, 0) * p.ld_base + mine0) * 2, *next_base1 = base + (row_of(0, 1) * p.ld_base + mine0) * 2;
    uint8_t *to0 = out + (row_of(0, 0) * p.ld_out + mine0) * 2, *to1 = out + (row_of(0, 1) * p.ld_out + mine0) * 2;
    const bool tall = rows > 16;

    // The step that is asked for next: its unit, 16 tokens and places.
    int ahead_left = (int)min((int64_t)units * Cfg::kCols, stop - c0), ahead_m = 0;  // columns from the warp's first on
    int ahead_steps = steps;
    uint32_t weights_slot = weights_at, base_slot = base_at;
    auto fetch = [&]() {
      if (ahead_steps > 0) {
        --ahead_steps;
        if (ahead_m == 0) {
          if (ahead_left >= kCols) {
#pragma unroll
            for (int j = 0; j < kTiles; ++j)
#pragma unroll
              for (int s = 0; s < kPairs; ++s)
                if (s < pairs) ptx::cp_async_16(weights_slot + (s * kTiles + j) * kChunk, next_weights + j * 2 * row_bytes + s * 64, part[s]);
          } else {
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
              const bool on = (g >> 1) * kMine + j * 2 + (g & 1) < ahead_left;
#pragma unroll
              for (int s = 0; s < kPairs; ++s)
                if (s < pairs)
                  ptx::cp_async_16(weights_slot + (s * kTiles + j) * kChunk, on ? next_weights + j * 2 * row_bytes + s * 64 : weights, on ? part[s] : 0);
            }
          }
          next_weights += Cfg::kCols * row_bytes;
          weights_slot = weights_slot == weights_at + (kDepth - 1) * Cfg::kWeights ? weights_at : weights_slot + Cfg::kWeights;
        }
        if (p.vec && q * kMine < ahead_left) {
          const uint8_t *from0 = next_base0, *from1 = next_base1;
          if (ahead_m > 0) {
            from0 += (row_of(ahead_m, 0) - row_of(0, 0)) * p.ld_base * 2, from1 += (row_of(ahead_m, 1) - row_of(0, 1)) * p.ld_base * 2;
          }
          if (ahead_m + g < rows) {
            if constexpr (kTiles == 4) ptx::cp_async_16(base_slot, from0, 16);
            else ptx::cp_async_8(base_slot, from0);
          }
          if (ahead_m + 8 + g < rows) {
            if constexpr (kTiles == 4) ptx::cp_async_16(base_slot + Cfg::kBase / 2, from1, 16);
            else ptx::cp_async_8(base_slot + Cfg::kBase / 2, from1);
          }
        }
        base_slot = base_slot == base_at + (kDepth - 1) * Cfg::kBase ? base_at : base_slot + Cfg::kBase;
        if (tall && ahead_m + 16 < rows) {
          ahead_m += 16;
        } else {
          ahead_m = 0, ahead_left -= Cfg::kCols, next_base0 += Cfg::kCols * 2, next_base1 += Cfg::kCols * 2;
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kDepth - 1; ++i) fetch();
    if (!waited) {
      ptx::grid_dependency_wait();
      ptx::launch_dependents();
      waited = true;
    }
    const float scaling = adapter >= 0 && p.scalings != nullptr ? __ldg(p.scalings + adapter) : 1.f;
    // (two rows' loads at a time)
    for (int i = warp; i < rows && used > 0; i += 2 * kWarps) {
      float v[2][kPairs];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float* h = p.h + ((int64_t)token[row0 + min(i + u * kWarps, rows - 1)] * p.S + slice) * p.R;
#pragma unroll
        for (int j = 0; j < kPairs; ++j) v[u][j] = j * 32 + lane < used ? __ldcg(h + j * 32 + lane) * scaling : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row = i + u * kWarps;
        if (row >= rows) break;
        uint16_t* to = reinterpret_cast<uint16_t*>(terms + row * Cfg::kPitch);
        const float inv = split_row<T>(v[u], kPairs * 32, lane, [&](int r, uint16_t hi, uint16_t lo) { to[r] = hi, to[kPairs * 32 + r] = lo; });
        if (lane == 0) unscale[row] = inv;
      }
    }
    __syncthreads();

    int m = 0, left = (int)min((int64_t)units * Cfg::kCols, stop - c0);
    int64_t along = 0;  // of the unit, in bytes
    uint32_t from = weights_at, staged = base_at;
    for (int step = 0; step < steps; ++step) {
      fetch();
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      const int cols = max(0, min(kMine, left - q * kMine));
      const bool both = rows - m > 8;
      float acc[kTiles][4] = {};
      // (rows past the last are not written, and meet only their own sums)
      const uint8_t *pa = terms + (m + g) * Cfg::kPitch + q * 16, *pb = pa + 8 * Cfg::kPitch;
      const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int s = 0; s < kPairs; ++s) {
        if (s >= pairs) break;
        const uint4 ah = *reinterpret_cast<const uint4*>(pa + s * 64), al = *reinterpret_cast<const uint4*>(pa + kPairs * 64 + s * 64);
        const uint4 bh = both ? *reinterpret_cast<const uint4*>(pb + s * 64) : zero, bl = both ? *reinterpret_cast<const uint4*>(pb + kPairs * 64 + s * 64) : zero;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          const uint4 w = ptx::lds_128(from + (s * kTiles + j) * kChunk);
          ptx::mma_16816<std::is_same<T, __half>::value>(acc[j], al.x, bl.x, al.y, bl.y, w.x, w.y);
          ptx::mma_16816<std::is_same<T, __half>::value>(acc[j], al.z, bl.z, al.w, bl.w, w.z, w.w);
          ptx::mma_16816<std::is_same<T, __half>::value>(acc[j], ah.x, bh.x, ah.y, bh.y, w.x, w.y);
          ptx::mma_16816<std::is_same<T, __half>::value>(acc[j], ah.z, bh.z, ah.w, bh.w, w.z, w.w);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = m + g + 8 * i;
        if ((i == 0 || both) && r < rows && cols > 0) {
          uint8_t* to_bytes = (i == 0 ? to0 : to1) + along;
          if (m > 0) to_bytes += (row_of(m, i) - row_of(0, i)) * p.ld_out * 2;
          T* to = reinterpret_cast<T*>(to_bytes);
          uint32_t now[kTiles] = {};
          if (p.vec) {
            if constexpr (kTiles == 4) *reinterpret_cast<uint4*>(now) = ptx::lds_128(staged + i * (Cfg::kBase / 2));
            else *reinterpret_cast<uint2*>(now) = ptx::lds_64(staged + i * (Cfg::kBase / 2));
          } else {
            const T* had = reinterpret_cast<const T*>(base + (row_of(m, i) * p.ld_base + mine0) * 2 + along);
#pragma unroll
            for (int j = 0; j < kMine; ++j)
              if (j < cols) now[j / 2] |= (uint32_t)bits(had[j]) << (j % 2 * 16);
          }
          if (used > 0) {
            const float inv = unscale[r];
#pragma unroll
            for (int j = 0; j < kTiles; ++j) {
              float2 was = unpack2<T>(now[j]);
              ptx::fma2(was.x, was.y, __float_as_uint(acc[j][2 * i]), __float_as_uint(acc[j][2 * i + 1]), inv);
              now[j] = pack2<T>(was.x, was.y);
            }
          }
          if (p.vec) {
            if constexpr (kTiles == 4)
              *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(now);
            else
              *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(now);
          } else {
#pragma unroll
            for (int j = 0; j < kMine; ++j)
              if (j < cols) {
                const uint16_t v = (uint16_t)(now[j / 2] >> (j % 2 * 16));
                to[j] = *reinterpret_cast<const T*>(&v);
              }
          }
        }
      }
      staged = staged == base_at + (kDepth - 1) * Cfg::kBase ? base_at : staged + Cfg::kBase;
      m += 16;
      if (m >= rows) {
        m = 0, left -= Cfg::kCols, along += Cfg::kCols * 2;
        from = from == weights_at + (kDepth - 1) * Cfg::kWeights ? weights_at : from + Cfg::kWeights;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  if (!waited) ptx::grid_dependency_wait();  // (no CTA ends before the launch in front: the one behind counts on that)
}

template <typename T, int kPairs, int kTiles>
static int launch_expand(Params& p, int block, cudaStream_t st) {
  using Cfg = ExpandCfg<kPairs, kTiles>;
  int units = 0;
  for (int s = 0; s < p.S; ++s) {
    p.chunk0[s] = units;
    units += (int)((p.col0[s + 1] - p.col0[s] + Cfg::kCols - 1) / Cfg::kCols);
  }
  p.chunk0[p.S] = units;
  p.sub = std::min(block, Cfg::kMostRows);
  // Few tokens and few columns: blocks of fewer rows, so that every SM has some.  (With a plan that would leave empty ones.)
  if (p.blocks.ids != nullptr)
    while (p.sub > 16 && (int64_t)units * ((p.blocks.ids_rows + p.sub - 1) / p.sub) < 2 * sm_count()) p.sub /= 2;
  p.subs = p.blocks.ids != nullptr ? 1 : block / p.sub;
  const size_t smem = (size_t)(Cfg::kRing + p.sub * Cfg::kPitch);
  const int64_t all = (int64_t)units * (p.blocks.ids != nullptr ? p.max_blocks + p.blocks.ids_rows / p.sub : p.max_blocks * p.subs), at_once = std::min<int64_t>(4, 227 * 1024 / (int64_t)(smem + 3072)) * sm_count();
  SGLB_REQUIRE(all < (1ll << 31), "lora_add: %lld tiles are too many", (long long)all);
  auto kern = expand_kernel<T, kPairs, kTiles>;
  static thread_local bool attr_set[64] = {false};  // the opt-in is per function and per device
  int dev = 0;
  SGLB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    SGLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kRing + Cfg::kMostRows * Cfg::kPitch));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  SGLB_CUDA(launch_pdl(kern, (unsigned)std::min(all, at_once), kWarps * 32, smem, st, p));
  return SGLB200_OK;
}

template <typename T>
static int expand(Params& p, int block, cudaStream_t st) {
  if (p.R <= 32) return launch_expand<T, 1, 4>(p, block, st);
  if (p.R <= 64) return launch_expand<T, 2, 4>(p, block, st);
  if (p.R <= 128) return launch_expand<T, 4, 4>(p, block, st);
  return launch_expand<T, 8, 2>(p, block, st);
}

// Every adapter (and "none") has at most one block that is not full.
static int64_t most_blocks(int64_t T, int L, int block) {
  const int64_t named = T < L + 1 ? T : L + 1;
  return T <= block ? named : T / block + named;
}
// Whether two arrays of 16-bit rows are one and the same or have no byte in common (rows of different strides: no byte between their ends).
static bool apart(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t rows, int64_t n) {
  const int64_t d = (int64_t)((intptr_t)b - (intptr_t)a);  // bytes
  if (d == 0 && (lda == ldb || rows == 1)) return true;
  if (d >= ((rows - 1) * lda + n) * 2 || -d >= ((rows - 1) * ldb + n) * 2) return true;
  const int64_t within = (d % (lda * 2) + lda * 2) % (lda * 2);  // where in a row of a one of b begins
  return lda == ldb && rows > 1 && within >= n * 2 && within <= (lda - n) * 2;
}
static int64_t up(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace lora
}  // namespace sglb200

using namespace sglb200;

extern "C" int64_t sglb200_lora_add_workspace_bytes(int64_t tokens, int num_adapters, int rank, int num_slices) {
  if (tokens <= 0 || num_adapters < 1 || rank < 1 || num_slices < 1) return 0;
  // (whichever blocks the call takes)
  const int64_t blocks = tokens / narrow::kSmallBlock + num_adapters + 1;
  return lora::up(4 * tokens) + lora::up(16 * blocks + 4) + lora::up(4 * tokens * num_slices * rank);
}

extern "C" int sglb200_lora_add(const void* x, const void* lora_a, const void* lora_b, const void* base, void* out, int dtype,
                                const int32_t* adapter_ids, const float* scalings, const int32_t* ranks, int64_t tokens, int num_adapters,
                                int rank, int64_t N, int64_t K, int64_t x_stride, int64_t base_stride, int64_t out_stride, int num_slices,
                                const int64_t* slice_sizes, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype != 0 && dtype != 1) return fail(SGLB200_E_UNSUPPORTED, "lora_add: dtype %d (0 bf16, 1 fp16)", dtype);
  SGLB_REQUIRE(tokens >= 0 && num_adapters >= 1 && rank >= 1 && N >= 1 && K >= 1 && num_slices >= 1,
               "lora_add: %lld tokens, %d adapters, rank %d, N %lld, K %lld, %d slices", (long long)tokens, num_adapters, rank, (long long)N,
               (long long)K, num_slices);
  if (num_adapters > lora::kMaxAdapters || rank > lora::kMaxRank || rank % 8 != 0 || num_slices > lora::kMaxSlices)
    return fail(SGLB200_E_UNSUPPORTED, "lora_add: %d adapters, rank %d, %d slices (at most %d, a multiple of 8 up to %d, %d)", num_adapters,
                rank, num_slices, lora::kMaxAdapters, lora::kMaxRank, lora::kMaxSlices);
  SGLB_REQUIRE(K % 8 == 0 && x_stride % 8 == 0 && x_stride >= K, "lora_add: K (%lld) and x's row stride (%lld) must be divisible by 8",
               (long long)K, (long long)x_stride);
  SGLB_REQUIRE(base_stride >= N && out_stride >= N, "lora_add: row strides %lld and %lld of %lld columns", (long long)base_stride,
               (long long)out_stride, (long long)N);
  SGLB_REQUIRE(tokens < (1ll << 31) - 65536 && N < (1ll << 31) - 65536 && K <= 1 << 20, "lora_add: %lld tokens, N %lld or K %lld is too large",
               (long long)tokens, (long long)N, (long long)K);
  SGLB_REQUIRE(std::max({x_stride, base_stride, out_stride}) < std::min<int64_t>(1ll << 40, (1ll << 60) / std::max<int64_t>(tokens, 1)), "lora_add: row strides %lld, %lld or %lld are too large",
               (long long)x_stride, (long long)base_stride, (long long)out_stride);
  SGLB_REQUIRE(slice_sizes != nullptr, "lora_add: null slice_sizes");
  lora::Params p{};
  int64_t columns = 0;
  bool even = true;
  for (int s = 0; s < num_slices; ++s) {
    SGLB_REQUIRE(slice_sizes[s] >= 1, "lora_add: slice %d has %lld columns", s, (long long)slice_sizes[s]);
    SGLB_REQUIRE(slice_sizes[s] <= N - columns, "lora_add: the slices have more than %lld columns", (long long)N);
    p.col0[s] = columns;
    even = even && columns % 8 == 0;
    columns += slice_sizes[s];
  }
  p.col0[num_slices] = columns;
  SGLB_REQUIRE(columns == N, "lora_add: the slices have %lld columns of %lld", (long long)columns, (long long)N);
  if (tokens == 0) return SGLB200_OK;
  SGLB_REQUIRE(x && lora_a && lora_b && base && out && adapter_ids, "lora_add: null pointer");
  SGLB_REQUIRE(aligned16(x) && aligned16(lora_a) && aligned16(lora_b), "lora_add: x, lora_a and lora_b must be 16-byte aligned");
  SGLB_REQUIRE(((uintptr_t)base & 1) == 0 && ((uintptr_t)out & 1) == 0, "lora_add: base and out must be aligned to 2 bytes");
  SGLB_REQUIRE(lora::apart(base, base_stride, out, out_stride, tokens, N), "lora_add: out overlaps base and is not base");
  const int64_t bytes = sglb200_lora_add_workspace_bytes(tokens, num_adapters, rank, num_slices);
  if (workspace == nullptr || workspace_bytes < bytes || !aligned16(workspace))
    return fail(SGLB200_E_WORKSPACE, "lora_add: %lld bytes of workspace are needed, aligned to 16", (long long)bytes);
  const bool scan = tokens <= narrow::kScanRows;
  const int block = scan || narrow::small_adapter_blocks(tokens, num_slices, rank, K, N) ? narrow::kSmallBlock : narrow::kTileBlock;
  const int64_t blocks = lora::most_blocks(tokens, num_adapters, block);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int32_t* order = static_cast<int32_t*>(workspace);
  int4* at = reinterpret_cast<int4*>(static_cast<uint8_t*>(workspace) + lora::up(4 * tokens));
  int32_t* count = reinterpret_cast<int32_t*>(at + blocks);
  float* h = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(at) + lora::up(16 * blocks + 4));
  if (scan) {
    p.blocks.ids = adapter_ids, p.blocks.ids_rows = (int)tokens, p.blocks.adapters = num_adapters;
  } else {
    p.blocks = {order, at, count, nullptr, 0, 0};
    const size_t smem = (size_t)34 * (num_adapters + 1) * sizeof(int32_t);
    if (smem > 48 * 1024) {
      static thread_local bool attr_set[64] = {false};  // the opt-in is per function and per device
      int dev = 0;
      SGLB_CUDA(cudaGetDevice(&dev));
      if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        SGLB_CUDA(cudaFuncSetAttribute(lora::plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       34 * (lora::kMaxAdapters + 1) * (int)sizeof(int32_t)));
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
      }
    }
    SGLB_CUDA(launch_pdl(lora::plan_kernel, 1u, (unsigned)lora::kPlanThreads, smem, st, adapter_ids, ranks, rank, (int)tokens, num_adapters, block, order,
                         at, (int)blocks, count));
  }
  narrow::Params n{};
  n.x = x, n.w = lora_a, n.y = h, n.ranks = ranks, n.blocks = p.blocks;
  n.T = tokens, n.N = (int64_t)num_slices * rank, n.K = K, n.ldx = x_stride, n.rank_rows = rank, n.adapters = num_adapters, n.block = block;
  int rc = narrow::product(n, dtype, blocks, st);
  if (rc) return rc;
  p.b = lora_b, p.base = base, p.out = out, p.h = h, p.scalings = scalings, p.ranks = ranks;
  p.N = N, p.ld_base = base_stride, p.ld_out = out_stride, p.R = rank, p.S = num_slices, p.max_blocks = (int)blocks;
  p.in_place = base == out;
  p.vec = even && N % 8 == 0 && base_stride % 8 == 0 && out_stride % 8 == 0 && aligned16(base) && aligned16(out);
  p.wait_probes = g_gemm_wait_probes;
  // (its row pitches are 32-bit numbers of bytes)
  if (block == narrow::kTileBlock && p.vec && rank <= lora::kTileRank && base_stride < 1ll << 30 && out_stride < 1ll << 30)
    return lora::expand_tile(p, dtype, st);
  const int rows = tokens <= 16 ? 16 : tokens <= 32 ? 32 : scan ? narrow::kScanRows : block;  // the most that a block can have
  return dtype == 0 ? lora::expand<__nv_bfloat16>(p, rows, st) : lora::expand<__half>(p, rows, st);
}
