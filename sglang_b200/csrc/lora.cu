// Low-rank adapters of many requests beside a shared projection:
//   out[t, n] = rnd( base[t, n] + scaling[l] * sum_{r < rank[l]} B[l, n, r] h[t, s(n) R + r] ),   h[t, j] = sum_k x[t, k] A[l, j, k],
// l the adapter that token t names (none: out = base) and s(n) the merged projection that column n belongs to.
//
// Up to three launches with programmatic serialization.  plan_kernel sorts the tokens by adapter into blocks (narrow.cuh); up to 64 tokens
// need none.  The narrow product gives h in float32.  expand_kernel adds the second product.
//
// h keeps 16 bits and more in the second product: the row's values times a power of two that brings the largest to [1, 2) (float16 would
// overflow or lose small ones without it) enter as two 16-bit terms, 16 bits of bfloat16 or 22 of float16; the weights are what they are.
// A rounding to one term would be off by 2^-9 of h, as much as the rounding of the output.
#include <algorithm>

#include "gemm_common.cuh"
#include "lora.cuh"
#include "ptx_sm100.cuh"

namespace sglb200 {
namespace lora {

// ---- plan -----------------------------------------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

// One CTA.  The tokens of an adapter stay in their order, so that those of a long request lie one after the other.  Warp w takes the w-th part
// of the tokens and counts them by adapter in a row of its own; neighbours mostly name the same adapter, so that it counts equal ids at once.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const int32_t* __restrict__ ids, int T, int L, int block, int32_t* order,
                                                            int32_t* start, int32_t* rows, int32_t* adapter, int32_t* count) {
  extern __shared__ int32_t counts[];  // [32 warps][L + 1], [L + 1] tokens and [L + 1] blocks before an adapter's
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, keys = L + 1;
  int32_t *mine = counts + warp * keys, *tokens_before = counts + 32 * keys, *blocks_before = tokens_before + keys;
  for (int i = tid; i < 32 * keys; i += kPlanThreads) counts[i] = 0;
  __syncthreads();
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int part = (T + kPlanThreads - 1) / kPlanThreads * 32, begin = min(warp * part, T), end = min(begin + part, T);
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
    int tokens = 0, blocks = 0;
    for (int at = 0; at < keys; at += 32) {
      const int l = at + lane, n = l < keys ? tokens_before[l] : 0, b = (n + block - 1) / block;
      int sn = n, sb = b;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int un = __shfl_up_sync(0xffffffffu, sn, off), ub = __shfl_up_sync(0xffffffffu, sb, off);
        if (lane >= off) sn += un, sb += ub;
      }
      if (l < keys) tokens_before[l] = tokens + sn - n, blocks_before[l] = blocks + sb - b;
      tokens += __shfl_sync(0xffffffffu, sn, 31), blocks += __shfl_sync(0xffffffffu, sb, 31);
    }
    if (lane == 0) *count = blocks;
  }
  __syncthreads();
  for (int l = warp; l < keys; l += 32) {
    const int first = tokens_before[l], n = (l + 1 < keys ? tokens_before[l + 1] : T) - first;
    for (int i = lane; i * block < n; i += 32) {
      const int b = blocks_before[l] + i;
      start[b] = first + i * block;
      rows[b] = min(block, n - i * block);
      adapter[b] = l < L ? l : -1;
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

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A CTA takes up to `sub` rows of a block and `passes` times 8 warps' columns.  kPairs: 32 values of the rank at most, which are two
// instructions; kTiles: groups of 8 columns of a warp.  As a sum does not mind the order of its terms, a lane's 16 consecutive bytes of a weight
// row (and of a row of h alike) are its part of both.  A lane holds the same two kTiles neighbouring columns of a token in all groups, so that
// base and out go by 4 kTiles bytes.  Weights, and base of the first 16 rows, come by asynchronous copies, each lane's to a place of its own,
// kDepth - 1 passes ahead and before h is there: they are what bounds this kernel where few tokens name an adapter.
template <int kPairs, int kTiles>
struct ExpandCfg {
  static constexpr int kLane = kPairs * kTiles * 16 + kTiles * 8;  // bytes of a lane and pass
  static constexpr int kDepth = kPairs == 1 ? 4 : kPairs == 2 && kTiles == 4 ? 3 : 2;
  static constexpr int kStage = kLane * kWarps * 32, kCols = 8 * kTiles * kWarps;
  static constexpr int kPitch = kPairs * 128 + 64;  // of a token's two terms: two rows of 64 bytes are read without a bank conflict
  static constexpr int kMostRows = (227 * 1024 - 4096 - kDepth * kStage) / kPitch >= 128 ? 128 : 64;
  static_assert(kDepth * kStage + kMostRows * kPitch <= 227 * 1024 - 4096);
};

template <typename T, int kPairs, int kTiles>
__global__ void __launch_bounds__(kWarps * 32) expand_kernel(const Params p) {
  using Cfg = ExpandCfg<kPairs, kTiles>;
  constexpr int kCols = 8 * kTiles, kMine = 2 * kTiles, kDepth = Cfg::kDepth;
  extern __shared__ __align__(16) uint8_t tile[];  // [kDepth] stages, then [rows of a CTA][kPitch]
  uint8_t* terms = tile + kDepth * Cfg::kStage;    // a token's high terms, then its low terms, 32 kPairs each
  __shared__ float unscale[narrow::kTileBlock];
  __shared__ int32_t token[narrow::kTileBlock];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
  const int piece = (int)(blockIdx.x % (p.max_blocks * p.subs)), block = piece / p.subs, row0 = piece % p.subs * p.sub;
  const int chunk = (int)(blockIdx.x / (p.max_blocks * p.subs));
  // The launch in front let this one in after its own wait for all that came before it, so only h is not there yet.
  int rows, adapter;
  if (p.blocks.ids != nullptr) {
    if (warp == 0) {
      int n = 0, a = -1;
      const bool there = narrow::scan_block(p.blocks, block, lane, token, n, a);
      if (lane == 0) found[0] = there ? n : 0, found[1] = a;
    }
    __syncthreads();
    rows = found[0], adapter = found[1];
  } else {
    if (block >= __ldcg(p.blocks.count)) return;
    adapter = __ldcg(p.blocks.adapter + block);
    const int start = __ldcg(p.blocks.start + block);
    rows = __ldcg(p.blocks.rows + block);
    if (tid < rows) token[tid] = __ldcg(p.blocks.order + start + tid);
    __syncthreads();
  }
  if (row0 >= rows || (adapter < 0 && p.in_place)) return;
  rows = min(rows - row0, p.sub);
  int slice = 0;
  while (slice + 1 < p.S && chunk >= p.chunk0[slice + 1]) ++slice;
  const int64_t end = p.col0[slice + 1];
  const int64_t c0 = p.col0[slice] + (int64_t)(chunk - p.chunk0[slice]) * p.passes * Cfg::kCols + warp * kCols;
  const int passes = c0 < end ? (int)min((int64_t)p.passes, (end - c0 + Cfg::kCols - 1) / Cfg::kCols) : 0;
  const int used = adapter < 0 ? 0 : p.ranks != nullptr ? min(max(__ldg(p.ranks + adapter), 0), p.R) : p.R;
  const int pairs = (used + 31) / 32;
  const uint8_t* weights = static_cast<const uint8_t*>(p.b) + (adapter < 0 ? 0 : (int64_t)adapter * p.N * p.R * 2);
  const T* base = static_cast<const T*>(p.base);
  T* out = static_cast<T*>(p.out);
  const int64_t ta = token[row0 + min(g, rows - 1)], tb = token[row0 + min(g + 8, rows - 1)];
  const uint32_t mine_at = ptx::smem_u32(tile) + tid * 16;  // (chunk i of a stage at i times 16 bytes of all threads)
  constexpr uint32_t kChunk = kWarps * 32 * 16;

  auto fetch = [&](int pass) {
    if (pass < passes) {
      const int64_t c = c0 + (int64_t)pass * Cfg::kCols;
      const uint32_t to = mine_at + pass % kDepth * Cfg::kStage;
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        const int64_t n = c + (g >> 1) * kMine + j * 2 + (g & 1);
        const uint8_t* from = weights + (n < end ? n : c) * p.R * 2 + q * 16;
#pragma unroll
        for (int s = 0; s < kPairs; ++s)
          if (s < pairs) {  // (beyond the rank anything may stand: zeros instead)
            const int there = n < end ? min(max((used - s * 32 - q * 8) * 2, 0), 16) : 0;
            ptx::cp_async_16(to + (s * kTiles + j) * kChunk, there > 0 ? from + s * 64 : weights, there);
          }
      }
      if (p.vec) {
        const int64_t n = c + q * kMine;
        const uint32_t base_to = ptx::smem_u32(tile) + pass % kDepth * Cfg::kStage + kPairs * kTiles * kChunk;
        if (n < end) {
          if constexpr (kTiles == 4) {
            if (g < rows) ptx::cp_async_16(base_to + tid * 16, base + ta * p.ld_base + n, 16);
            if (g + 8 < rows) ptx::cp_async_16(base_to + kChunk + tid * 16, base + tb * p.ld_base + n, 16);
          } else {
            if (g < rows) ptx::cp_async_8(base_to + tid * 8, base + ta * p.ld_base + n);
            if (g + 8 < rows) ptx::cp_async_8(base_to + kChunk / 2 + tid * 8, base + tb * p.ld_base + n);
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kDepth - 1; ++i) fetch(i);
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
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
      uint16_t* at = reinterpret_cast<uint16_t*>(terms + row * Cfg::kPitch);
      const float inv = split_row<T>(v[u], kPairs * 32, lane, [&](int r, uint16_t hi, uint16_t lo) { at[r] = hi, at[kPairs * 32 + r] = lo; });
      if (lane == 0) unscale[row] = inv;
    }
  }
  __syncthreads();

  for (int pass = 0; pass < passes; ++pass) {
    fetch(pass + kDepth - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
    const uint32_t from = mine_at + pass % kDepth * Cfg::kStage;
    const int64_t mine = c0 + (int64_t)pass * Cfg::kCols + q * kMine;
    const int cols = (int)max((int64_t)0, min((int64_t)kMine, end - mine));
    for (int m = 0; m < rows; m += 16) {
      float acc[kTiles][4] = {};
      // (rows past the last are not written, and meet only their own sums)
      const uint8_t *pa = terms + (m + g) * Cfg::kPitch + q * 16, *pb = pa + 8 * Cfg::kPitch;
#pragma unroll
      for (int s = 0; s < kPairs; ++s) {
        if (s >= pairs) break;
        const uint4 ah = *reinterpret_cast<const uint4*>(pa + s * 64), bh = *reinterpret_cast<const uint4*>(pb + s * 64);
        const uint4 al = *reinterpret_cast<const uint4*>(pa + kPairs * 64 + s * 64), bl = *reinterpret_cast<const uint4*>(pb + kPairs * 64 + s * 64);
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          const uint4 w = ptx::lds_128(from + (s * kTiles + j) * kChunk);
          mma16816<T>(acc[j], al.x, bl.x, al.y, bl.y, w.x, w.y);
          mma16816<T>(acc[j], al.z, bl.z, al.w, bl.w, w.z, w.w);
          mma16816<T>(acc[j], ah.x, bh.x, ah.y, bh.y, w.x, w.y);
          mma16816<T>(acc[j], ah.z, bh.z, ah.w, bh.w, w.z, w.w);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = m + g + 8 * i;
        if (r >= rows || cols == 0) continue;
        const int64_t t = token[row0 + r];
        const T* had = base + t * p.ld_base + mine;
        T* to = out + t * p.ld_out + mine;
        uint32_t now[kTiles] = {};
        if (p.vec) {
          if constexpr (kTiles == 4) {
            *reinterpret_cast<uint4*>(now) = m == 0 ? ptx::lds_128(from + (kPairs * kTiles + i) * kChunk) : *reinterpret_cast<const uint4*>(had);
          } else {
            const uint8_t* staged = tile + pass % kDepth * Cfg::kStage + kPairs * kTiles * kChunk + i * (kChunk / 2) + tid * 8;
            *reinterpret_cast<uint2*>(now) = m == 0 ? ptx::lds_64(ptx::smem_u32(staged)) : *reinterpret_cast<const uint2*>(had);
          }
        } else {
#pragma unroll
          for (int j = 0; j < kMine; ++j)
            if (j < cols) now[j / 2] |= (uint32_t)bits(had[j]) << (j % 2 * 16);
        }
        if (used > 0) {
          const float inv = unscale[r];
#pragma unroll
          for (int j = 0; j < kTiles; ++j) {
            const float2 was = unpack2<T>(now[j]);
            now[j] = pack2<T>(was.x + acc[j][2 * i] * inv, was.y + acc[j][2 * i + 1] * inv);
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
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <typename T, int kPairs, int kTiles>
static int launch_expand(Params& p, int block, cudaStream_t st) {
  using Cfg = ExpandCfg<kPairs, kTiles>;
  int64_t units = 0;
  for (int s = 0; s < p.S; ++s) units += (p.col0[s + 1] - p.col0[s] + Cfg::kCols - 1) / Cfg::kCols;
  // Blocks are cut until there are as many CTAs as run at once, then a CTA takes as many passes as leave that many.
  const int64_t want = (int64_t)std::min(4, (227 * 1024) / (Cfg::kDepth * Cfg::kStage + 16 * Cfg::kPitch + 3072)) * sm_count();
  p.sub = std::min(block, Cfg::kMostRows);
  while (p.sub > 16 && units * p.max_blocks * (block / p.sub) < want) p.sub /= 2;
  p.subs = block / p.sub;
  p.passes = (int)std::min<int64_t>(16, (units * p.max_blocks * p.subs + want - 1) / want);
  int chunks = 0;
  for (int s = 0; s < p.S; ++s) {
    p.chunk0[s] = chunks;
    const int64_t per = (int64_t)Cfg::kCols * p.passes;
    chunks += (int)((p.col0[s + 1] - p.col0[s] + per - 1) / per);
  }
  p.chunk0[p.S] = chunks;
  const int64_t grid = (int64_t)chunks * p.max_blocks * p.subs;
  SGLB_REQUIRE(grid < (1ll << 31), "lora_add: %lld tiles are too many", (long long)grid);
  auto kern = expand_kernel<T, kPairs, kTiles>;
  static thread_local bool attr_set[64] = {false};  // the opt-in is per function and per device
  int dev = 0;
  SGLB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    SGLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kDepth * Cfg::kStage + Cfg::kMostRows * Cfg::kPitch));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  SGLB_CUDA(launch_pdl(kern, (unsigned)grid, kWarps * 32, (size_t)(Cfg::kDepth * Cfg::kStage + p.sub * Cfg::kPitch), st, p));
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
static int64_t up(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace lora
}  // namespace sglb200

using namespace sglb200;

extern "C" int64_t sglb200_lora_add_workspace_bytes(int64_t tokens, int num_adapters, int rank, int num_slices) {
  if (tokens <= 0 || num_adapters < 1 || rank < 1 || num_slices < 1) return 0;
  // (whichever blocks the call takes)
  const int64_t blocks = tokens / narrow::kSmallBlock + num_adapters + 1;
  return lora::up(4 * tokens) + lora::up(4 * (3 * blocks + 1)) + lora::up(4 * tokens * num_slices * rank);
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
  SGLB_REQUIRE(slice_sizes != nullptr, "lora_add: null slice_sizes");
  lora::Params p{};
  int64_t at = 0;
  bool even = true;
  for (int s = 0; s < num_slices; ++s) {
    SGLB_REQUIRE(slice_sizes[s] >= 1, "lora_add: slice %d has %lld columns", s, (long long)slice_sizes[s]);
    p.col0[s] = at;
    even = even && at % 8 == 0;
    at += slice_sizes[s];
    SGLB_REQUIRE(at <= N, "lora_add: the slices have more than %lld columns", (long long)N);
  }
  p.col0[num_slices] = at;
  SGLB_REQUIRE(at == N, "lora_add: the slices have %lld columns of %lld", (long long)at, (long long)N);
  if (tokens == 0) return SGLB200_OK;
  SGLB_REQUIRE(x && lora_a && lora_b && base && out && adapter_ids, "lora_add: null pointer");
  SGLB_REQUIRE(aligned16(x) && aligned16(lora_a) && aligned16(lora_b), "lora_add: x, lora_a and lora_b must be 16-byte aligned");
  SGLB_REQUIRE(((uintptr_t)base & 1) == 0 && ((uintptr_t)out & 1) == 0, "lora_add: base and out must be aligned to 2 bytes");
  const int64_t bytes = sglb200_lora_add_workspace_bytes(tokens, num_adapters, rank, num_slices);
  if (workspace == nullptr || workspace_bytes < bytes || !aligned16(workspace))
    return fail(SGLB200_E_WORKSPACE, "lora_add: %lld bytes of workspace are needed, aligned to 16", (long long)bytes);
  const bool scan = tokens <= narrow::kScanRows;
  const int block = scan ? narrow::kSmallBlock : narrow::block_rows(tokens, (int64_t)num_slices * rank, K, num_adapters);
  const int64_t blocks = lora::most_blocks(tokens, num_adapters, block);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int32_t* order = static_cast<int32_t*>(workspace);
  int32_t* start = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(workspace) + lora::up(4 * tokens));
  float* h = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(start) + lora::up(4 * (3 * blocks + 1)));
  if (scan) {
    p.blocks.ids = adapter_ids, p.blocks.ids_rows = (int)tokens, p.blocks.adapters = num_adapters;
  } else {
    p.blocks = {order, start, start + blocks, start + 2 * blocks, start + 3 * blocks, nullptr, 0, 0};
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
    SGLB_CUDA(launch_pdl(lora::plan_kernel, 1u, (unsigned)lora::kPlanThreads, smem, st, adapter_ids, (int)tokens, num_adapters, block, order,
                         start, start + blocks, start + 2 * blocks, start + 3 * blocks));
  }
  narrow::Params n{};
  n.x = x, n.w = lora_a, n.y = h, n.ranks = ranks, n.blocks = p.blocks;
  n.T = tokens, n.N = (int64_t)num_slices * rank, n.K = K, n.ldx = x_stride, n.rank_rows = rank, n.adapters = num_adapters, n.block = block;
  int rc = narrow::product(n, dtype, blocks, st);
  if (rc) return rc;
  p.b = lora_b, p.base = base, p.out = out, p.h = h, p.scalings = scalings, p.ranks = ranks;
  p.N = N, p.ld_base = base_stride, p.ld_out = out_stride, p.R = rank, p.S = num_slices, p.max_blocks = (int)blocks;
  p.in_place = base == out && base_stride == out_stride;
  p.vec = even && N % 8 == 0 && base_stride % 8 == 0 && out_stride % 8 == 0 && aligned16(base) && aligned16(out);
  p.wait_probes = g_gemm_wait_probes;
  // (its row pitches are 32-bit numbers of bytes)
  if (block == narrow::kTileBlock && p.vec && rank <= lora::kTileRank && base_stride < 1ll << 30 && out_stride < 1ll << 30)
    return lora::expand_tile(p, dtype, st);
  const int rows = tokens <= 16 ? 16 : tokens <= 32 ? 32 : block;  // the most that a block can have
  return dtype == 0 ? lora::expand<__nv_bfloat16>(p, rows, st) : lora::expand<__half>(p, rows, st);
}
