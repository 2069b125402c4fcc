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
#include "gemm_common.cuh"
#include "lora.cuh"
#include "ptx_sm100.cuh"

namespace sglb200 {
namespace lora {

// ---- plan -----------------------------------------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

// One CTA.  Tokens of one adapter in any order: their rows do not meet.  Neighbours mostly name the same adapter, so that a warp counts
// equal ids at once.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const int32_t* __restrict__ ids, int T, int L, int block, int32_t* order,
                                                            int32_t* start, int32_t* rows, int32_t* adapter, int32_t* count) {
  __shared__ int32_t cursor[kMaxAdapters + 1];
  const int tid = threadIdx.x, lane = tid & 31;
  for (int i = tid; i <= L; i += kPlanThreads) cursor[i] = 0;
  __syncthreads();
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  const int padded = (T + 31) & ~31;
  for (int i = tid; i < padded; i += kPlanThreads) {
    const int id = i < T ? ids[i] : -1;
    const int key = i >= T ? L + 1 : id >= 0 && id < L ? id : L;
    const uint32_t same = __match_any_sync(0xffffffffu, key);
    if (i < T && (int)__ffs(same) - 1 == lane) atomicAdd(&cursor[key], __popc(same));
  }
  __syncthreads();
  if (tid < 32) {  // first token and first block of every adapter
    int tokens = 0, blocks = 0;
    for (int at = 0; at <= L; at += 32) {
      const int l = at + lane, n = l <= L ? cursor[l] : 0, b = (n + block - 1) / block;
      int sn = n, sb = b;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int un = __shfl_up_sync(0xffffffffu, sn, off), ub = __shfl_up_sync(0xffffffffu, sb, off);
        if (lane >= off) sn += un, sb += ub;
      }
      if (l <= L) {
        for (int i = 0; i < b; ++i) {
          const int at_block = blocks + sb - b + i;
          start[at_block] = tokens + sn - n + i * block;
          rows[at_block] = min(block, n - i * block);
          adapter[at_block] = l < L ? l : -1;
        }
        cursor[l] = tokens + sn - n;
      }
      tokens += __shfl_sync(0xffffffffu, sn, 31), blocks += __shfl_sync(0xffffffffu, sb, 31);
    }
    if (lane == 0) *count = blocks;
  }
  __syncthreads();
  for (int i = tid; i < padded; i += kPlanThreads) {
    const int id = i < T ? ids[i] : -1;
    const int key = i >= T ? L + 1 : id >= 0 && id < L ? id : L;
    const uint32_t same = __match_any_sync(0xffffffffu, key);
    const int leader = __ffs(same) - 1;
    int at = 0;
    if (i < T && leader == lane) at = atomicAdd(&cursor[key], __popc(same));
    at = __shfl_sync(0xffffffffu, at, leader) + __popc(same & ((1u << lane) - 1));
    if (i < T) order[at] = i;
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

// kSteps: instructions over the rank, at most; kTiles: groups of 8 columns of a warp.  A lane holds the same two kTiles neighbouring columns
// of a token in all groups, so that base and out go by 4 kTiles bytes.  A warp asks for the next 16 tokens' base before it multiplies these.
template <typename T, int kSteps, int kTiles>
__global__ void __launch_bounds__(kWarps * 32) expand_kernel(const Params p) {
  constexpr int kCols = 8 * kTiles, kMine = 2 * kTiles;
  extern __shared__ __align__(16) uint8_t tile[];  // [rows of a CTA][pitch]: a token's high terms, then its low terms
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
  }
  if (row0 >= rows || (adapter < 0 && p.in_place)) return;
  rows = min(rows - row0, p.sub);
  int slice = 0;
  while (slice + 1 < p.S && chunk >= p.chunk0[slice + 1]) ++slice;
  const int64_t end = p.col0[slice + 1];
  const int64_t c0 = p.col0[slice] + (int64_t)(chunk - p.chunk0[slice]) * p.passes * kWarps * kCols + warp * kCols;
  const int used = adapter < 0 ? 0 : p.ranks != nullptr ? min(max(__ldg(p.ranks + adapter), 0), p.R) : p.R;
  const T* weights = static_cast<const T*>(p.b) + (adapter < 0 ? 0 : (int64_t)adapter * p.N * p.R);
  const T* base = static_cast<const T*>(p.base);
  T* out = static_cast<T*>(p.out);

  uint2 w[kSteps][kTiles];
  auto load_weights = [&](int64_t c) {
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      const int64_t n = c + (g >> 1) * kMine + j * 2 + (g & 1);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int r = s * 16 + q * 4;
        w[s][j] = n < end && r < used ? __ldg(reinterpret_cast<const uint2*>(weights + n * p.R + r)) : make_uint2(0, 0);
      }
    }
    if (used % 4 != 0) {  // beyond the rank anything may stand
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int r = s * 16 + q * 4;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          if (r + 1 >= used) w[s][j].x &= 0xffffu;
          if (r + 2 >= used) w[s][j].y = 0;
          if (r + 3 >= used) w[s][j].y &= 0xffffu;
        }
      }
    }
  };
  // Two tokens' kMine columns at c, 16 bytes (8 for two groups) at a time where all lie so.
  auto load_base = [&](int64_t c, int m, uint32_t (&old)[2][kTiles]) {
    const int64_t mine = c + q * kMine;
    const int cols = (int)max((int64_t)0, min((int64_t)kMine, end - mine));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = m + g + 8 * i;
#pragma unroll
      for (int j = 0; j < kTiles; ++j) old[i][j] = 0;
      if (r >= rows || cols == 0) continue;
      const T* from = base + (int64_t)token[row0 + r] * p.ld_base + mine;
      if (p.vec) {
        if constexpr (kTiles == 4)
          *reinterpret_cast<uint4*>(old[i]) = *reinterpret_cast<const uint4*>(from);
        else
          *reinterpret_cast<uint2*>(old[i]) = *reinterpret_cast<const uint2*>(from);
      } else {
#pragma unroll
        for (int j = 0; j < kMine; ++j)
          if (j < cols) old[i][j / 2] |= (uint32_t)bits(from[j]) << (j % 2 * 16);
      }
    }
  };
  uint32_t old[2][kTiles] = {};
  if (c0 < end) load_weights(c0);
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  __syncthreads();  // (the tokens)
  if (c0 < end) load_base(c0, 0, old);
  const float scaling = adapter >= 0 && p.scalings != nullptr ? __ldg(p.scalings + adapter) : 1.f;
  // (two rows' loads at a time)
  constexpr int kV = (kSteps + 1) / 2;
  for (int i = warp; i < rows; i += 2 * kWarps) {
    float v[2][kV];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float* h = p.h + ((int64_t)token[row0 + min(i + u * kWarps, rows - 1)] * p.S + slice) * p.R;
#pragma unroll
      for (int j = 0; j < kV; ++j) v[u][j] = j * 32 + lane < used ? __ldcg(h + j * 32 + lane) * scaling : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = i + u * kWarps;
      if (row >= rows) break;
      uint16_t* at = reinterpret_cast<uint16_t*>(tile + row * p.pitch);
      const float inv = split_row<T>(v[u], p.R, lane, [&](int r, uint16_t hi, uint16_t lo) { at[r] = hi, at[p.R + r] = lo; });
      if (lane == 0) unscale[row] = inv;
    }
  }
  __syncthreads();
  const int steps = (used + 15) / 16;

  for (int pass = 0; pass < p.passes; ++pass) {
    const int64_t c = c0 + (int64_t)pass * kWarps * kCols;
    if (c >= end) break;
    const int64_t next_c = c + kWarps * kCols;
    const bool more = pass + 1 < p.passes && next_c < end;
    if (pass > 0) load_weights(c);
    const int64_t mine = c + q * kMine;
    const int cols = (int)max((int64_t)0, min((int64_t)kMine, end - mine));
    for (int m = 0; m < rows; m += 16) {
      const int ra = m + g, rb = m + g + 8;
      uint32_t ahead[2][kTiles] = {};
      if (m + 16 < rows) {
        load_base(c, m + 16, ahead);
      } else if (more) {
        load_base(next_c, 0, ahead);
      }
      float acc[kTiles][4] = {};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (s >= steps) break;
        const bool in = s * 16 + q * 4 < p.R;  // (R is a multiple of 8: a last instruction may have half its columns)
        const uint8_t* pa = tile + ra * p.pitch + (s * 16 + q * 4) * 2;
        const uint8_t* pb = tile + rb * p.pitch + (s * 16 + q * 4) * 2;
        const uint2 zero = make_uint2(0, 0);
        // (rows past the last are not written, and meet only their own sums)
        const uint2 ah = in ? *reinterpret_cast<const uint2*>(pa) : zero, bh = in ? *reinterpret_cast<const uint2*>(pb) : zero;
        const uint2 al = in ? *reinterpret_cast<const uint2*>(pa + p.R * 2) : zero, bl = in ? *reinterpret_cast<const uint2*>(pb + p.R * 2) : zero;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          mma16816<T>(acc[j], al.x, bl.x, al.y, bl.y, w[s][j].x, w[s][j].y);
          mma16816<T>(acc[j], ah.x, bh.x, ah.y, bh.y, w[s][j].x, w[s][j].y);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = m + g + 8 * i;
        if (r >= rows || cols == 0) continue;
        T* to = out + (int64_t)token[row0 + r] * p.ld_out + mine;
        const float inv = unscale[r];
        uint32_t now[kTiles];
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          if (used == 0) {
            now[j] = old[i][j];
          } else {
            const float2 was = unpack2<T>(old[i][j]);
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
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < kTiles; ++j) old[i][j] = ahead[i][j];
    }
  }
}

template <typename T, int kSteps, int kTiles>
static int launch_expand(Params& p, int block, cudaStream_t st) {
  constexpr int kCols = 8 * kTiles * kWarps;
  int64_t units = 0;
  for (int s = 0; s < p.S; ++s) units += (p.col0[s + 1] - p.col0[s] + kCols - 1) / kCols;
  // Blocks are cut until there are four CTAs for every SM, then a CTA takes as many passes as leave that many.
  const int64_t want = 4 * sm_count();
  p.sub = block;
  while (p.sub > 16 && units * p.max_blocks * (block / p.sub) < want) p.sub /= 2;
  p.subs = block / p.sub;
  const int64_t passes = units * p.max_blocks * p.subs / want;
  p.passes = (int)(passes < 1 ? 1 : passes > 8 ? 8 : passes);
  int chunks = 0;
  for (int s = 0; s < p.S; ++s) {
    p.chunk0[s] = chunks;
    const int64_t per = (int64_t)kCols * p.passes;
    chunks += (int)((p.col0[s + 1] - p.col0[s] + per - 1) / per);
  }
  p.chunk0[p.S] = chunks;
  // rows 32 bytes apart modulo 128: four rows of 32 bytes are read without a bank conflict
  p.pitch = (4 * p.R + 127) / 128 * 128 + 32;
  const size_t smem = (size_t)p.sub * p.pitch;
  const int64_t grid = (int64_t)chunks * p.max_blocks * p.subs;
  SGLB_REQUIRE(grid < (1ll << 31), "lora_add: %lld tiles are too many", (long long)grid);
  auto kern = expand_kernel<T, kSteps, kTiles>;
  if (smem > 40 * 1024) {  // (beside the static ones)
    static thread_local bool attr_set[64] = {false};  // the opt-in is per function and per device
    int dev = 0;
    SGLB_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
      SGLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, narrow::kTileBlock * (4 * kMaxRank + 160)));
      if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
  }
  SGLB_CUDA(launch_pdl(kern, (unsigned)grid, kWarps * 32, smem, st, p));
  return SGLB200_OK;
}

template <typename T>
static int expand(Params& p, int block, cudaStream_t st) {
  if (p.R <= 16) return launch_expand<T, 1, 4>(p, block, st);
  if (p.R <= 32) return launch_expand<T, 2, 4>(p, block, st);
  if (p.R <= 64) return launch_expand<T, 4, 4>(p, block, st);
  if (p.R <= 128) return launch_expand<T, 8, 4>(p, block, st);
  return launch_expand<T, 16, 2>(p, block, st);
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
  SGLB_REQUIRE(tokens < (1ll << 31) - 256 && N < (1ll << 31) - 65536 && K <= 1 << 20, "lora_add: %lld tokens, N %lld or K %lld is too large",
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
    SGLB_CUDA(launch_pdl(lora::plan_kernel, 1u, (unsigned)lora::kPlanThreads, (size_t)0, st, adapter_ids, (int)tokens, num_adapters, block, order,
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
  return dtype == 0 ? lora::expand<__nv_bfloat16>(p, block, st) : lora::expand<__half>(p, block, st);
}
