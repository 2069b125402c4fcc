// y[t, n] = sum_k x[t, k] w[n, k], few n, float32 sums (see narrow.cuh).
//
// narrow_kernel: the weights on the M side of mma.sync (16 of their rows), up to 32 activation rows on its N side, operands straight from
// global memory into registers: a lane takes 16 consecutive bytes of its row, and as a sum does not mind the order of its terms, those are
// its part of two instructions, of the weights' rows and the activations' alike.  K is split over the warps of a CTA and the CTAs of a
// cluster, whose sums meet in a fixed order.  Bound by latency: in a graph of calls 1 x 256 x 7168 takes 3.4 us (1.1 TB/s), of which first loads
// 1, the sums and two cluster barriers 1.5; 64 x 128 x 2048 3.6 us.
#include <algorithm>

#include "gemm_common.cuh"
#include "narrow.cuh"
#include "narrow_rule.h"
#include "ptx_sm100.cuh"

namespace sglb200 {
namespace narrow {

constexpr int kWarps = 8;
constexpr int kStep = 32;  // columns of K a warp takes at a time

// What a warp adds up of 16 weight rows and up to kG groups of 8 activation rows, `rows` in all, over steps s0 .. s1 of K, to
// part[16][pitch]; `row_of(i)`: the i-th activation row.  kAhead steps are asked for at once.
template <typename T, int kG, int kAhead, class RowOf>
__device__ __forceinline__ void add_up(const Params& p, const T* wa, const T* wb, bool a_on, bool b_on, int rows, int s0, int s1, int lane,
                                       float* part, int pitch, RowOf row_of) {
  constexpr bool kF16 = std::is_same<T, __half>::value;
  const int g = lane >> 2, q = lane & 3;
  const T* x[kG];
#pragma unroll
  for (int j = 0; j < kG; ++j) x[j] = static_cast<const T*>(p.x) + row_of(min(j * 8 + g, rows - 1)) * p.ldx;
  float acc[kG][4] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll(kAhead)
  for (int s = s0; s < s1; ++s) {
    const int64_t k = (int64_t)s * kStep + q * 8;
    const bool in = k < p.K;  // (K is a multiple of 8)
    const uint4 a = in && a_on ? __ldg(reinterpret_cast<const uint4*>(wa + k)) : zero;
    const uint4 b = in && b_on ? __ldg(reinterpret_cast<const uint4*>(wb + k)) : zero;
    uint4 v[kG];
#pragma unroll
    for (int j = 0; j < kG; ++j) v[j] = in && (kG == 1 || j * 8 < rows) ? ld_nc_16(x[j] + k) : zero;
#pragma unroll
    for (int j = 0; j < kG; ++j)
      if (kG == 1 || j * 8 < rows) {
        ptx::mma_16816<kF16>(acc[j], a.x, b.x, a.y, b.y, v[j].x, v[j].y);
        ptx::mma_16816<kF16>(acc[j], a.z, b.z, a.w, b.w, v[j].z, v[j].w);
      }
  }
#pragma unroll
  for (int j = 0; j < kG; ++j) {
    if (j * 8 >= rows) break;
    *reinterpret_cast<float2*>(part + g * pitch + j * 8 + q * 2) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(part + (g + 8) * pitch + j * 8 + q * 2) = make_float2(acc[j][2], acc[j][3]);
  }
}

// Up to kG groups of 8 activation rows.  `part` and `sums` are padded so that neither their writes nor their reads meet in a bank:
// unpadded, 64 rows x 256 x 7168 took 12.8 us.
template <typename T, int kG>
__global__ void __launch_bounds__(kWarps * 32, 3) narrow_kernel(const Params p) {
  constexpr int kCols = kG * 8, kPartPitch = kCols + 8, kSumPitch = 17;
  __shared__ float part[kWarps][16][kPartPitch];
  __shared__ float sums[kCols * kSumPitch];
  __shared__ int32_t row[kSmallBlock];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = ptx::warp_index(), g = lane >> 2;
  const uint32_t tile = cluster_id(), of_block = tile / (uint32_t)p.n_tiles;
  const int rank = cluster_rank(), n0 = (int)(tile - of_block * p.n_tiles) * 16;
  const int64_t block = of_block;
  ptx::grid_dependency_wait();
  ptx::launch_dependents();
  int64_t start = block * kSmallBlock, adapter = 0;
  int rows = (int)min((int64_t)kSmallBlock, p.T - start);
  const bool sorted = p.blocks.order != nullptr || p.blocks.ids != nullptr;
  int used = p.rank_rows;
  if (p.blocks.ids != nullptr) {
    if (warp == 0) {
      int n = 0, a = -1;
      scan_pick(scan_ids(p.blocks, kSmallBlock, lane), (int)block, kSmallBlock, lane, row, n, a);  // (0 rows: there is no such block)
      if (lane == 0) found[0] = n, found[1] = a;
    }
    __syncthreads();
    rows = found[0], adapter = found[1];
    if (rows == 0 || adapter < 0) return;  // (uniform over the cluster)
    if (p.ranks != nullptr) used = min(max(__ldg(p.ranks + adapter), 0), p.rank_rows);
  } else if (p.blocks.order != nullptr) {
    const int4 at = __ldcg(p.blocks.at + block);
    start = at.x, rows = at.y, adapter = at.z, used = at.w;
    if (adapter < 0) return;
    if (tid < rows) row[tid] = p.blocks.order[start + tid];
    __syncthreads();
  }
  const T* w = static_cast<const T*>(p.w) + adapter * p.N * p.K;
  const int na = n0 + g, nb = n0 + g + 8;
  const bool whole = used == p.rank_rows;
  const bool a_on = na < p.N && (whole || na % p.rank_rows < used), b_on = nb < p.N && (whole || nb % p.rank_rows < used);
  const T* wa = w + (a_on ? na : 0) * p.K;
  const T* wb = w + (b_on ? nb : 0) * p.K;
  const int steps = (int)((p.K + kStep - 1) / kStep), parts = p.splits * kWarps, mine = rank * kWarps + warp;
  const int parts_log = 31 - __clz(parts);
  const int s0 = mine * steps >> parts_log, s1 = (mine + 1) * steps >> parts_log;  // (at most 64 x 32768)
  auto row_of = [&](int i) { return sorted ? (int64_t)row[i] : start + i; };
  float* to = &part[warp][0][0];
  // (blocks of a batch of many adapters have few rows)
  if (rows <= 8) add_up<T, 1, 4>(p, wa, wb, a_on, b_on, rows, s0, s1, lane, to, kPartPitch, row_of);
  else if (kG > 2 && rows <= 16) add_up<T, 2, 2>(p, wa, wb, a_on, b_on, rows, s0, s1, lane, to, kPartPitch, row_of);
  else add_up<T, kG, (kG <= 2 ? 3 : 1)>(p, wa, wb, a_on, b_on, rows, s0, s1, lane, to, kPartPitch, row_of);
  __syncthreads();
  // The warps' sums, then the CTAs', each in ascending order of K.
  for (int i = tid; i < 16 * kCols; i += kWarps * 32) {
    const int t = i % kCols, n = i / kCols;
    if (t >= rows) continue;
    float v = 0.f;
#pragma unroll
    for (int u = 0; u < kWarps; ++u) v += part[u][n][t];
    sums[t * kSumPitch + n] = v;
  }
  if (p.splits > 1) {
    ptx::cluster_sync();
  } else {
    __syncthreads();
  }
  const uint32_t at = ptx::smem_u32(sums);
  for (int i = tid + rank * kWarps * 32; i < 16 * rows; i += p.splits * kWarps * 32) {
    // (neighbouring threads take neighbouring rows of the weights, which lie side by side in y)
    const int n = i & 15, t = i >> 4;
    if (n0 + n >= p.N) continue;
    float v = 0.f;
    if (p.splits > 1) {
      float o[8];
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s < p.splits)
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o[s]) : "r"(ptx::cluster_map(at + (t * kSumPitch + n) * 4, s)) : "memory");
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s < p.splits) v += o[s];
    } else {
      v = sums[t * kSumPitch + n];
    }
    p.y[(sorted ? (int64_t)row[t] : start + t) * p.N + n0 + n] = v;
  }
  if (p.splits > 1) ptx::cluster_sync_relaxed();  // no CTA leaves while another reads its shared memory
}

template <typename T, int kG>
static int launch(const Params& p, int64_t blocks, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  const int64_t grid = blocks * p.n_tiles * p.splits;
  SGLB_REQUIRE(grid < (1ll << 31), "narrow product: %lld tiles are too many", (long long)grid);
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3(kWarps * 32, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.splits, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  SGLB_CUDA(cudaLaunchKernelEx(&cfg, narrow_kernel<T, kG>, p));
  return SGLB200_OK;
}

template <typename T>
static int dispatch(Params& p, int64_t blocks, cudaStream_t st) {
  p.n_tiles = (int)((p.N + 15) / 16);
  const int64_t tiles = blocks * p.n_tiles, steps = (p.K + kStep - 1) / kStep;
  p.splits = 1;
  // (two CTAs an SM: clusters that do not run at once would take a second round)
  while (p.splits < 8 && tiles <= cluster_fits().paired[p.splits * 2] && steps >= p.splits * 2 * kWarps) p.splits *= 2;
  if (p.T <= 8) return launch<T, 1>(p, blocks, st);
  if (p.T <= 16) return launch<T, 2>(p, blocks, st);
  return launch<T, 4>(p, blocks, st);
}

int product(Params p, int dtype, int64_t max_blocks, cudaStream_t st) {
  if (p.block == kTileBlock) return tile_product(p, dtype, max_blocks, st);
  return dtype == 0 ? dispatch<__nv_bfloat16>(p, max_blocks, st) : dispatch<__half>(p, max_blocks, st);
}

}  // namespace narrow
}  // namespace sglb200

using namespace sglb200;

extern "C" int sglb200_router_logits(const void* x, const void* w, int dtype, float* y, int64_t tokens, int64_t num_experts, int64_t K,
                                     int64_t x_stride, void* stream) {
  if (dtype != 0 && dtype != 1) return fail(SGLB200_E_UNSUPPORTED, "router_logits: dtype %d (0 bf16, 1 fp16)", dtype);
  SGLB_REQUIRE(tokens >= 0 && num_experts >= 1 && K >= 1, "router_logits: %lld tokens, %lld experts, K %lld", (long long)tokens,
               (long long)num_experts, (long long)K);
  SGLB_REQUIRE(K % 8 == 0 && x_stride % 8 == 0 && x_stride >= K, "router_logits: K (%lld) and the rows' stride (%lld) must be divisible by 8",
               (long long)K, (long long)x_stride);
  SGLB_REQUIRE(tokens < (1ll << 31) - 256 && num_experts <= 1 << 16 && K <= 1 << 20, "router_logits: %lld tokens, %lld experts or K %lld is too large",
               (long long)tokens, (long long)num_experts, (long long)K);
  SGLB_REQUIRE(x_stride < std::min<int64_t>(1ll << 40, (1ll << 60) / std::max<int64_t>(tokens, 1)), "router_logits: the rows' stride %lld is too large", (long long)x_stride);
  if (tokens == 0) return SGLB200_OK;
  SGLB_REQUIRE(x && w && y, "router_logits: null pointer");
  SGLB_REQUIRE(aligned16(x) && aligned16(w) && aligned16(y), "router_logits: pointers must be 16-byte aligned");
  narrow::Params p{};
  p.x = x, p.w = w, p.y = y, p.T = tokens, p.N = num_experts, p.K = K, p.ldx = x_stride, p.rank_rows = (int)num_experts;
  p.adapters = 1, p.block = narrow::small_blocks(tokens, num_experts, K) ? narrow::kSmallBlock : narrow::kTileBlock;
  return narrow::product(p, dtype, (tokens + p.block - 1) / p.block, static_cast<cudaStream_t>(stream));
}
