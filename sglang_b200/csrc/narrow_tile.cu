// y[t, n] = sum_k x[t, k] w[n, k] for many rows (see narrow.cuh), on tcgen05.mma.kind::f16.
//
// A tile is 128 activation rows by up to 256 weight rows, in stages of 64 columns.  The weights and activations that lie one after the other
// come by TMA; of sorted activations 32 rows at a time that do (the tokens of a long request), the others by asynchronous copies of 16 bytes of
// four warps (two took 0.65 us a stage of 128 rows, TMA gathers of four rows 2 us).  K is split over the CTAs of a cluster, which add their
// sums through distributed shared memory in a fixed order.
//
// Router, 8192 x 256 x 7168: 38 us a call on inputs from memory, 0.52 of the measured copy rate, the tensor pipe busy half of the time, and 33 on inputs
// in L2; 511 x 160 x 5120: 7.7 and 7.1 us, a start and a sum over the cluster.
//
// The instruction cuts off what does not fit its sum, each time: over 7168 columns that would be off by more than a float32 product is.  So
// the sums of 256 columns begin from zero, in two buffers of tensor memory in turn, and meet in the registers of eight warps.
#include <algorithm>

#include "gemm_common.cuh"
#include "narrow.cuh"
#include "ptx_sm100.cuh"

namespace sglb200 {
namespace narrow {

constexpr int kThreads = 320, kSortedThreads = 448;  // eight warps for the sums, one that loads, one that multiplies, four that copy sorted rows
constexpr int kStageK = 64;        // columns of a stage: 128 bytes, one swizzle span
constexpr int kChunk = 4;          // stages that are summed up in tensor memory
constexpr int kMaxStages = 8;
constexpr uint32_t kRing = 192 * 1024;
constexpr uint32_t kXBytes = kTileBlock * kStageK * 2;

struct Ctl {
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
  int first[4];  // the first row of 32 of the tile that lie one after the other, else -1
  int row[kTileBlock];
};

struct TileParams {
  Params p;
  int nt;        // weight rows of a tile, a multiple of 16
  int stages, kb_total, fp16;
  uint32_t wait_probes;
  int* status;   // 1 where a pipeline wait has run out
};

#define NARROW_WAIT(bar, parity) \
  (t.wait_probes != ptx::kProbesNone && (ptx::mbar_test(bar, parity) || ptx::mbar_wait_quiet(bar, parity)))

// The sums of a tile out of the (up to kMost) CTAs' shared memory, in ascending order of K; each CTA adds up its share of the rows.  A thread
// has four columns of every `step`-th row and asks for kAtOnce rows' parts at a time.
template <int kMost, int kAtOnce, int kAll, bool kSorted>
__device__ __forceinline__ void store_sums(const TileParams& t, uint32_t base, int rows, int rank, int n0, int64_t start, const int* row_of) {
  const Params& p = t.p;
  const int row0 = rank * rows / p.splits, row1 = (rank + 1) * rows / p.splits, quads = t.nt / 4, step = kAll / quads;
  const int tid = threadIdx.x, c = tid % quads * 4;
  const bool vec = p.N % 4 == 0;
  if (n0 + c >= p.N || tid >= step * quads) return;
  for (int row = row0 + tid / quads; row < row1; row += kAtOnce * step) {
    float4 v[kAtOnce][kMost];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (row + u * step >= row1) break;
      const uint32_t at = base + (uint32_t)((row + u * step) * (t.nt + 4) + c) * 4;
      if constexpr (kMost == 1) {
        v[u][0] = ptx::lds_f32x4(at);
      } else {
#pragma unroll
        for (int s = 0; s < kMost; ++s)
          if (s < p.splits)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v[u][s].x), "=f"(v[u][s].y), "=f"(v[u][s].z), "=f"(v[u][s].w)
                         : "r"(ptx::cluster_map(at, s))
                         : "memory");
      }
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int mine = row + u * step;
      if (mine >= row1) break;
      float4 sum = v[u][0];
#pragma unroll
      for (int s = 1; s < kMost; ++s)
        if (s < p.splits) sum.x += v[u][s].x, sum.y += v[u][s].y, sum.z += v[u][s].z, sum.w += v[u][s].w;
      float* to = p.y + (kSorted ? (int64_t)row_of[mine] : start + mine) * p.N + n0 + c;
      if (vec) {
        *reinterpret_cast<float4*>(to) = sum;
      } else {
        const float one[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n0 + c + j < p.N) to[j] = one[j];
      }
    }
  }
}

// kUnits: groups of 16 columns of a tile that each of the two warpgroups adds up, at most.
template <int kUnits, bool kSorted>
__global__ void __launch_bounds__(kSorted ? kSortedThreads : kThreads, 1)
    narrow_tile_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const TileParams t) {
  constexpr uint32_t kBuf = kUnits * 32;  // columns of tensor memory of a buffer
  constexpr bool sorted = kSorted;
  constexpr int kAll = kSorted ? kSortedThreads : kThreads, kCopies = 4 * 32;
  const Params& p = t.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Ctl* ctl = reinterpret_cast<Ctl*>(ring + kRing);
  const int tid = threadIdx.x, warp = ptx::warp_index(), lane = tid & 31;
  volatile int* abort_flag = &ctl->abort_flag;
  const uint32_t tile = cluster_id(), of_block = tile / (uint32_t)p.n_tiles;
  const int rank = cluster_rank(), n0 = (int)(tile - of_block * p.n_tiles) * t.nt;
  const int64_t block = of_block;
  const uint32_t full = ptx::smem_u32(ctl->full), empty = ptx::smem_u32(ctl->empty), acc_full = ptx::smem_u32(ctl->acc_full),
                 acc_empty = ptx::smem_u32(ctl->acc_empty);
  // (tensor memory is taken once the kernel in front has ended; the kernel behind may start when every CTA has its own)
  ptx::grid_dependency_wait();
  int64_t start = block * kTileBlock;
  int rows = (int)min((int64_t)kTileBlock, p.T - start), adapter = 0;
  if (sorted) {
    const int4 at = __ldcg(p.blocks.at + block);
    start = at.x, rows = at.y, adapter = at.z;
    if (adapter < 0) {  // (uniform over the cluster)
      ptx::launch_dependents();
      return;
    }
    if (warp < 4) {
      const int i = warp * 32 + lane, row = __ldcg(p.blocks.order + start + min(i, rows - 1)), first = __shfl_sync(0xffffffffu, row, 0);
      const bool run = __all_sync(0xffffffffu, i >= rows || row == first + lane);
      ctl->row[i] = row;
      if (lane == 0) ctl->first[warp] = run ? first : -1;
    }
  }
  if (warp == 9) {
    ptx::tmem_alloc(ptx::smem_u32(&ctl->tmem_base), 2 * kBuf);
    ptx::tmem_relinquish();
  }
  if (sorted) __syncthreads();
  // 32 rows that have to be copied one by one, a bit each; the number of 32 that hold rows
  const int groups = (rows + 31) / 32;
  int scattered = 0;
  if (sorted)
    for (int i = 0; i < groups; ++i) scattered |= ctl->first[i] < 0 ? 1 << i : 0;
  if (tid == 0) {
    for (int s = 0; s < t.stages; ++s) ptx::mbar_init(full + s * 8, scattered ? kCopies + 1 : 1), ptx::mbar_init(empty + s * 8, 1);
    for (int b = 0; b < 2; ++b) ptx::mbar_init(acc_full + b * 8, 1), ptx::mbar_init(acc_empty + b * 8, 8);
    ctl->abort_flag = 0;
    ptx::mbar_fence_init();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  ptx::launch_dependents();
  const uint32_t tmem = ctl->tmem_base;
  const int kb0 = rank * t.kb_total / p.splits, kb1 = (rank + 1) * t.kb_total / p.splits;
  const uint32_t w_bytes = (uint32_t)t.nt * kStageK * 2, stage_bytes = kXBytes + w_bytes, base = ptx::smem_u32(ring);
  const int units = t.nt / 16, half = (units + 1) / 2;

  if (warp == 8) {
    if (ptx::elect_one()) {
      // (counters and not remainders of the stage's number: a thread by itself takes half a microsecond for two divisions)
      int s = 0;
      uint32_t ph = 1;  // a barrier's phase before its first counts as complete
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!NARROW_WAIT(empty + s * 8, ph)) {
          *abort_flag = 1;
          break;
        }
        const uint32_t at = base + s * stage_bytes, bar = full + s * 8;
        if (++s == t.stages) s = 0, ph ^= 1;
        ptx::mbar_arrive_expect_tx(bar, w_bytes + (sorted ? (uint32_t)(groups - __popc(scattered)) * (kXBytes / 4) : kXBytes));
        ptx::tma_load_3d(at + kXBytes, &map_w, bar, kb * kStageK * 2, n0, adapter);
        if (!sorted) {
          ptx::tma_load_2d(at, &map_x, bar, kb * kStageK * 2, (int)start);
        } else {
          for (int j = 0; j < groups; ++j)
            if (!(scattered >> j & 1)) ptx::tma_load_2d(at + j * (kXBytes / 4), &map_x, bar, kb * kStageK * 2, ctl->first[j]);
        }
      }
    }
    __syncwarp();
  } else if (warp >= 10) {
    if (scattered) {
      // Rows warp, + 4, .. of four at a time; a lane has 16 bytes of one of them.  (Rows past the last hold what they held; their sums are
      // nobody's.)
      const int c = lane & 7, r0 = (warp - 10) * 4 + (lane >> 3);
      const uint8_t* from[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        from[j] = static_cast<const uint8_t*>(p.x) + (int64_t)ctl->row[r0 + j * 16] * p.ldx * 2 + c * 16;
      const uint32_t to = (uint32_t)(r0 * 128 + ((c ^ (r0 & 7)) << 4));  // (rows 16 apart have the same swizzle)
      int s = 0;
      uint32_t ph = 1;
      for (int kb = kb0; kb < kb1; ++kb) {
        const bool ok = NARROW_WAIT(empty + s * 8, ph);
        if (!__all_sync(0xffffffffu, ok)) {
          if (lane == 0) *abort_flag = 1;
          break;
        }
        const int64_t k = (int64_t)kb * kStageK;
        const uint32_t bytes = k + c * 8 < p.K ? 16 : 0;  // (K is a multiple of 8; zeros beyond)
        const int64_t off = bytes ? k * 2 : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if ((scattered >> (j / 2) & 1) && r0 + j * 16 < rows) ptx::cp_async_16(base + s * stage_bytes + to + j * 2048, from[j] + off, bytes);
        ptx::cp_async_arrive(full + s * 8);
        if (++s == t.stages) s = 0, ph ^= 1;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    __syncwarp();
  } else if (warp == 9) {
    if (ptx::elect_one()) {
      const uint32_t id = ptx::idesc_f16(kTileBlock, t.nt, t.fp16);
      bool ok = true;
      int s = 0, left = kChunk;  // stages of a chunk
      uint32_t ph = 0, buf = 0, acc_ph = 1;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (left == kChunk) ok = NARROW_WAIT(acc_empty + buf * 8, acc_ph);
        if (ok) ok = NARROW_WAIT(full + s * 8, ph);
        if (!ok) break;
        if (scattered) ptx::fence_async_smem();  // (the copies' writes, which the barrier has shown, before the tensor core's reads)
        ptx::tc_fence_after();
        const uint32_t at = base + s * stage_bytes, x_lo = ptx::desc_lo128(at), w_lo = ptx::desc_lo128(at + kXBytes);
#pragma unroll
        for (int k = 0; k < kStageK / 16; ++k)
          ptx::mma_f16(tmem + buf * kBuf, ptx::pack_f32x2(x_lo + 2 * k, ptx::kDescHi128), ptx::pack_f32x2(w_lo + 2 * k, ptx::kDescHi128), id,
                       left < kChunk || k > 0 ? 1u : 0u);
        ptx::mma_commit(empty + s * 8);
        if (++s == t.stages) s = 0, ph ^= 1;
        if (--left == 0 || kb + 1 == kb1) {
          ptx::mma_commit(acc_full + buf * 8);
          left = kChunk, acc_ph ^= buf, buf ^= 1;
        }
      }
      if (!ok) *abort_flag = 1;
    }
    __syncwarp();
  } else {
    // ------------------------------ sums: lane = activation row, column = weight row ------------------------------
    float acc[kUnits * 16];
#pragma unroll
    for (int j = 0; j < kUnits * 16; ++j) acc[j] = 0.f;
    const int first = warp < 4 ? 0 : half, mine = warp < 4 ? half : units - half;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) * 32 << 16) + first * 16;
    const int chunks = (kb1 - kb0 + kChunk - 1) / kChunk;
    bool ok = true;
    for (int c = 0; c < chunks; ++c) {
      ok = NARROW_WAIT(acc_full + (c & 1) * 8, (c >> 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ptx::tc_fence_after();
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (u >= mine) break;
        uint32_t v[16];
        ptx::tmem_ld_32x16(lanes + (c & 1) * kBuf + u * 16, v);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[u * 16 + j] += __uint_as_float(v[j]);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(acc_empty + (c & 1) * 8);
    }
    if (!ok) {
      *abort_flag = 1;
    } else {  // the operands have been consumed
      float* part = reinterpret_cast<float*>(ring) + ((warp & 3) * 32 + lane) * (t.nt + 4) + first * 16;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (u >= mine) break;
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          *reinterpret_cast<float4*>(part + u * 16 + j) = make_float4(acc[u * 16 + j], acc[u * 16 + j + 1], acc[u * 16 + j + 2], acc[u * 16 + j + 3]);
      }
    }
  }
  __syncwarp();
  if (p.splits > 1) ptx::cluster_sync(); else __syncthreads();
  if (ctl->abort_flag == 0) {
    if (p.splits == 1) store_sums<1, 4, kAll, kSorted>(t, base, rows, rank, n0, start, ctl->row);
    else if (p.splits == 2) store_sums<2, 4, kAll, kSorted>(t, base, rows, rank, n0, start, ctl->row);
    else if (p.splits <= 4) store_sums<4, 2, kAll, kSorted>(t, base, rows, rank, n0, start, ctl->row);
    else store_sums<8, 2, kAll, kSorted>(t, base, rows, rank, n0, start, ctl->row);
  }
  if (p.splits > 1) ptx::cluster_sync_relaxed();  // no CTA leaves while another reads its shared memory
  ptx::tc_fence_before();
  __syncthreads();
  if (ctl->abort_flag != 0 && tid == 0) {
    atomicExch(t.status, 1);
    // give copies that may still be in flight time to land before the CTA's shared memory is released
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) {
    }
  }
  __syncthreads();
  if (warp == 9) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 2 * kBuf);
  }
}

template <int kUnits, bool kSorted>
static int launch(const CUtensorMap& mx, const CUtensorMap& mw, const TileParams& t, int64_t blocks, cudaStream_t st) {
  constexpr size_t kSmem = 1024 + kRing + sizeof(Ctl);
  static_assert(kSmem <= 227 * 1024);
  auto kern = narrow_tile_kernel<kUnits, kSorted>;
  static thread_local bool attr_set[64] = {false};  // the opt-in is per function and per device
  int dev = 0;
  SGLB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    SGLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t grid = blocks * t.p.n_tiles * t.p.splits;
  SGLB_REQUIRE(grid < (1ll << 31), "narrow product: %lld tiles are too many", (long long)grid);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3(kSorted ? kSortedThreads : kThreads, 1, 1);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)t.p.splits, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  SGLB_CUDA(cudaLaunchKernelEx(&cfg, kern, mx, mw, t));
  return SGLB200_OK;
}

int tile_product(const Params& given, int dtype, int64_t max_blocks, cudaStream_t st) {
  TileParams t{};
  t.p = given;
  Params& p = t.p;
  t.kb_total = (int)((p.K + kStageK - 1) / kStageK), t.fp16 = dtype, t.wait_probes = g_gemm_wait_probes;
  int rc = gemm_status_word(&t.status);
  if (rc) return rc;
  // Up to 256 weight rows a tile, so that the activations are fetched once (128 for sorted rows, whose warps have fewer registers); where there are
  // so few tiles that K can be split eight ways for twice as many, half as many rows, down to 32.
  const ClusterFits& fits = cluster_fits();
  const bool sorted = p.blocks.order != nullptr;
  const int most = sorted ? 128 : 256;
  int64_t n_tiles = (p.N + most - 1) / most;
  while (max_blocks * n_tiles * 2 <= fits.alone[8] && p.N > n_tiles * 32) n_tiles *= 2;
  t.nt = (int)(((p.N + n_tiles - 1) / n_tiles + 15) / 16 * 16);
  p.n_tiles = (int)((p.N + t.nt - 1) / t.nt);
  const int64_t tiles = max_blocks * p.n_tiles;
  p.splits = 1;
  for (int s = 2; s <= 8; ++s)  // as many CTAs as run at once
    if (tiles <= fits.alone[s] && t.kb_total >= s * kChunk) p.splits = s;
  t.stages = (int)std::min<uint32_t>(kMaxStages, kRing / (kXBytes + (uint32_t)t.nt * kStageK * 2));
  CUtensorMap mx, mw;
  const uint64_t xd[2] = {(uint64_t)p.K * 2, (uint64_t)p.T}, xs[1] = {(uint64_t)p.ldx * 2};
  const uint32_t xb[2] = {kStageK * 2, sorted ? kTileBlock / 4u : (uint32_t)kTileBlock};
  rc = get_tile_map(p.x, 2, xd, xs, xb, true, &mx);
  if (rc) return rc;
  const uint64_t wd[3] = {(uint64_t)p.K * 2, (uint64_t)p.N, (uint64_t)p.adapters}, ws[2] = {(uint64_t)p.K * 2, (uint64_t)(p.N * p.K * 2)};
  const uint32_t wb[3] = {kStageK * 2, (uint32_t)t.nt, 1};
  rc = get_tile_map(p.w, 3, wd, ws, wb, true, &mw);
  if (rc) return rc;
  if (sorted) return t.nt <= 64 ? launch<2, true>(mx, mw, t, max_blocks, st) : launch<4, true>(mx, mw, t, max_blocks, st);
  if (t.nt <= 64) return launch<2, false>(mx, mw, t, max_blocks, st);
  if (t.nt <= 128) return launch<4, false>(mx, mw, t, max_blocks, st);
  return launch<8, false>(mx, mw, t, max_blocks, st);
}

}  // namespace narrow
}  // namespace sglb200
