// The product of 4-bit operands for many rows: pairs of CTAs (two SMs) multiply tiles of 256 rows x BN columns.
//
// A slab of K (256 columns) is 128 bytes of each row.  With a pair, each CTA fetches its own 128 rows of A and half of B's, and one
// instruction (tcgen05.mma.cta_group::2, issued by the even CTA) multiplies 256 x BN x 64 out of both shared memories: 64 bytes
// fetched per clock and SM at the full rate of the tensor cores for BN = 256, against 96 for a CTA by itself, where some 60 arrive.
// The scales of a slab (in blocked order, so that they are contiguous) lie in the same stage; the thread that multiplies copies
// them into tensor memory, two sets in turn, right in front of the instructions that read them.
//
// 4096 x 36864 x 7168 387 us in a burst: 5.6 PFLOP/s, 3.35 times the measured bf16 burst rate (cta_group::1, 128 x 128 tiles: 995
// us); one after the other 463 to 468.  What is left is mostly power: the tensor cores are the load.  With a second staging area
// for the output there is room for four stages instead of five: 405 us there, 4096 x 24576 x 1536 107 instead of 92, 4096 x 32768 x
// 512 88 instead of 91.
//
// Persistent.  Warps: 0-7 epilogue (two groups of four, each half of the columns), 8 fetches, 9 multiplies (in the even CTA).  With
// BN = 256 there is one accumulator, which the epilogue empties into registers, rounded, before it stores anything; with 192 and
// 128 columns there are two.  Every wait is bounded; one that runs out sets sglb200_gemm_status().
#include <algorithm>

#include "fp4_gemm.cuh"

namespace sglb200 {
namespace fp4 {

__device__ int g_fp4_pair_status = 0;  // 0 ok, 1 = a pipeline wait expired

constexpr int kPairThreads = 320;

template <int kBN, int kG>
struct PairCfg {
  static constexpr int BN = kBN, G = kG;
  static constexpr int kBlocks = kStageBlocks<G>;
  static constexpr uint32_t kBBytes = BN / 2 * kBK / 2;               // this CTA's half of B
  static constexpr uint32_t kSfA = kBlocks * kBlockBytes, kSfB = 2 * kSfA;  // this CTA's 128 rows; all of the tile's columns
  static constexpr uint32_t kStage = kOperandBytes + kBBytes + kSfA + kSfB;
  static constexpr uint32_t kOut = 2 * 128 * 128;                     // staged output: 64 columns of each half
  static constexpr int kStages = (227 * 1024 - 1024 - 512 - kOut) / kStage;
  static constexpr int kAccs = BN == 256 ? 1 : 2;
  static constexpr int kSet = kBlocks * 4 * 3;                        // tensor-memory columns of a slab's scales: A's, B's
  static constexpr int kSfAt = kAccs * BN;
  static constexpr size_t kSmem = 1024 + kStages * kStage + kOut + 512;
  static_assert(kSfAt + 2 * kSet <= 512 && kStages >= 3 && kStages <= 8 && kStage % 1024 == 0);
};

struct PairCtl {
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
};

// Loads whose arrival an mbarrier of the pair's even CTA counts.
__device__ __forceinline__ void pair_load_2d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void pair_load_3d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
// One arrival at the same mbarrier of both CTAs when everything issued so far has finished.
__device__ __forceinline__ void pair_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
               : "memory");
}
__device__ __forceinline__ void cluster_arrive_bar(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void group_sync(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }

// Two sums -> a word of the output's type.
__device__ __forceinline__ uint32_t pack_out(float a, float b, int fp16) {
  if (fp16) {
    const __half2 o = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&o);
  }
  const __nv_bfloat162 o = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&o);
}
__device__ __forceinline__ float2 bias_pair(uint32_t w, int fp16) {
  if (fp16) return f16x2_to_f32(w);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

template <class Cfg>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    fp4_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                    const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                    const __grid_constant__ CUtensorMap map_c, const Params p) {
  constexpr int BN = Cfg::BN, G = Cfg::G, S = Cfg::kStages, kAccs = Cfg::kAccs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* out = ring + S * Cfg::kStage;
  PairCtl* ctl = reinterpret_cast<PairCtl*>(out + Cfg::kOut);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)(blockIdx.x & 1), pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);
  volatile int* abort_flag = &ctl->abort_flag;
  const uint32_t bar_full = ptx::smem_u32(ctl->full), bar_empty = ptx::smem_u32(ctl->empty);
  const uint32_t bar_afull = ptx::smem_u32(ctl->acc_full), bar_aempty = ptx::smem_u32(ctl->acc_empty);

  if (tid == 8 * 32) {
    ptx::tma_prefetch_desc(&map_a);
    ptx::tma_prefetch_desc(&map_b);
    ptx::tma_prefetch_desc(&map_sa);
    ptx::tma_prefetch_desc(&map_sb);
    for (int s = 0; s < S; ++s) ptx::mbar_init(bar_full + s * 8, 1), ptx::mbar_init(bar_empty + s * 8, 1);
    for (int i = 0; i < kAccs; ++i) ptx::mbar_init(bar_afull + i * 8, 1), ptx::mbar_init(bar_aempty + i * 8, 16);
    ctl->abort_flag = 0;
    ptx::mbar_fence_init();
  }
  ptx::grid_dependency_wait();  // tensor memory is taken once the kernel in front has ended (see fp4_gemm.cu)
  if (warp == 9) pair_tmem_alloc(ptx::smem_u32(&ctl->tmem_base), 512);
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync();
  ptx::tc_fence_after();
  ptx::launch_dependents();
  const uint32_t tmem = ctl->tmem_base;
  const int tiles = p.tiles_m * p.tiles_n;

  if (warp == 8) {
    // ------------------------------ operands ------------------------------
    if (ptx::elect_one()) {
      const uint32_t lead_full = ptx::cluster_map(bar_full, 0);
      int s = 0;
      uint32_t ph = 1;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int m_tile, n_tile;
        tile_coord(t, p.tiles_m, p.tiles_n, p.group_m, m_tile, n_tile);
        const int row_a = m_tile * 256 + rank * 128, row_b = n_tile * BN + rank * (BN / 2);
        for (int kb = 0; kb < p.kb_total; ++kb) {
          ok = FP4_WAIT(bar_empty + s * 8, ph);
          if (!ok) break;
          const uint32_t at = ptx::smem_u32(ring) + s * Cfg::kStage, bar = lead_full + s * 8;
          if (rank == 0) ptx::mbar_arrive_expect_tx(bar_full + s * 8, 2 * Cfg::kStage);  // of both CTAs
          pair_load_2d(at, &map_a, bar, kb * (kBK / 2), row_a);
          pair_load_2d(at + kOperandBytes, &map_b, bar, kb * (kBK / 2), row_b);
          const uint32_t sf = at + kOperandBytes + Cfg::kBBytes;
          pair_load_3d(sf, &map_sa, bar, 0, kb * Cfg::kBlocks * 2, m_tile * 2 + rank);
          pair_load_3d(sf + Cfg::kSfA, &map_sb, bar, 0, kb * Cfg::kBlocks * 2, n_tile * BN / 128);
          if (++s == S) s = 0, ph ^= 1;
        }
      }
      if (!ok) *abort_flag = 1;
    }
    __syncwarp();
  } else if (warp == 9) {
    // ------------------------------ products ------------------------------
    if (rank == 0 && ptx::elect_one()) {
      int s = 0, turn = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = pair, i = 0; t < tiles && ok; t += pairs, ++i) {
        int m_tile, n_tile;
        tile_coord(t, p.tiles_m, p.tiles_n, p.group_m, m_tile, n_tile);
        const int a = i % kAccs;
        if (i >= kAccs) ok = FP4_WAIT(bar_aempty + a * 8, ((i / kAccs) & 1) ^ 1);
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t acc = tmem + a * BN;
        const uint32_t b_col = (uint32_t)(n_tile * BN % 128 / 32);  // of B's scales, where a tile begins inside a block
        for (int kb = 0; kb < p.kb_total; ++kb, ++turn) {
          ok = FP4_WAIT(bar_full + s * 8, ph);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint32_t at = ptx::smem_u32(ring) + s * Cfg::kStage, sf = at + kOperandBytes + Cfg::kBBytes;
          const uint32_t sfa = tmem + Cfg::kSfAt + (turn & 1) * Cfg::kSet, sfb = sfa + Cfg::kBlocks * 4;
#pragma unroll
          for (int b = 0; b < Cfg::kBlocks; ++b) {
            copy_scales<2>(sfa + 4 * b, ptx::pack_f32x2(desc_lo(sf + b * kBlockBytes), kDescHiScale));
            copy_scales<2>(sfb + 8 * b, ptx::pack_f32x2(desc_lo(sf + Cfg::kSfA + b * kBlockBytes), kDescHiScale));
            copy_scales<2>(sfb + 8 * b + 4, ptx::pack_f32x2(desc_lo(sf + 2 * Cfg::kSfA + b * kBlockBytes), kDescHiScale));
          }
          const uint32_t a_lo = desc_lo(at), b_lo = desc_lo(at + kOperandBytes);
          const int mmas = stage_mmas(p, kb);
#pragma unroll
          for (int k = 0; k < kBK / kMmaK; ++k) {
            if (k >= mmas) break;
            const int b = G == 16 ? k : k >> 1;
            mma<2, G>(acc, ptx::pack_f32x2(a_lo + 2 * k, kDescHiTile), ptx::pack_f32x2(b_lo + 2 * k, kDescHiTile),
                      idesc<G>(256, BN) | (G == 32 && (k & 1) ? kSecondHalf : 0u), sfa + 4 * b, sfb + 8 * b + b_col,
                      kb > 0 || k > 0 ? 1u : 0u);
          }
          pair_commit(bar_empty + s * 8);
          if (++s == S) s = 0, ph ^= 1;
        }
        pair_commit(bar_afull + a * 8);
      }
      if (!ok) *abort_flag = 1;
    }
    __syncwarp();
  } else {
    // ------------------------------ sums out of tensor memory ------------------------------
    // The groups' columns are multiples of 64, the width of a store: 128 and 128, 128 and 64, 64 and 64.
    constexpr int kFirst = BN == 128 ? 64 : 128;
    const int group = warp >> 2, q = warp & 3, cols = group == 0 ? kFirst : BN - kFirst;
    const uint32_t lead_aempty = ptx::cluster_map(bar_aempty, 0);
    const float alpha = p.alpha ? __ldcg(p.alpha) : 1.0f;
    const uint32_t stage = ptx::smem_u32(out) + group * (128 * 128);
    const int row = q * 32 + lane;
    bool ok = true;
    for (int t = pair, i = 0; t < tiles; t += pairs, ++i) {
      int m_tile, n_tile;
      tile_coord(t, p.tiles_m, p.tiles_n, p.group_m, m_tile, n_tile);
      const int a = i % kAccs, n0 = n_tile * BN + group * kFirst;
      if (ok) ok = FP4_WAIT(bar_afull + a * 8, (i / kAccs) & 1);
      if (!ok) break;
      ptx::tc_fence_after();
      const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + a * BN + group * kFirst;
      uint32_t word[kFirst / 2];
#pragma unroll
      for (int c = 0; c < kFirst; c += 32) {
        if (c >= cols) break;  // (the same for the whole group)
        uint32_t r[32];
        ptx::tmem_ld_32x32(from + c, r);
        ptx::tmem_ld_wait();
        if (p.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            const int n = n0 + c + j;  // (N is a multiple of 8)
            uint4 bw = make_uint4(0, 0, 0, 0);
            if (n < p.N) bw = __ldcg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.bias) + n));
            const uint32_t b4[4] = {bw.x, bw.y, bw.z, bw.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 b = bias_pair(b4[k], p.out_fp16);
              word[(c + j) / 2 + k] = pack_out(__uint_as_float(r[j + 2 * k]) * alpha + b.x, __uint_as_float(r[j + 2 * k + 1]) * alpha + b.y, p.out_fp16);
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k)
            word[c / 2 + k] = pack_out(__uint_as_float(r[2 * k]) * alpha, __uint_as_float(r[2 * k + 1]) * alpha, p.out_fp16);
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) cluster_arrive_bar(lead_aempty + a * 8);
      // 64 columns at a time through the staging area (rows of 128 bytes, swizzled) and out by TMA, which clips at the edges
#pragma unroll
      for (int c = 0; c < kFirst; c += 64) {
        if (c >= cols) break;
        if (warp % 4 == 0 && lane == 0) ptx::tma_store_wait_read();
        group_sync(1 + group);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          ptx::sts_128(stage + row * 128 + ((j ^ (row & 7)) << 4),
                       make_uint4(word[c / 2 + 4 * j], word[c / 2 + 4 * j + 1], word[c / 2 + 4 * j + 2], word[c / 2 + 4 * j + 3]));
        ptx::fence_async_smem();
        group_sync(1 + group);
        if (warp % 4 == 0 && lane == 0) {
          ptx::tma_store_2d(&map_c, stage, n0 + c, m_tile * 256 + rank * 128);
          ptx::tma_store_commit();
        }
      }
    }
    if (!ok) *abort_flag = 1;
    if (warp % 4 == 0 && lane == 0) ptx::tma_store_wait_read();
  }

  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  if (ctl->abort_flag != 0 && tid == 0) {
    atomicExch(&g_fp4_pair_status, 1);
    // give copies that may still be in flight time to land before the CTA's shared memory is released
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) {
    }
  }
  __syncthreads();
  ptx::cluster_sync();  // neither CTA leaves while the other's instructions read its memory
  if (warp == 9) {
    ptx::tc_fence_after();
    pair_tmem_dealloc(tmem, 512);
  }
}

template <class Cfg>
static int launch_pair(const void* A, const void* B, Params& p, cudaStream_t st) {
  CUtensorMap ma, mb, msa, msb, mc;
  const uint64_t half = (uint64_t)p.K / 2;
  int rc = get_tensor_map(A, half, (uint64_t)p.M, 1, 128, 2, &ma);
  if (rc == SGLB200_OK) rc = get_tensor_map(B, half, (uint64_t)p.N, 1, Cfg::BN / 2, 2, &mb);
  // scales: 256 bytes, the two halves of each block of a row of blocks, rows of blocks
  const auto scales = [&](const void* s, int64_t rows, uint32_t row_blocks, CUtensorMap* out) {
    const uint64_t dims[3] = {256, (uint64_t)p.group_blocks * 2, (uint64_t)(rows + 127) / 128}, strides[2] = {256, (uint64_t)p.group_blocks * kBlockBytes};
    const uint32_t box[3] = {256, Cfg::kBlocks * 2, row_blocks};
    return get_tile_map(s, 3, dims, strides, box, false, out);
  };
  if (rc == SGLB200_OK) rc = scales(p.a_s, p.M, 1, &msa);
  if (rc == SGLB200_OK) rc = scales(p.b_s, p.N, 2, &msb);
  if (rc == SGLB200_OK) rc = get_out_map(p.C, (uint64_t)p.N, (uint64_t)p.M, p.out_fp16, 128, &mc);
  if (rc != SGLB200_OK) return rc;
  p.tiles_m = (int)((p.M + 255) / 256), p.tiles_n = (int)((p.N + Cfg::BN - 1) / Cfg::BN);
  p.group_m = choose_group_m(p.M, p.K / 2, 256);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  SGLB_REQUIRE(tiles < (1ll << 31), "group_fp4_scaled_mm: %lld tiles are too many", (long long)tiles);
  auto kern = fp4_pair_kernel<Cfg>;
  static thread_local bool attr_set[64] = {false};  // the opt-in is per function and per device
  int dev = 0;
  SGLB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    SGLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg::kSmem));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t pairs = std::min(tiles, std::max<int64_t>(1, cluster_fits().alone[2]));
  SGLB_CUDA(launch_pdl(kern, (unsigned)(2 * pairs), kPairThreads, Cfg::kSmem, st, ma, mb, msa, msb, mc, p));
  return SGLB200_OK;
}

int pair_mm(const void* A, const void* B, Params& p, int group_size, int bn, cudaStream_t st) {
#define GO(BN) return group_size == 16 ? launch_pair<PairCfg<BN, 16>>(A, B, p, st) : launch_pair<PairCfg<BN, 32>>(A, B, p, st)
  if (bn == 128) GO(128);
  if (bn == 192) GO(192);
  GO(256);
#undef GO
}

}  // namespace fp4

int fp4_pair_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, fp4::g_fp4_pair_status, sizeof(int)) != cudaSuccess) return -1;
  return v;
}
int fp4_pair_status_clear() {
  const int zero = 0;
  SGLB_CUDA(cudaMemcpyToSymbol(fp4::g_fp4_pair_status, &zero, sizeof(int)));
  return SGLB200_OK;
}

}  // namespace sglb200
