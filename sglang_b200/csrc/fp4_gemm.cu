// Products of 4-bit operands:  C[m, n] = out_t( alpha * sum_k a[m, k] * b[n, k] + bias[n] ),  a and b e2m1 codes times the scale of
// their group, on tcgen05.mma.kind::mxf4nvf4, which takes the scales from tensor memory and applies them inside the MMA.
//
// Many rows go to pairs of CTAs (fp4_pair.cu).  fp4_rows_kernel, for few rows or few tiles: the weights on the M side (128 of their
// rows), NT activation rows on the N side, so that nothing is multiplied for padding of few rows up to 128; K split over the CTAs of a
// cluster, which add their partial sums through distributed shared memory in a fixed order; without a split the sums go from tensor
// memory straight to the output.  Two CTAs an SM, each with a ring of 80 to 100 KB: 1 x 36864 x 7168 takes 25.1 us (0.90 of the measured
// copy rate), 64 rows 28.8 (0.82) with the same weights again and 30.4 with other ones in between, of which three are start and end.
//
// Over how many CTAs K is split follows the rule of the 8-bit kernel (rows_splits), whose slabs are as many bytes.  Measured for
// this one, us over 1, 2, 3, 4, 6 and 8 CTAs: 33 rows, 2112 x 7168 15.2, 10.8, 9.0, 8.2, 7.6 (taken), 8.2; 4096 x 14336 26.9, 17.2,
// 13.7, 12.5 (taken), 11.9, 11.6; 10240 x 8192 18.0, 15.3, 13.5 (taken), 19.0, 18.6, 23.3; 48 rows, 4096 x 4096 10.6, 9.1, 8.1, 7.6
// (taken), 8.6, 9.2; 64 rows, 7168 x 2048 8.0, 8.4, 8.5, 8.4 (taken), 13.4, 14.8; 1536 x 7168 15.8, 11.8, 9.8, 8.4, 8.0, 7.9
// (taken); 2816 x 16768 32.1, 20.4, 15.6, 13.4, 11.9 (taken), 12.5.  What it charges more than 32 rows for pushed sums, which this
// kernel does not push, changes none of twelve shapes at 33, 48, 64 and 128 rows. It loses where tiles are one or two more than
// SMs: 64 x 19200 x 7168 takes three CTAs, 25.1, and one would be 20.1.
#include <algorithm>

#include "fp4_gemm.cuh"
#include "fp4_rules.h"

namespace sglb200 {
namespace fp4 {

__device__ int g_fp4_status = 0;  // 0 ok, 1 = a pipeline wait expired

constexpr int kRowsThreads = 192;  // four warps for the epilogue, one that loads, one that multiplies

template <int kNT, int kG>
struct RowsCfg {
  static constexpr int NT = kNT, G = kG;
  static constexpr uint32_t kTokBytes = NT * kBK / 2;
  static constexpr uint32_t kScaleBytes = kStageBlocks<G> * kBlockBytes;  // of one operand
  static constexpr uint32_t kStage = kOperandBytes + kTokBytes + 2 * kScaleBytes;
  static constexpr uint32_t kPart = NT * kPartPitch * 4;
  static constexpr int kStages = 104 * 1024 / kStage;  // two CTAs per SM
  static constexpr uint32_t kRing = kStages * kStage > kPart ? kStages * kStage : kPart;
  // tensor memory: the sums, then two sets of scales (weights', activations'), used in turn
  static constexpr int kSet = 2 * kStageBlocks<G> * 4;
  static constexpr int kUsed = NT + 2 * kSet;
  static constexpr int kTmem = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : 256;
  static_assert(kStages >= 2 && kUsed <= 256);
};

struct RowsCtl {
  uint64_t full[8], empty[8], acc_full;
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __forceinline__ float load_bias(const Params& p, int n) {
  return p.out_fp16 ? __half2float(static_cast<const __half*>(p.bias)[n]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]);
}
__device__ __forceinline__ uint16_t round_out(const Params& p, float v) {
  return p.out_fp16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}
__device__ __forceinline__ void store_out(const Params& p, int64_t at, float v) { static_cast<uint16_t*>(p.C)[at] = round_out(p, v); }

// The output of a tile whose K was split over the CTAs of a cluster: their partial sums ([column][kPartPitch weight rows] at `part` in
// every CTA's shared memory) in ascending K order, the bias, one rounding.  CTA `rank` adds columns rank, rank + splits, ..; a thread
// four neighbouring weight rows of a column, whose parts are all requested before the first is added.
__device__ __forceinline__ void sum_parts(const Params& p, int n_tile, int row0, int cols, int rank, uint32_t part, int tid) {
  const int splits = p.splits, mine = (cols - rank + splits - 1) / splits;
  for (int i = tid; i < mine * 32; i += kRowsThreads) {
    const int col = rank + (i >> 5) * splits, quad = (i & 31) * 4, n = n_tile * 128 + quad;
    if (n >= p.N) continue;  // (N is a multiple of 8)
    const uint32_t at = part + (col * kPartPitch + quad) * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < splits; s0 += 8) {
      float4 v[8];
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s0 + s < splits) {
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[s].x), "=f"(v[s].y), "=f"(v[s].z), "=f"(v[s].w)
                       : "r"(ptx::cluster_map(at, s0 + s))
                       : "memory");
        }
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s0 + s < splits) sum.x += v[s].x, sum.y += v[s].y, sum.z += v[s].z, sum.w += v[s].w;
    }
    if (p.bias != nullptr) sum.x += load_bias(p, n), sum.y += load_bias(p, n + 1), sum.z += load_bias(p, n + 2), sum.w += load_bias(p, n + 3);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.C) + (int64_t)(row0 + col) * p.N + n) =
        make_uint2(round_out(p, sum.x) | (uint32_t)round_out(p, sum.y) << 16, round_out(p, sum.z) | (uint32_t)round_out(p, sum.w) << 16);
  }
}

template <class Cfg>
__global__ void __launch_bounds__(kRowsThreads, 2)
    fp4_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params p) {
  constexpr int NT = Cfg::NT, G = Cfg::G, S = Cfg::kStages;
  static_assert(S <= 8);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  RowsCtl* ctl = reinterpret_cast<RowsCtl*>(ring + Cfg::kRing);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &ctl->abort_flag;
  const int splits = p.splits, rank = (int)(blockIdx.x % splits), tile = (int)(blockIdx.x / splits);
  int m_tile, n_tile;
  tile_coord(tile, p.tiles_m, p.tiles_n, p.group_m, m_tile, n_tile);
  const int kb0 = (int)((int64_t)rank * p.kb_total / splits), kb1 = (int)((int64_t)(rank + 1) * p.kb_total / splits);
  const uint32_t bar_full = ptx::smem_u32(ctl->full), bar_empty = ptx::smem_u32(ctl->empty), bar_acc = ptx::smem_u32(&ctl->acc_full);

  if (tid == 0) {
    for (int s = 0; s < S; ++s) ptx::mbar_init(bar_full + s * 8, 1), ptx::mbar_init(bar_empty + s * 8, 1);
    ptx::mbar_init(bar_acc, 1);
    ctl->abort_flag = 0;
    ptx::mbar_fence_init();
  }
  // Tensor memory is taken once the kernel in front has ended, so that no CTA holds some while it waits for CTAs that need it;
  // the kernel behind may start when every CTA has its own.
  ptx::grid_dependency_wait();
  if (warp == 5) {
    ptx::tmem_alloc(ptx::smem_u32(&ctl->tmem_base), Cfg::kTmem);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  ptx::launch_dependents();
  const uint32_t tmem = ctl->tmem_base;

  if (warp == 4) {
    if (ptx::elect_one()) {
      const int x_block = (int)((int64_t)m_tile * NT / 128);
      for (int kb = kb0, i = 0; kb < kb1; ++kb, ++i) {
        const int s = i % S;
        if (i >= S && !FP4_WAIT(bar_empty + s * 8, ((i / S) & 1) ^ 1)) {
          *abort_flag = 1;
          break;
        }
        const uint32_t at = ptx::smem_u32(ring) + s * Cfg::kStage, bar = bar_full + s * 8;
        const uint32_t scale_bytes = stage_blocks<G>(p, kb) * kBlockBytes;
        ptx::mbar_arrive_expect_tx(bar, kOperandBytes + Cfg::kTokBytes + 2 * scale_bytes);
        ptx::tma_load_3d(at, &map_w, bar, kb * (kBK / 2), n_tile * 128, 0);
        ptx::tma_load_2d(at + kOperandBytes, &map_x, bar, kb * (kBK / 2), m_tile * NT);
        const int64_t block = (int64_t)kb * kStageBlocks<G>;
        const uint32_t sc = at + kOperandBytes + Cfg::kTokBytes;
        bulk_load(sc, p.b_s + ((int64_t)n_tile * p.group_blocks + block) * kBlockBytes, scale_bytes, bar);
        bulk_load(sc + Cfg::kScaleBytes, p.a_s + ((int64_t)x_block * p.group_blocks + block) * kBlockBytes, scale_bytes, bar);
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    if (ptx::elect_one()) {
      // rows 32 j .. of a block of activation scales have column j of each four
      const uint32_t x_col = (uint32_t)(m_tile * NT % 128 / 32);
      bool ok = true;
      for (int kb = kb0, i = 0; kb < kb1; ++kb, ++i) {
        const int s = i % S;
        ok = FP4_WAIT(bar_full + s * 8, (i / S) & 1);
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t at = ptx::smem_u32(ring) + s * Cfg::kStage, sc = at + kOperandBytes + Cfg::kTokBytes;
        const uint32_t sfw = tmem + NT + (i & 1) * Cfg::kSet, sfx = sfw + kStageBlocks<G> * 4;
        const int blocks = stage_blocks<G>(p, kb), mmas = stage_mmas(p, kb);
        for (int b = 0; b < blocks; ++b) {
          copy_scales<1>(sfw + 4 * b, ptx::pack_f32x2(desc_lo(sc + b * kBlockBytes), kDescHiScale));
          copy_scales<1>(sfx + 4 * b, ptx::pack_f32x2(desc_lo(sc + Cfg::kScaleBytes + b * kBlockBytes), kDescHiScale));
        }
        const uint32_t w_lo = desc_lo(at), x_lo = desc_lo(at + kOperandBytes);
        for (int k = 0; k < mmas; ++k) {
          const int b = G == 16 ? k : k >> 1;
          mma<1, G>(tmem, ptx::pack_f32x2(w_lo + 2 * k, kDescHiTile), ptx::pack_f32x2(x_lo + 2 * k, kDescHiTile),
                    idesc<G>(128, NT) | (G == 32 && (k & 1) ? kSecondHalf : 0u), sfw + 4 * b, sfx + 4 * b + x_col,
                    i > 0 || k > 0 ? 1u : 0u);
        }
        ptx::mma_commit(bar_empty + s * 8);
      }
      if (!ok) *abort_flag = 1;
      ptx::mma_commit(bar_acc);
    }
    __syncwarp();
  } else {
    // ------------------------------ sums out of tensor memory: lane = weight row, column = activation row ------------------------------
    if (!FP4_WAIT(bar_acc, 0)) {
      *abort_flag = 1;
    } else {
      ptx::tc_fence_after();
      const float alpha = p.alpha ? __ldcg(p.alpha) : 1.0f;
      const int n = n_tile * 128 + warp * 32 + lane, m0 = m_tile * NT;
      const float bias = splits == 1 && p.bias != nullptr && n < p.N ? load_bias(p, n) : 0.f;
      float* part = reinterpret_cast<float*>(ring) + warp * 32 + lane;  // the operands have been consumed
#pragma unroll
      for (int c = 0; c < NT; c += 16) {
        if (m0 + c >= p.M) break;  // (columns past the last row are nobody's)
        uint32_t r[16];
        ptx::tmem_ld_32x16(tmem + ((uint32_t)(warp * 32) << 16) + c, r);
        ptx::tmem_ld_wait();
        if (splits == 1) {  // a warp stores 32 neighbouring values of a row
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (n < p.N && m0 + c + j < p.M) store_out(p, (int64_t)(m0 + c + j) * p.N + n, alpha * __uint_as_float(r[j]) + bias);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) part[(c + j) * kPartPitch] = alpha * __uint_as_float(r[j]);
        }
      }
      ptx::tc_fence_before();
    }
  }

  __syncwarp();
  if (splits > 1) {
    ptx::cluster_sync();
    if (ctl->abort_flag == 0) sum_parts(p, n_tile, m_tile * NT, min(NT, (int)p.M - m_tile * NT), rank, ptx::smem_u32(ring), tid);
    ptx::cluster_sync();  // no CTA leaves while another reads its shared memory
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (ctl->abort_flag != 0 && tid == 0) {
    atomicExch(&g_fp4_status, 1);
    // give copies that may still be in flight time to land before the CTA's shared memory is released
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) {
    }
  }
  __syncthreads();
  if (warp == 5) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, Cfg::kTmem);
  }
}

template <class Cfg>
static int launch_rows(const void* A, const void* B, Params& p, cudaStream_t st) {
  CUtensorMap mw, mx;
  int rc = get_tensor_map(B, (uint64_t)p.K / 2, (uint64_t)p.N, 1, 128, 3, &mw);
  if (rc) return rc;
  rc = get_tensor_map(A, (uint64_t)p.K / 2, (uint64_t)p.M, 1, Cfg::NT, 2, &mx);
  if (rc) return rc;
  p.tiles_m = (int)((p.M + Cfg::NT - 1) / Cfg::NT), p.tiles_n = (int)((p.N + 127) / 128);
  p.group_m = choose_group_m(p.M, p.K / 2, Cfg::NT);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  p.splits = rows_splits(tiles, p.kb_total, p.M, cluster_fits());
  constexpr size_t kSmem = 1024 + Cfg::kRing + sizeof(RowsCtl);
  static_assert(kSmem <= 113 * 1024);
  auto kern = fp4_rows_kernel<Cfg>;
  static thread_local bool attr_set[64] = {false};  // the opt-ins are per function and per device
  int dev = 0;
  SGLB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    SGLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
    SGLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  SGLB_REQUIRE(tiles * p.splits < (1ll << 31), "group_fp4_scaled_mm: %lld tiles are too many", (long long)tiles);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * p.splits), 1, 1);
  cfg.blockDim = dim3(kRowsThreads, 1, 1);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.splits, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  SGLB_CUDA(cudaLaunchKernelEx(&cfg, kern, mw, mx, p));
  return SGLB200_OK;
}

// Up to 64 rows the weights on the M side.  Above that likewise, 64 rows a tile, where that makes no more tiles than SMs (their K is
// then split over clusters: 128 x 512 x 8192 6.6 us, by pairs 14.2; 512 x 2112 x 7168 13.5 and 14.3; but 65 x 10240 x 8192, 160 tiles,
// 22.6 and 17.0), and 128 rows a tile up to 128 rows (65 x 36864 x 7168 31.5 and 32.9; 128 rows 34.0 and 34.7); else pairs.
template <int G>
static int scaled_mm(const void* A, const void* B, Params& p, cudaStream_t st) {
  if (p.M <= 16) return launch_rows<RowsCfg<16, G>>(A, B, p, st);
  if (p.M <= 32) return launch_rows<RowsCfg<32, G>>(A, B, p, st);
  if (p.M <= 64 || (p.M + 63) / 64 * ((p.N + 127) / 128) <= sm_count()) return launch_rows<RowsCfg<64, G>>(A, B, p, st);
  if (p.M <= 128) return launch_rows<RowsCfg<128, G>>(A, B, p, st);
  return pair_mm(A, B, p, G, pair_columns(p.M, p.N, p.kb_total, std::max<int64_t>(1, cluster_fits().alone[2])), st);
}

}  // namespace fp4

int fp4_gemm_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, fp4::g_fp4_status, sizeof(int)) != cudaSuccess) return -1;
  return v != 0 ? v : fp4_pair_status();
}
int fp4_gemm_status_clear() {
  const int zero = 0;
  SGLB_CUDA(cudaMemcpyToSymbol(fp4::g_fp4_status, &zero, sizeof(int)));
  return fp4_pair_status_clear();
}

}  // namespace sglb200

using namespace sglb200;

extern "C" {

int sglb200_group_fp4_scaled_mm(const void* A, const void* B, const void* a_s, const void* b_s, const float* alpha, void* C,
                                const void* bias, int64_t M, int64_t N, int64_t K, int group_size, int out_dtype, void* stream) {
  if (group_size != 16 && group_size != 32)
    return fail(SGLB200_E_UNSUPPORTED, "group_fp4_scaled_mm: group_size %d is neither 16 nor 32", group_size);
  if (out_dtype != 0 && out_dtype != 1)
    return fail(SGLB200_E_UNSUPPORTED, "group_fp4_scaled_mm: output dtype must be bfloat16 or float16");
  SGLB_REQUIRE(M >= 0 && N > 0 && K > 0, "group_fp4_scaled_mm: M %lld, N %lld, K %lld", (long long)M, (long long)N, (long long)K);
  SGLB_REQUIRE(K % 32 == 0 && N % 8 == 0, "group_fp4_scaled_mm: K (%lld) must be divisible by 32 and N (%lld) by 8", (long long)K,
               (long long)N);
  SGLB_REQUIRE(M < (1ll << 31) - 256 && N < (1ll << 31) - 256 && K <= 1 << 20, "group_fp4_scaled_mm: M %lld, N %lld or K %lld is too large",
               (long long)M, (long long)N, (long long)K);
  if (M == 0) return SGLB200_OK;
  SGLB_REQUIRE(A && B && a_s && b_s && C, "group_fp4_scaled_mm: null pointer");
  SGLB_REQUIRE(aligned16(A) && aligned16(B) && aligned16(a_s) && aligned16(b_s) && aligned16(C) && aligned16(bias),
               "group_fp4_scaled_mm: pointers must be 16-byte aligned");
  SGLB_REQUIRE(((uintptr_t)alpha & 3) == 0, "group_fp4_scaled_mm: alpha is not aligned to 4 bytes");
  fp4::Params p{};
  p.a_s = static_cast<const uint8_t*>(a_s), p.b_s = static_cast<const uint8_t*>(b_s);
  p.alpha = alpha, p.C = C, p.bias = bias;
  p.M = M, p.N = N, p.K = K;
  p.group_blocks = (int)((K / group_size + 3) / 4), p.kb_total = (int)((K + fp4::kBK - 1) / fp4::kBK);
  p.out_fp16 = out_dtype;
  p.wait_probes = g_gemm_wait_probes;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return group_size == 16 ? fp4::scaled_mm<16>(A, B, p, st) : fp4::scaled_mm<32>(A, B, p, st);
}

}  // extern "C"
