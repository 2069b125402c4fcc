// What the 4-bit products share: launch parameters, the block-scaled MMA and the copy of scales into tensor memory.
#pragma once
#include "common.cuh"
#include "fp4_math.cuh"
#include "gemm_common.cuh"
#include "gemm_rows.cuh"
#include "ptx_sm100.cuh"

namespace sglb200 {
namespace fp4 {

constexpr int kBK = 256;                      // columns per stage: 128 bytes, one swizzle span
constexpr int kMmaK = 64;                     // columns per instruction
constexpr uint32_t kOperandBytes = 128 * kBK / 2;  // 128 rows of codes

// A row's blocks of 4 groups that belong to a stage, at most.
template <int kGroup>
constexpr int kStageBlocks = kBK / kGroup / 4;

struct Params {
  const uint8_t* a_s;  // scales in blocked order
  const uint8_t* b_s;
  const float* alpha;  // device, optional
  void* C;
  const void* bias;    // optional, in the output's type
  int64_t M, N, K;
  int group_blocks;    // blocks of 4 groups in a row
  int kb_total;        // stages of K
  int tiles_m, tiles_n;
  int group_m;         // m-tiles that sweep over n together
  int splits;          // CTAs of a cluster, each with its part of K
  int out_fp16;
  uint32_t wait_probes;
};

// e2m1 x e2m1 -> f32, both operands K-major, M and N of one instruction; scales e4m3 (0) or e8m0 (1 at bit 23).
template <int kGroup>
__host__ __device__ constexpr uint32_t idesc(int m, int n) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (kGroup == 32 ? 1u << 23 : 0u) | ((uint32_t)(m >> 4) << 24);
}
// Two instructions share a block of e8m0 scales (4 groups of 32 columns): the second one takes bytes 2 and 3.
constexpr uint32_t kSecondHalf = (2u << 4) | (2u << 29);

constexpr uint32_t kDescHiTile = (1024u >> 4) | (1u << 14) | (2u << 29);  // rows of 128 bytes, 128-byte swizzle
constexpr uint32_t kDescHiScale = (128u >> 4) | (1u << 14);               // 16-byte rows, eight of them 128 bytes apart
__device__ __forceinline__ uint32_t desc_lo(uint32_t smem) { return ((smem & 0x3ffffu) >> 4) | (1u << 16); }

// The blocks of 4 groups of stage kb.
template <int kGroup>
__device__ __forceinline__ int stage_blocks(const Params& p, int kb) {
  return min(kStageBlocks<kGroup>, p.group_blocks - kb * kStageBlocks<kGroup>);
}
// Instructions of stage kb: columns past K have no codes (zeros) and no scales.
__device__ __forceinline__ int stage_mmas(const Params& p, int kb) {
  return min(kBK / kMmaK, (int)((p.K - (int64_t)kb * kBK + kMmaK - 1) / kMmaK));
}

// Contiguous bytes into shared memory, completing on an mbarrier; both ends and the size multiples of 16.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// One block of scales (32 rows x 16 bytes) into 4 columns of tensor memory, repeated for each quarter of the lanes.
template <int kCtas>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  if constexpr (kCtas == 1)
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

template <int kCtas, int kGroup>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
#define FP4_MMA(CG, VEC)                                                                                                      \
  asm volatile("{\n\t.reg .pred p;\n\t"                                                                                        \
               "setp.ne.b32 p, %6, 0;\n\t"                                                                                     \
               "tcgen05.mma.cta_group::" CG ".kind::mxf4nvf4.block_scale.scale_vec::" VEC " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" \
               ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(accumulate)                                           \
               : "memory")
  if constexpr (kCtas == 1 && kGroup == 16) FP4_MMA("1", "4X");
  if constexpr (kCtas == 1 && kGroup == 32) FP4_MMA("1", "2X");
  if constexpr (kCtas == 2 && kGroup == 16) FP4_MMA("2", "4X");
  if constexpr (kCtas == 2 && kGroup == 32) FP4_MMA("2", "2X");
#undef FP4_MMA
}

#define FP4_WAIT(bar, parity) \
  (p.wait_probes != ptx::kProbesNone && (ptx::mbar_test(bar, parity) || ptx::mbar_wait_quiet(bar, parity)))


// fp4_pair.cu: the product by pairs of CTAs, in tiles of 256 rows x `bn` (128, 192 or 256) columns.
int pair_mm(const void* A, const void* B, Params& p, int group_size, int bn, cudaStream_t st);

}  // namespace fp4

int fp4_pair_status();
int fp4_pair_status_clear();

}  // namespace sglb200
