// Products of 16-bit rows with few weight rows over a long K, float32 out: the router's logits, and the first half of a low-rank adapter.
#pragma once
#include "common.cuh"

namespace sglb200 {
namespace narrow {

// Rows that share their weights come in blocks: of 32 of them for narrow_kernel, of 128 for narrow_tile_kernel.
constexpr int kSmallBlock = 32, kTileBlock = 128;

// The blocks that the rows of a batch are sorted into by adapter.  Either a plan: `order` the rows, then per block where it starts in the
// order, its rows and its adapter (-1: rows that name none), and for as many as there could be beyond the `count` that there are, 0 rows.  Or, for up to kScanRows rows, which one warp
// looks through faster than a launch of its own takes: `ids`, from which every CTA finds its block.
constexpr int kScanRows = 64;
struct Blocks {
  const int32_t* order;  // neither order nor ids: the rows as they lie, all of one adapter
  const int4* at;        // {start, rows, adapter, its rank}
  const int32_t* count;
  const int32_t* ids;
  int ids_rows, adapters;
};

// One warp's look at the rows' ids, lane l's rows l and l + 32, for blocks of up to `most` (a power of two) rows: the adapters, which of its
// adapter's rows a row is, and the rows that begin a block.
struct Scan {
  int k0, k1, nth0, nth1;
  uint32_t all0, all1, first0, first1;
  __device__ __forceinline__ int blocks() const { return __popc(first0) + __popc(first1); }
};
__device__ __forceinline__ Scan scan_ids(const Blocks& b, int most, int lane) {
  auto key = [&](int t) {
    const int id = t < b.ids_rows ? __ldg(b.ids + t) : -1;
    return id >= 0 && id < b.adapters ? id : -1;
  };
  Scan s;
  s.k0 = key(lane), s.k1 = key(lane + 32);
  s.all0 = b.ids_rows >= 32 ? 0xffffffffu : (1u << b.ids_rows) - 1;
  s.all1 = b.ids_rows >= 64 ? 0xffffffffu : b.ids_rows > 32 ? (1u << (b.ids_rows - 32)) - 1 : 0;
  const uint32_t before = (1u << lane) - 1;
  s.nth0 = __popc(__match_any_sync(0xffffffffu, s.k0) & s.all0 & before);
  s.nth1 = 0;
  if (s.all1 != 0) {
    s.nth1 = __popc(__match_any_sync(0xffffffffu, s.k1) & s.all1 & before);
#pragma unroll
    for (int i = 0; i < 32; ++i) s.nth1 += __shfl_sync(0xffffffffu, s.k0, i) == s.k1;
  }
  s.first0 = __ballot_sync(0xffffffffu, (s.nth0 & (most - 1)) == 0) & s.all0;
  s.first1 = __ballot_sync(0xffffffffu, (s.nth1 & (most - 1)) == 0) & s.all1;
  return s;
}
// Block `block`, in the order of their first rows: its rows (to `row`, ascending) and its adapter, if it is one of them.
__device__ __forceinline__ void scan_pick(const Scan& s, int block, int most, int lane, int32_t* row, int& rows, int& adapter) {
  const uint32_t before = (1u << lane) - 1;
  const bool low = block < __popc(s.first0);
  const uint32_t firsts = low ? s.first0 : s.first1;
  const uint32_t it = __ballot_sync(0xffffffffu, (firsts >> lane & 1u) && __popc(firsts & before) == (low ? block : block - __popc(s.first0)));
  if (it == 0) return;
  const int from = __ffs(it) - 1;
  adapter = __shfl_sync(0xffffffffu, low ? s.k0 : s.k1, from);
  const int nth = __shfl_sync(0xffffffffu, low ? s.nth0 : s.nth1, from);
  const bool in0 = s.k0 == adapter && (s.all0 >> lane & 1u) && s.nth0 >= nth && s.nth0 < nth + most;
  const bool in1 = s.k1 == adapter && (s.all1 >> lane & 1u) && s.nth1 >= nth && s.nth1 < nth + most;
  if (in0) row[s.nth0 - nth] = lane;
  if (in1) row[s.nth1 - nth] = lane + 32;
  rows = __popc(__ballot_sync(0xffffffffu, in0)) + __popc(__ballot_sync(0xffffffffu, in1));
}

struct Params {
  const void* x;       // [T, K], rows `ldx` apart
  const void* w;       // [adapters, N, K]
  float* y;            // [T, N]
  const int32_t* ranks;  // per adapter or nullptr: of every `rank_rows` rows of w the first ranks[adapter] count, the others give 0
  Blocks blocks;
  int64_t T, N, K, ldx;
  int64_t adapters;
  int rank_rows;
  int block;           // rows of a block
  int n_tiles, splits;
};

// A cluster has the K of one tile.  (Its number and a CTA's in it come without a division.)
__device__ __forceinline__ uint32_t cluster_id() {
  uint32_t v;
  asm("mov.u32 %0, %%clusterid.x;" : "=r"(v));
  return v;
}
__device__ __forceinline__ int cluster_rank() {
  int v;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(v));
  return v;
}

// y = x w^T in blocks of p.block rows, `max_blocks` the most blocks there can be.
int product(Params p, int dtype, int64_t max_blocks, cudaStream_t st);

// narrow_tile.cu: the same for many rows.
int tile_product(const Params& p, int dtype, int64_t max_blocks, cudaStream_t st);

}  // namespace narrow
}  // namespace sglb200
