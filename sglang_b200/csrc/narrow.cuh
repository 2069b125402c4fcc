// Products of 16-bit rows with few weight rows over a long K, float32 out: the router's logits, and the first half of a low-rank adapter.
#pragma once
#include "common.cuh"

namespace sglb200 {
namespace narrow {

// Rows that share their weights come in blocks: of 64 of them for narrow_kernel, of 128 for narrow_tile_kernel.
constexpr int kSmallBlock = 64, kTileBlock = 128;

// What the rows of a batch are sorted into: `order` the rows by adapter, then per block where it starts in the order, its rows and its
// adapter (-1: rows that name none, behind the others); `count` the number of blocks.
struct Blocks {
  const int32_t* order;    // or nullptr: the rows as they lie, all of one adapter
  const int32_t* start;
  const int32_t* rows;
  const int32_t* adapter;
  const int32_t* count;
};

struct Params {
  const void* x;       // [T, K], rows `ldx` apart
  const void* w;       // [adapters, N, K]
  float* y;            // [T, N], in the blocks' order
  const int32_t* ranks;  // per adapter or nullptr: of every `rank_rows` rows of w the first ranks[adapter] count, the others give 0
  Blocks blocks;
  int64_t T, N, K, ldx;
  int64_t adapters;
  int rank_rows;
  int block;           // rows of a block
  int n_tiles, splits;
};

// Rows of a block for T rows and N weight rows of each of `adapters` adapters.
int block_rows(int64_t T, int64_t N, int64_t K, int64_t adapters);

// y = x w^T in blocks of p.block rows, `max_blocks` the most blocks there can be.
int product(Params p, int dtype, int64_t max_blocks, cudaStream_t st);

// narrow_tile.cu: the same for many rows; a status word as gemm_rows.cu's, and its reset.
int tile_product(const Params& p, int dtype, int64_t max_blocks, cudaStream_t st);
int tile_status();
int tile_status_clear();

}  // namespace narrow
}  // namespace sglb200
