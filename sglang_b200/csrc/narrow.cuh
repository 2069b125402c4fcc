// Products of 16-bit rows with few weight rows over a long K, float32 out: the router's logits, and the first half of a low-rank adapter.
#pragma once
#include "common.cuh"

namespace sglb200 {
namespace narrow {

// Rows that share their weights come in blocks of up to kBlock.
constexpr int kBlock = 64;

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
  int rank_rows;
  int n_tiles, splits;
};

// y = x w^T, `max_blocks` the most blocks there can be.
int product(Params p, int dtype, int64_t max_blocks, cudaStream_t st);

}  // namespace narrow
}  // namespace sglb200
