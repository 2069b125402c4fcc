// Which of the two narrow products a call takes (narrow.cuh): narrow_kernel in blocks of 32 rows, or narrow_tile_kernel in blocks of 128.  Plain C++
// without CUDA, so that the rules can be tested.
#pragma once
#include <stdint.h>

namespace sglb200 {
namespace narrow {

// narrow_kernel fetches its share of the weights and of the activations anew for every 16 weight rows and every block; narrow_tile_kernel starts a
// microsecond later (tensor memory, a pipeline, 128 rows).  They are equal at about 28000 outputs, where a cluster has half of the CTAs for its K, and
// somewhat later where K is short.
//
// us here / there, in a graph of calls, both as they are:
//   K 7168   256 x 64 5.9 / 6.7, 384 x 64 6.2 / 6.7, 96 x 256 6.2 / 6.6, 192 x 160 7.8 / 6.7, 512 x 64 7.9 / 6.8, 4096 x 8 11.2 / 9.0
//   K 4096   768 x 32 4.9 / 5.5, 96 x 256 5.0 / 5.4, 192 x 160 6.1 / 5.5, 1024 x 32 6.0 / 5.6, 128 x 256 6.1 / 5.6, 4096 x 32 13.0 / 7.1
//   K 2048   512 x 64 4.7 / 4.8, 768 x 64 5.0 / 4.9, 1024 x 64 6.0 / 5.4, 128 x 256 4.8 / 4.8, 256 x 256 6.1 / 5.5, 256 x 128 4.7 / 4.8
//   K 1024   512 x 64 4.0 / 4.6, 4096 x 16 4.7 / 4.5, 768 x 64 4.0 / 4.6, 1024 x 96 4.4 / 6.0
// (For K of 1024 narrow_kernel stays ahead by up to a microsecond beyond the border, which is where it was.)
inline bool small_blocks(int64_t T, int64_t E, int64_t K) { return T * E <= (K > 2048 ? 28672 : 32768); }

// The same for the adapters' first product, of N = slices x rank weight rows, and the second, which goes with the block: mma.sync or, up to
// kMostTileRank, tcgen05 (lora.cu).  `columns`: of the output.
//
// us in blocks of 32 / of 128, tokens of three requests, of sixteen, and of sixteen in any order:
//   7168 x 2112, rank 16           256 11.2 / 17.1, 11.3 / 19.0, 12.8 / 20.9      1024 14.9 / 19.4, 15.1 / 22.4, 18.7 / 23.6
//   7168 x 36864, twice rank 32    192 20.2 / 22.4, 24.6 / 39.5, 25.2 / 41.0      320 28.4 / 24.7, 36.0 / 42.7, 38.0 / 45.7
//   7168 x 36864, twice rank 64    96 19.2 / 21.6, 39.4 / 42.0, 41.9 / 42.8       160 27.8 / 23.1, 44.6 / 43.5, 44.4 / 43.8
//   8192 x 10240, three times 64   192 19.5 / 20.8, 26.8 / 31.9, 26.7 / 34.1      288 28.7 / 21.8, 36.6 / 32.9, 37.8 / 34.8
//   4096 x 4096, rank 128          257 16.3 / 18.3, 19.1 / 20.9, 22.0 / 22.2      512 22.4 / 21.8, 22.2 / 21.6, 28.7 / 23.3
//   4096 x 6144, rank 256          512 42.5 / 47.7, 45.2 / 62.4, 56.5 / 78.0      1536 98.7 / 80.2, 104.3 / 104.1, 119.9 / 111.4
// They are equal at about 500 million multiply-adds of both products, and at three times as many where tcgen05 does not take the second.  For more than
// 512 tokens blocks of 32 rows are taken up to 16384 values of h, as they were (768 tokens of rank 32 beside 2112 columns would be 16.9 / 22.5).
constexpr int kMostTileRank = 128;
inline bool small_adapter_blocks(int64_t T, int64_t slices, int64_t rank, int64_t K, int64_t columns) {
  const int64_t each = rank * (slices * K + columns);  // multiply-adds of a token: below 2^8 (2^23 + 2^31)
  return (T <= 512 || T * slices * rank <= 16384) && T <= (rank > kMostTileRank ? 1500000000 : 500000000) / each;
}

}  // namespace narrow
}  // namespace sglb200
