// What the 4-bit kernels' host code chooses, by sizes: the width of a pair's tile (fp4_gemm.cu) and how an experts' product is taken
// (fp4_moe.cu).  Plain C++ without CUDA: what a GPU holds comes in as counts, so that the rules can be tested for any.
#pragma once
#include <stdint.h>

#include <algorithm>
#include <cmath>

namespace sglb200 {
namespace fp4 {

// Columns of a pair's tile: as many waves of them as there are, times the time of a wave in hundredths of a microsecond (0.46 a slab
// for 256 columns, 0.39 for 192, 0.33 for 128, and half a microsecond).  us over 256, 192 and 128: 4096 x 36864 x 7168 387, 433, 570;
// 257 x 10240 x 8192 29.0, 27.6, 35.9; 1024 x 10240 x 8192 42, 40, 57; 1024 x 2112 x 7168 15.3, 15.3, 14.7; 257 x 36864 x 7168 56, 65, 78.
// `slabs`: of 256 columns of K; `pairs`: that the GPU holds.
inline int pair_columns(int64_t M, int64_t N, int64_t slabs, int64_t pairs) {
  const int64_t tiles_m = (M + 255) / 256;
  int best = 256;
  int64_t best_cost = -1;
  for (int bn = 256; bn >= 128; bn -= 64) {
    const int64_t waves = (tiles_m * ((N + bn - 1) / bn) + pairs - 1) / pairs;
    const int64_t cost = waves * (slabs * (bn == 256 ? 46 : bn == 192 ? 39 : 33) + 50);
    if (best_cost < 0 || cost < best_cost) best = bn, best_cost = cost;
  }
  return best;
}

// ---- experts of a few tokens ----

constexpr int kMoeWarps = 16;                 // warps that multiply
constexpr int kStep = 256;                    // columns per step: a lane takes 64 of a row, 32 bytes of codes and four scales
constexpr int kMoeMaxStages = 6;
constexpr int64_t kMoeStageBytes = 32 * 1024 + kMoeWarps * 16 * 20;  // (the larger ones: where K is whole steps a little is left over)
constexpr int64_t kMoeCtlBytes = 8728;        // the control block
constexpr int64_t kMoeMostSmem = 227 * 1024;

constexpr int64_t moe_smem(int steps, int cols, int stages) {
  return 1024 + stages * kMoeStageBytes + (int64_t)steps * 512 * cols + kMoeWarps * 512 * ((cols + 7) / 8) + kMoeCtlBytes;
}

// Experts that `slots` picks name, taken as spread evenly.
inline double expected_live(int64_t slots, int64_t experts) {
  double none = 1.0;
  for (int64_t i = 0; i < slots; ++i) none *= 1.0 - 1.0 / experts;
  return experts * (1.0 - none);
}

// Passes of those experts: one each, and one more for every further pass_rows rows (an expert's rows taken as normally distributed).
inline double expected_passes(int64_t slots, int64_t experts, int pass_rows, double live) {
  const double mean = (double)slots / experts, sd = std::sqrt(mean * (1.0 - 1.0 / experts)) + 0.01;
  double more = 0.0;
  for (double rows = pass_rows + 0.5; rows < std::min(mean + 4.0 * sd, (double)slots); rows += pass_rows) {
    more += 1.0 / (1.0 + std::exp(std::max(-30.0, 1.702 * (rows - mean) / sd)));
  }
  return live + experts * more;
}

struct ExpertsPlan {
  int steps;      // of K
  int cols;       // columns of an instruction that a pass's rows take; 1 of the second product: one term at a time
  int pass_rows;  // activation rows per pass
  int warps_k;    // warps that split K; the others split tiles
  int sets;       // items per pass
  int stages;     // of the ring; 0: the rows do not fit
};

// The first (`up`) or second product of `slots` rows with w [experts, rows, K].
inline ExpertsPlan plan_experts(int64_t slots, int64_t experts, int64_t K, int64_t rows, bool up, int64_t sms) {
  ExpertsPlan p{};
  p.steps = (int)((K + kStep - 1) / kStep);
  // Rows per pass, and the columns that they take (two a row of h): every pass of an expert reads its weights again (from the L2,
  // by other CTAs at the same time), and columns take the place of stages; eight columns cost the same with one row in them as with
  // all. us of a layer over 8, 16 and 32 columns of x: 2 rows an expert (128 of 2048 x 768) 92, 102, 102; 4 (64 of 2048 x 1024) 85,
  // 94, 93; 12 (32 of 1376 x 1440) 107, 106, 120; 16 (16 of 2080 x 1056) 95, 90, 90; 64 (4 of 2048 x 2048) 84, 79, 80.  Of h: 4
  // rows 85, 94, 105; 8 (64 of 2048 x 1024) 114, 104, 122; 16 (32 of 7168 x 512) 184, 158, 155; 32 (8 of 4096 x 1024) 96, 97, 93;
  // 64 (one of 4096 x 1024) 53, 41, 38.  Four instead of eight leave long rows more stages, which is worth 2 % where experts have a
  // row or two (7168 x 512) and costs 14 % where they have four.
  const int terms = up ? 1 : 2;
  const double live = expected_live(slots, experts), cols_each = slots / live * terms;
  p.cols = cols_each > 18 ? 32 : cols_each > 10 ? 16 : cols_each > 3 || moe_smem(p.steps, 8, 4) <= kMoeMostSmem ? 8 : 4;
  while (p.cols > terms && (moe_smem(p.steps, p.cols, 2) > kMoeMostSmem || p.cols >= 2 * terms * slots)) p.cols /= 2;
  if (moe_smem(p.steps, p.cols, 2) > kMoeMostSmem) p.cols = 1;
  p.pass_rows = std::max(1, p.cols / terms);
  const double passes = expected_passes(slots, experts, p.pass_rows, live);
  // Warps that split K, the others taking tiles of their own: more of them make more and shorter items, which fill the GPU and its
  // last round better, but each item has an end, of two barriers and the shared memory between where K is split and of a count
  // where the slots are summed.  Times in turns of the ring: an end is 0.2 of one for the first product, 0.7 with a split K (the
  // second: 0.5, 1.2); scales that come by asynchronous copies come slower in short runs.  us of a layer over 1, 2, 4 and 8 for the
  // first product: one token, 8 experts of 7168 x 256 41, 31, 26, 24; 101 named of 7168 x 2048 451, 475, 475, 497; 11 of 4096 x
  // 2048 62, 57, 54, 57; 24 of 7136 x 544 84, 78, 66, 67.  For the second: 106 of 7168 x 2048 580, 606, 642, 723.
  double best = 0.0;
  for (int k = 1; k <= kMoeWarps && k <= p.steps; k *= 2) {
    const int per = kMoeWarps / k, sets = (int)((rows / 16 + per - 1) / per), turns = (p.steps + k - 1) / k;
    const double rounds = passes * sets / sms, slow = !up || K % kStep == 0 ? 1.0 : k == 1 ? 1.25 : k == 2 ? 1.08 : 1.0;
    const double cost = (rounds <= 1.0 ? 1.0 : rounds + 0.5) * (turns * slow + (k == 1 ? 0.2 : 0.7) + (up ? 0.0 : k == 1 ? 0.3 : 0.5));
    if (k == 1 || cost < best) best = cost, p.warps_k = k, p.sets = sets;
  }
  p.stages = kMoeMaxStages;
  while (p.stages > 2 && moe_smem(p.steps, p.cols, p.stages) > kMoeMostSmem) --p.stages;
  if (moe_smem(p.steps, p.cols, p.stages) > kMoeMostSmem) p.stages = 0;
  return p;
}

}  // namespace fp4
}  // namespace sglb200
