// The adapters' second product for many rows, out = base + h B^T (lora.cu), on tcgen05.mma.kind::f16: bound by reading base and writing out.
//
// A tile is 128 sorted tokens by 128 columns.  The tiles of all blocks, columns fastest, are cut evenly over one CTA an SM, whatever the
// blocks' sizes; a CTA builds the two terms of h anew where a block or a merged projection begins.  One warp copies the weights into a ring,
// one multiplies into two buffers of tensor memory, sixteen add base and store.
//
// The columns of 32 are multiplied in the order i + 2 q + 8 j for column 8 q + 2 j + i: a lane that reads two neighbouring columns of each
// eight from tensor memory then holds eight neighbouring ones of out, and base and out go by 16 bytes a lane, 64 a row.  Base comes by
// asynchronous copies, each lane's to a place of its own, three tiles ahead (one, where the rank is above 64): loaded into registers, however
// early, it was waited for in one piece, and 4096 tokens beside 36864 columns took 146 us and more.  Now 2048 tokens take 65 us
// and 4096 about 120 (5.1 TB/s), where a plain copy in this pattern of tiles takes 107 to 111.
#include <algorithm>

#include "gemm_common.cuh"
#include "lora.cuh"
#include "ptx_sm100.cuh"

namespace sglb200 {
namespace lora {

namespace {

constexpr int kRows = narrow::kTileBlock, kCols = 128;
constexpr int kAdders = 16, kThreads = (kAdders + 2) * 32;  // warps that add and store, one that copies weights, one that multiplies
constexpr uint32_t kSpan = 128 * 128;  // 128 rows of 64 columns of the rank, one swizzle span wide

// kKB: spans of 64 columns of the rank.
template <int kKB>
struct Cfg {
  static constexpr int kStages = kKB == 1 ? 3 : 2;  // of weights
  static constexpr int kAhead = kKB == 1 ? 4 : 2;   // tiles of base
  static constexpr uint32_t kBase = (2 + kStages) * kKB * kSpan, kSmem = 1024 + kBase + kAhead * kRows * kCols * 2;
  static_assert(kSmem + 4096 <= 227 * 1024);
};

#define LORA_WAIT(bar, parity) \
  (p.wait_probes != ptx::kProbesNone && (ptx::mbar_test(bar, parity) || ptx::mbar_wait_quiet(bar, parity)))

// A run of tiles of one block and one merged projection.
struct Run {
  int adapter, rows, start, used;
  int column, end;   // the first column, and the projection's end
  int slice, count;  // tiles
  bool multiply;     // (else out = base)
};

// The run that begins at tile `at` of all, of which `end` are this CTA's.
__device__ __forceinline__ Run run_at(const Params& p, int at, int end) {
  Run r;
  const int per = p.chunk0[p.S], block = at / per, tile = at - block * per;
  int s = 0;
  while (s + 1 < p.S && tile >= p.chunk0[s + 1]) ++s;
  r.slice = s;
  r.column = (int)p.col0[s] + (tile - p.chunk0[s]) * kCols, r.end = (int)p.col0[s + 1];
  r.count = min(p.chunk0[s + 1] - tile, end - at);
  const int4 of = __ldcg(p.blocks.at + block);
  r.start = of.x, r.rows = of.y, r.adapter = of.z, r.used = of.w;
  r.multiply = r.used > 0;
  return r;
}

struct Ctl {
  uint64_t full[3], empty[3], acc_full[2], acc_empty[2], h_full;
  uint32_t tmem_base;
  int abort_flag;
  float unscale[2][kRows];
};

template <typename T, int kKB>
__global__ void __launch_bounds__(kThreads, 1) expand_tile_kernel(const Params p) {
  constexpr int kStages = Cfg<kKB>::kStages, kAhead = Cfg<kKB>::kAhead;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Ctl ctl;
  uint8_t* spans = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t h_at = ptx::smem_u32(spans), ring = h_at + 2 * kKB * kSpan;
  const int tid = threadIdx.x, warp = ptx::warp_index(), lane = tid & 31;
  volatile int* abort_flag = &ctl.abort_flag;
  const uint32_t full = ptx::smem_u32(ctl.full), empty = ptx::smem_u32(ctl.empty), acc_full = ptx::smem_u32(ctl.acc_full),
                 acc_empty = ptx::smem_u32(ctl.acc_empty), h_full = ptx::smem_u32(&ctl.h_full);
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) ptx::mbar_init(full + s * 8, 32), ptx::mbar_init(empty + s * 8, 1);
    for (int b = 0; b < 2; ++b) ptx::mbar_init(acc_full + b * 8, 1), ptx::mbar_init(acc_empty + b * 8, kAdders);
    ptx::mbar_init(h_full, kAdders);
    ctl.abort_flag = 0;
    ptx::mbar_fence_init();
  }
  ptx::grid_dependency_wait();
  if (warp == kAdders + 1) {
    ptx::tmem_alloc(ptx::smem_u32(&ctl.tmem_base), 2 * kCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  ptx::launch_dependents();
  const uint32_t tmem = ctl.tmem_base;
  int begin, end;
  share(__ldcg(p.blocks.count) * p.chunk0[p.S], begin, end);

  if (warp == kAdders) {
    // ------------------------------ weights: chunks of 16 bytes, row n to its place in the order above ------------------------------
    int i = 0;
    bool ok = true;
    for (int at = begin; at < end && ok;) {
      const Run r = run_at(p, at, end);
      at += r.count;
      if (!r.multiply) continue;
      const T* weights = static_cast<const T*>(p.b) + (int64_t)r.adapter * p.N * p.R;
      const int chunks = (r.used + 15) / 16 * 2;  // of a row
      for (int c = 0; c < r.count; ++c, ++i) {
        const int s = i % kStages;
        if (i >= kStages) ok = LORA_WAIT(empty + s * 8, ((i / kStages) & 1) ^ 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int n0 = r.column + c * kCols, cols = min(kCols, r.end - n0);
        const uint32_t to = ring + s * kKB * kSpan;
        if (cols == kCols && r.used % 8 == 0) {
          // Lane l: 16 bytes l % 8 of every span of rows l / 8, + 4, ..; what the order makes of them differs by constants.
          const int k = lane & 7, l = lane >> 3;
#pragma unroll
          for (int span = 0; span < kKB; ++span) {
            const int chunk = span * 8 + k;
            if (chunk >= chunks) break;
            const uint32_t bytes = chunk * 8 < r.used ? 16 : 0;
            const T* src = bytes ? weights + (int64_t)(n0 + l) * p.R + chunk * 8 : weights;
            const int64_t step = bytes ? 4 * p.R : 0;
            const uint32_t dst = to + span * kSpan + ((l & 1) | (l & 2) << 2) * 128 + ((k ^ (l & 1)) << 4);
#pragma unroll
            for (int it = 0; it < kCols / 4; ++it) {
              constexpr auto place = [](int n) { return (n & ~31) | ((n & 6) << 2) | ((n & 24) >> 2) | (n & 1); };
              const uint32_t pos = place(it * 4);  // (a multiple of two, below 8 the bits that l does not set)
              ptx::cp_async_16((dst + pos * 128) ^ ((pos & 7) << 4), src, bytes);
              src += step;
            }
          }
        } else {
          for (int id = lane; id < kCols * chunks; id += 32) {
            const int n = id / chunks, k = id - n * chunks;
            const int pos = (n & ~31) | ((n & 6) << 2) | ((n & 24) >> 2) | (n & 1);
            const uint32_t dst = to + (k >> 3) * kSpan + pos * 128 + (((k & 7) ^ (pos & 7)) << 4);
            const int left = n < cols ? r.used - k * 8 : 0;  // values that count of these eight
            const T* src = weights + (int64_t)(n0 + n) * p.R + k * 8;
            if (left <= 0 || left >= 8) {
              ptx::cp_async_16(dst, left > 0 ? src : weights, left > 0 ? 16 : 0);
            } else {  // (beyond the rank anything may stand)
              uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
              uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
              for (int j = 0; j < 4; ++j) w[j] = 2 * j + 1 < left ? w[j] : 2 * j < left ? w[j] & 0xffffu : 0u;
              ptx::sts_128(dst, v);
            }
          }
        }
        if (r.used % 8 == 0) {
          ptx::cp_async_arrive(full + s * 8);
        } else {  // (ordinary stores among them)
          asm volatile("cp.async.wait_all;" ::: "memory");
          ptx::fence_async_smem();
          ptx::mbar_arrive(full + s * 8);
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!ok && lane == 0) *abort_flag = 1;
    __syncwarp();
  } else if (warp == kAdders + 1) {
    if (ptx::elect_one()) {
      const uint32_t id = ptx::idesc_f16(kRows, kCols, std::is_same<T, __half>::value);
      int i = 0, runs = 0;
      bool ok = true;
      for (int at = begin; at < end && ok;) {
        const Run r = run_at(p, at, end);
        at += r.count;
        if (!r.multiply) continue;
        ok = LORA_WAIT(h_full, runs & 1);
        ++runs;
        const int steps = (r.used + 15) / 16;
        for (int c = 0; c < r.count && ok; ++c, ++i) {
          const int s = i % kStages, buf = i & 1;
          if (i >= 2) ok = LORA_WAIT(acc_empty + buf * 8, ((i >> 1) & 1) ^ 1);
          if (ok) ok = LORA_WAIT(full + s * 8, (i / kStages) & 1);
          if (!ok) break;
          ptx::fence_async_smem();  // (the copies' writes, which the barrier has shown, before the tensor core's reads)
          ptx::tc_fence_after();
#pragma unroll 1
          for (int term = 1; term >= 0; --term)  // the low terms first
#pragma unroll 1
            for (int k = 0; k < steps; ++k) {
              const uint32_t a = ptx::desc_lo128(h_at + (term * kKB + k / 4) * kSpan) + 2 * (k % 4);
              const uint32_t b = ptx::desc_lo128(ring + (s * kKB + k / 4) * kSpan) + 2 * (k % 4);
              ptx::mma_f16(tmem + buf * kCols, ptx::pack_f32x2(a, ptx::kDescHi128), ptx::pack_f32x2(b, ptx::kDescHi128), id,
                           term == 0 || k > 0 ? 1u : 0u);
            }
          ptx::mma_commit(empty + s * 8);
          ptx::mma_commit(acc_full + buf * 8);
        }
      }
      if (!ok) *abort_flag = 1;
    }
    __syncwarp();
  } else {
    // ------------------------------ out = base + sums ------------------------------
    const int g = lane >> 2, q = lane & 3, quarter = warp & 3, wide = warp >> 2;  // 32 rows and 32 columns of a tile
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + wide * 32;
    const int row_mine = quarter * 32 + g, col_mine = wide * 32 + q * 8;  // and the rows 8, 16 and 24 below
    const uint32_t base_pitch = (uint32_t)(p.ld_base * 2), out_pitch = (uint32_t)(p.ld_out * 2);
    const uint32_t mine = h_at + Cfg<kKB>::kBase + warp * 2048 + lane * 16;
    // The terms of h of a run, and its rows' factors to `set`.
    auto build = [&](const Run& r, int of_rows, int set) {  // lane u of `of_rows`: the token of row warp + u * kAdders
      const int used = r.used, rows = r.rows;
      const float scaling = p.scalings != nullptr ? __ldg(p.scalings + r.adapter) : 1.f;
      const float* h = p.h + r.slice * p.R;
      constexpr int kRowsHere = kRows / kAdders, kV = 2 * kKB;
      float v[kRowsHere][kV];
#pragma unroll
      for (int u = 0; u < kRowsHere; ++u) {
        const float* from = h + (int64_t)__shfl_sync(0xffffffffu, of_rows, u) * p.S * p.R;
#pragma unroll
        for (int j = 0; j < kV; ++j) v[u][j] = j * 32 + lane < used ? __ldcg(from + j * 32 + lane) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kRowsHere; ++u) {
        const int row = warp + u * kAdders;
        if (row >= rows) break;
#pragma unroll
        for (int j = 0; j < kV; ++j) v[u][j] *= scaling;
        const uint32_t at_row = (uint32_t)row * 128;
        const float inv = split_row<T>(v[u], (used + 15) / 16 * 16, lane, [&](int k, uint16_t hi, uint16_t lo) {
          const uint32_t o = (k >> 6) * kSpan + at_row + ((((k >> 3) & 7) ^ (row & 7)) << 4) + (k & 7) * 2;
          *reinterpret_cast<uint16_t*>(spans + o) = hi;
          *reinterpret_cast<uint16_t*>(spans + kKB * kSpan + o) = lo;
        });
        if (lane == 0) ctl.unscale[set][row] = inv;
      }
      ptx::fence_async_smem();
      asm volatile("bar.sync 1, %0;" ::"n"(kAdders * 32) : "memory");
      if (lane == 0) ptx::mbar_arrive(h_full);
    };
    // A run for a lane: its rows' tokens, its first column and where it stops (0: nothing to do).
    struct Mine {
      uint32_t token[4];
      int rows, n, stop, of_rows;
    };
    auto open = [&](const Run& r, Mine& m) {
      m.of_rows = __ldcg(p.blocks.order + r.start + min(warp + lane % (kRows / kAdders) * kAdders, r.rows - 1));
      m.rows = r.rows - row_mine, m.n = r.column + col_mine, m.stop = r.multiply || !p.in_place ? r.end : 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) m.token[j] = j * 8 < m.rows ? (uint32_t)__ldcg(p.blocks.order + r.start + row_mine + j * 8) : 0u;
    };
    // The run that is asked for, and what the run behind this one is, if it has been opened already.
    Run ahead_run{}, next_run{};
    Mine ahead, next;
    int ahead_at = begin, ahead_left = 0, next_at = -1;
    // Asks for the base of the next tile that has not been asked for, to place `slot`.
    auto fetch = [&](int slot) {
      if (ahead_at < end) {
        if (ahead_left == 0) {
          ahead_run = run_at(p, ahead_at, end);
          open(ahead_run, ahead);
          ahead_left = ahead_run.count;
          if (next_at < 0) next_at = ahead_at, next_run = ahead_run, next = ahead;
        }
        if (ahead.n < ahead.stop) {
          const uint8_t* from = static_cast<const uint8_t*>(p.base) + (int64_t)ahead.n * 2;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j * 8 < ahead.rows) ptx::cp_async_16(mine + slot * (kRows * kCols * 2) + j * 512, from + (uint64_t)ahead.token[j] * base_pitch, 16);
        }
        ++ahead_at, --ahead_left, ahead.n += kCols;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int t = 0; t < kAhead - 1; ++t) fetch(t);
    int i = 0, built = 0, slot = 0;
    bool ok = true;
    for (int at = begin; at < end;) {
      Run r;
      Mine m;
      if (next_at == at) {
        r = next_run, m = next;
      } else {  // (runs shorter than what is asked for ahead)
        r = run_at(p, at, end);
        open(r, m);
      }
      next_at = -1;
      at += r.count;
      const bool multiply = r.multiply;
      float inv[4] = {};
      if (multiply) {  // (the products of the run before are done: its last sums have been waited for)
        build(r, m.of_rows, built & 1);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j * 8 < m.rows) inv[j] = ctl.unscale[built & 1][row_mine + j * 8];
        ++built;
      }
      for (int c = 0; c < r.count; ++c, m.n += kCols) {
        fetch(slot == 0 ? kAhead - 1 : slot - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        const int buf = i & 1;
        // (a wait that ran out ends the waiting and storing, not the loops: the warps meet in `build`)
        if (multiply && ok) {
          ok = LORA_WAIT(acc_full + buf * 8, (i >> 1) & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) *abort_flag = 1;
        }
        ptx::tc_fence_after();
        uint8_t* to = static_cast<uint8_t*>(p.out) + (int64_t)m.n * 2;
        const bool store = m.n < m.stop && ok;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          uint32_t sum[16];
          __syncwarp();
          if (multiply) {
            ptx::tmem_ld_16x256<4>(lanes + ((uint32_t)(hh * 16) << 16) + buf * kCols, sum);
            ptx::tmem_ld_wait();
            if (hh == 1) {
              ptx::tc_fence_before();
              __syncwarp();
              if (lane == 0) ptx::mbar_arrive(acc_empty + buf * 8);
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int j = 2 * hh + e;
            if (store && j * 8 < m.rows) {
              uint4 now = ptx::lds_128(mine + slot * (kRows * kCols * 2) + j * 512);
              if (multiply) {
                uint32_t* w = reinterpret_cast<uint32_t*>(&now);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  float2 v = unpack2<T>(w[k]);
                  ptx::fma2(v.x, v.y, sum[4 * k + 2 * e], sum[4 * k + 2 * e + 1], inv[j]);
                  w[k] = pack2<T>(v.x, v.y);
                }
              }
              *reinterpret_cast<uint4*>(to + (uint64_t)m.token[j] * out_pitch) = now;
            }
          }
        }
        if (multiply) ++i;
        slot = slot + 1 == kAhead ? 0 : slot + 1;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (ctl.abort_flag != 0 && tid == 0) {
    atomicExch(p.status, 1);
    // give products that may still be in flight time to end before tensor and shared memory are released
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) {
    }
  }
  __syncthreads();
  if (warp == kAdders + 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 2 * kCols);
  }
}

template <typename T, int kKB>
int launch(const Params& p, cudaStream_t st) {
  auto kern = expand_tile_kernel<T, kKB>;
  static thread_local bool attr_set[64] = {false};  // the opt-in is per function and per device
  int dev = 0;
  SGLB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    SGLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<kKB>::kSmem));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t tiles = (int64_t)p.max_blocks * p.chunk0[p.S], ctas = sm_count();
  SGLB_REQUIRE(tiles < (1ll << 31), "lora_add: %lld tiles are too many", (long long)tiles);
  SGLB_CUDA(launch_pdl(kern, (unsigned)std::min(tiles, ctas), kThreads, (size_t)Cfg<kKB>::kSmem, st, p));
  return SGLB200_OK;
}

}  // namespace

int expand_tile(Params& p, int dtype, cudaStream_t st) {
  int tiles = 0;
  for (int s = 0; s < p.S; ++s) {
    p.chunk0[s] = tiles;
    tiles += (int)((p.col0[s + 1] - p.col0[s] + kCols - 1) / kCols);
  }
  p.chunk0[p.S] = tiles;
  const int rc = gemm_status_word(&p.status);
  if (rc) return rc;
  if (p.R <= 64) return dtype == 0 ? launch<__nv_bfloat16, 1>(p, st) : launch<__half, 1>(p, st);
  return dtype == 0 ? launch<__nv_bfloat16, 2>(p, st) : launch<__half, 2>(p, st);
}

}  // namespace lora
}  // namespace sglb200
