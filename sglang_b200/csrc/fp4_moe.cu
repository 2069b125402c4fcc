// The routed experts of a few tokens, 4-bit weights (e2m1, groups of 16 with e4m3 scales in rows' order, a factor per expert) and
// 16-bit activations, in two launches:
//
//   h[s, i]   = silu(a13_e * sum_k G_e[i, k] x[t, k]) * (a13_e * sum_k U_e[i, k] x[t, k])     for slot s = (t, j), e = ids[s]
//   out[t, n] = factor * sum_j weights[s] * a2_e * sum_i W2_e[n, i] h[s, i]
//
// Few tokens name many experts once or twice each, so a layer is one read of those experts' weights: 0.5625 bytes a weight, and
// the weights come in faster (12 T/s) than they could be expanded for anything but the matrix instructions.  A weight times its group's
// scale has six significant bits and lies within fp16, so it goes into mma.m16n8k16 exactly; the weights are the 16-row side, read
// straight from their rows in the order in which the instruction's lanes hold them (the order of k within a sum is free), and up to
// eight activation rows are the other.  bf16 activations become fp16 under a power of two per row that brings the row's largest
// magnitude to 2^14: exact down to 2^-28 of it and off by at most 2^-39 of it below.  h is kept in float32 and enters the second
// product as fp16 likewise (2^-12 of a value, an eighth of what rounding the output to bf16 costs).
//
// A CTA's item is one expert and a few 16-row tiles; its warps split the tiles and K.  Partial sums meet in shared memory in a fixed
// order.  The second launch writes every slot's product to a scratch, and whichever CTA is the last of a set of columns adds the
// slots of a token in their order, so results do not depend on the order of CTAs.
#include <algorithm>
#include <type_traits>

#include "fp4_math.cuh"
#include "ptx_sm100.cuh"

namespace sglb200 {
namespace fp4 {

constexpr int kMoeWarps = 8, kMoeThreads = kMoeWarps * 32;
constexpr int kMoeMaxExperts = 1024, kMoeMaxSlots = 1024;
constexpr int kChunk = 128;   // columns per step: four lanes of 16 bytes of codes
constexpr int kMoeRows = 8;   // activation rows per pass

struct MoeParams {
  const void* x;            // up: [tokens, K] 16-bit; down: h [slots, K] float32
  const uint8_t* w;         // [experts, rows, K / 2]
  const uint8_t* ws;        // [experts, rows, K / 16]
  const float* alpha;       // [experts] or nullptr
  const int32_t* ids;       // [slots]
  const float* weights;     // [slots] (down)
  float* h;                 // up: [slots, rows / 2]; down: products [slots, rows]
  void* out;                // down: [tokens, rows]
  int32_t* done;            // a counter per set of columns (zeroed by the up launch)
  int done_count;
  int64_t K, rows;          // rows of w: 2 I or H
  int slots, topk, experts, tokens;
  int chunks;               // of K
  int warps_k;              // warps that split K; the others split tiles
  int sets;                 // items per expert
  float factor;
};

struct MoeTables {
  uint16_t count[kMoeMaxExperts];   // slots of an expert, then where they begin
  uint16_t live[kMoeMaxExperts];    // experts that are named, ascending
  uint16_t begin[kMoeMaxExperts + 1];
  uint16_t slot[kMoeMaxSlots];      // slots in experts' order
  int warp_sum[kMoeWarps];
  int row_exp[kMoeRows][kMoeWarps]; // largest magnitudes, as float bits
  int num_live, last;
};

// Which experts are named and by which slots; ids outside the experts are skipped.  (The order of an expert's slots depends on the
// order of the atomics; it decides only which column of an instruction a slot takes, and columns do not mix.)
__device__ __forceinline__ void route(const MoeParams& p, MoeTables* tb) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t* count32 = reinterpret_cast<uint32_t*>(tb->count);
  for (int i = tid; i < kMoeMaxExperts / 2; i += kMoeThreads) count32[i] = 0;
  __syncthreads();
  int place[kMoeMaxSlots / kMoeThreads], id[kMoeMaxSlots / kMoeThreads];
#pragma unroll
  for (int j = 0; j < kMoeMaxSlots / kMoeThreads; ++j) {
    const int s = tid + j * kMoeThreads;
    id[j] = s < p.slots ? p.ids[s] : -1;
    if ((uint32_t)id[j] < (uint32_t)p.experts) {
      const uint32_t shift = (id[j] & 1) * 16;
      place[j] = (int)(atomicAdd(&count32[id[j] >> 1], 1u << shift) >> shift & 0xffffu);
    } else {
      id[j] = -1;
    }
  }
  __syncthreads();
  // exclusive scan over the experts, four a thread: (named, slots) packed
  int mine = 0, c[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int e = tid * 4 + k;
    c[k] = tb->count[e];
    mine += c[k] ? (1 << 16) + c[k] : 0;
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) tb->warp_sum[warp] = incl;
  __syncthreads();
  int before = incl - mine;
  for (int w = 0; w < warp; ++w) before += tb->warp_sum[w];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (c[k]) {
      tb->live[before >> 16] = (uint16_t)(tid * 4 + k);
      tb->begin[before >> 16] = (uint16_t)(before & 0xffff);
    }
    tb->count[tid * 4 + k] = (uint16_t)(before & 0xffff);
    before += c[k] ? (1 << 16) + c[k] : 0;
  }
  if (tid == kMoeThreads - 1) {
    tb->num_live = before >> 16;
    tb->begin[before >> 16] = (uint16_t)(before & 0xffff);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kMoeMaxSlots / kMoeThreads; ++j)
    if (id[j] >= 0) tb->slot[tb->count[id[j]] + place[j]] = (uint16_t)(tid + j * kMoeThreads);
  __syncthreads();
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t lds_32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Where a slot's activations are: the token's row, or the slot's row of h.
template <typename T>
__device__ __forceinline__ const T* act_row(const MoeParams& p, int slot) {
  const int row = std::is_same<T, float>::value ? slot : slot / p.topk;
  return static_cast<const T*>(p.x) + (int64_t)row * p.K;
}

// Eight activations as float32.
template <typename T>
__device__ __forceinline__ void load8(const T* src, float (&v)[8]) {
  if constexpr (std::is_same<T, float>::value) {
    const float4 a = __ldcg(reinterpret_cast<const float4*>(src)), b = __ldcg(reinterpret_cast<const float4*>(src) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 q = __ldcg(reinterpret_cast<const uint4*>(src));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 f = f16x2_to_f32(w[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
}

// The power of two that brings `amax` into [2^14, 2^15); 1 where it is zero or not finite.
__device__ __forceinline__ int row_shift(float amax) {
  const int e = (int)(__float_as_uint(amax) >> 23) & 0xff;
  return e == 0xff || amax == 0.f ? 0 : min(max(14 + 127 - e, -126), 126);
}
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }

// Rows [r0, r0 + n) of the expert's slots, as fp16 in the order in which lanes take them: 16-byte pieces of 8 columns, piece
// (chunk, jj, row, t) = columns chunk * 128 + t * 32 + jj * 8 ..; columns past K are zeros.  All threads; ends with a barrier.
template <typename T>
__device__ __forceinline__ void stage_rows(const MoeParams& p, MoeTables* tb, int r0, int n, uint4* xs) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int pieces = p.chunks * 16;  // of a row
  __syncthreads();                   // the rows before these have been used
  if constexpr (!std::is_same<T, __half>::value) {
    for (int r = 0; r < n; ++r) {
      const T* src = act_row<T>(p, tb->slot[r0 + r]);
      float amax = 0.f;
      for (int q = tid; q * 8 < p.K; q += kMoeThreads) {
        float v[8];
        load8(src + q * 8, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
        // a NaN is not seen here and stays one under any power of two
      }
      amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
      if (lane == 0) tb->row_exp[r][warp] = __float_as_int(amax);
    }
    __syncthreads();
    if (tid < n) {
      int m = 0;
      for (int w = 0; w < kMoeWarps; ++w) m = max(m, tb->row_exp[tid][w]);
      tb->row_exp[tid][0] = m;
    }
    __syncthreads();
  }
  for (int r = 0; r < n; ++r) {
    const T* src = act_row<T>(p, tb->slot[r0 + r]);
    float f = 1.f;
    bool fine = true;
    if constexpr (!std::is_same<T, __half>::value) {
      const float amax = __int_as_float(tb->row_exp[r][0]);
      f = pow2(row_shift(amax));
      fine = amax < __int_as_float(0x7f800000);
    }
    for (int q = tid; q < pieces; q += kMoeThreads) {
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (q * 8 < p.K) load8(src + q * 8, v);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a = v[2 * i] * f, b = v[2 * i + 1] * f;
        if (!fine) {  // an infinite row: its finite values stay finite
          if (fabsf(a) < __int_as_float(0x7f800000)) a = fminf(fmaxf(a, -65504.f), 65504.f);
          if (fabsf(b) < __int_as_float(0x7f800000)) b = fminf(fmaxf(b, -65504.f), 65504.f);
        }
        const __half2 h = __floats2half2_rn(a, b);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
      const int chunk = q >> 4, t = (q >> 2) & 3, jj = q & 3;
      xs[((chunk * 4 + jj) * kMoeRows + r) * 4 + t] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __syncthreads();
}

template <typename T>
__device__ __forceinline__ float row_unscale(const MoeTables* tb, int r) {
  if constexpr (std::is_same<T, __half>::value) return 1.f;
  return pow2(-row_shift(__int_as_float(tb->row_exp[r][0])));
}

// kUp: T is the activations' type and a tile is 8 gate and the 8 matching up rows; else T is float (h) and OutT the output's type.
template <typename T, typename OutT, bool kUp, int MT, int D>
__global__ void __launch_bounds__(kMoeThreads)
    fp4_experts_kernel(const MoeParams p) {
  extern __shared__ uint8_t smem_raw[];
  MoeTables* tb = reinterpret_cast<MoeTables*>(smem_raw);
  uint8_t* rest = smem_raw + (sizeof(MoeTables) + 15) / 16 * 16;
  constexpr uint32_t kStage = MT * 1280;  // a warp's chunk: per tile 2 x 512 bytes of codes, 2 x 128 of scales
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = ptx::smem_u32(rest) + warp * (D * kStage);
  float* red = reinterpret_cast<float*>(rest + kMoeWarps * D * kStage);  // [warp][MT][4][32]
  uint4* xs = reinterpret_cast<uint4*>(red + kMoeWarps * MT * 128);

  ptx::grid_dependency_wait();
  if (kUp && blockIdx.x == 0)
    for (int i = tid; i < p.done_count; i += kMoeThreads) p.done[i] = 0;
  route(p, tb);
  const int warps_m = kMoeWarps / p.warps_k, wk = warp % p.warps_k, wm = warp / p.warps_k;
  const int c0 = wk * p.chunks / p.warps_k, c1 = (wk + 1) * p.chunks / p.warps_k;
  const int tiles = (int)(p.rows / 16);  // of an expert (16 rows of w each)
  const int64_t code_row = p.K / 2, scale_row = p.K / 16;
  const int items = tb->num_live * p.sets;
  int staged_live = -1, staged_r0 = -1;

  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int live = item / p.sets, set = item - live * p.sets;
    const int expert = tb->live[live], first = tb->begin[live], rows_n = tb->begin[live + 1] - first;
    const int tile0 = (set * warps_m + wm) * MT;
    // this lane's two rows of each tile
    const uint8_t *wp[MT][2], *sp[MT][2];
    bool tile_live[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      tile_live[m] = tile0 + m < tiles;
      const int tile = tile_live[m] ? tile0 + m : 0;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int64_t row = (int64_t)expert * p.rows + (kUp ? (int64_t)tile * 8 + g + u * (p.rows / 2) : (int64_t)tile * 16 + g + u * 8);
        wp[m][u] = p.w + row * code_row + t * 16;
        sp[m][u] = p.ws + row * scale_row + t * 2;
      }
    }
    for (int r0 = 0; r0 < rows_n; r0 += kMoeRows) {
      const int n = min(kMoeRows, rows_n - r0);
      const auto issue = [&](int c, int d) {
        const bool in = c * kChunk + t * 32 < p.K;
        const uint32_t at = ring + d * kStage + lane * 16, sat = ring + d * kStage + MT * 1024 + lane * 4;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const bool ok = in && tile_live[m];
            cp_async_16(at + (m * 2 + u) * 512, ok ? wp[m][u] + c * 64 : p.w, ok);
            cp_async_4(sat + (m * 2 + u) * 128, ok ? reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(sp[m][u] + c * 8) & ~uintptr_t(3)) : p.ws, ok);
          }
      };
#pragma unroll
      for (int d = 0; d < D; ++d) {
        if (c0 + d < c1) issue(c0 + d, d);
        cp_async_commit();
      }
      if (staged_live != live || staged_r0 != r0) {
        stage_rows<T>(p, tb, first + r0, n, xs);
        staged_live = live, staged_r0 = r0;
      }
      float acc[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
      int d = 0;
      for (int c = c0; c < c1; ++c) {
        cp_async_wait<D - 1>();
        uint4 code[MT][2];
        uint32_t sc[MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            code[m][u] = ptx::lds_128(ring + d * kStage + lane * 16 + (m * 2 + u) * 512);
            const uint32_t word = lds_32(ring + d * kStage + MT * 1024 + lane * 4 + (m * 2 + u) * 128);
            sc[m][u] = cvt_f16x2_e4m3x2(word >> ((reinterpret_cast<uintptr_t>(sp[m][u]) & 2) * 8) & 0xffffu);
          }
        if (c + D < c1) issue(c + D, d);
        cp_async_commit();
        d = d + 1 == D ? 0 : d + 1;
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          const uint4 b = g < n ? xs[((c * 4 + jj) * kMoeRows + g) * 4 + t] : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            uint32_t a[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t word = jj == 0 ? code[m][u].x : jj == 1 ? code[m][u].y : jj == 2 ? code[m][u].z : code[m][u].w;
              const uint32_t s = __byte_perm(sc[m][u], 0, jj < 2 ? 0x1010 : 0x3232);
              cvt_f16x2_e2m1x8(word, a[u]);
#pragma unroll
              for (int i = 0; i < 4; ++i) a[u][i] = hmul2(a[u][i], s);
            }
            mma_f16(acc[m], a[0][0], a[1][0], a[0][1], a[1][1], b.x, b.y);
            mma_f16(acc[m], a[0][2], a[1][2], a[0][3], a[1][3], b.z, b.w);
          }
        }
      }
      // sums over the warps of a K split: lane (g, t) has rows g (0, 1) and g + 8 (2, 3), columns 2 t, 2 t + 1
      __syncthreads();  // (the sums before these have been read)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) red[((warp * MT + m) * 4 + j) * 32 + lane] = acc[m][j];
      __syncthreads();
      const float alpha = p.alpha ? p.alpha[expert] : 1.f;
      // thread -> (tile of the item, pair of values): j = 0, 1 with 2, 3
      for (int i = tid; i < warps_m * MT * 64; i += kMoeThreads) {
        const int l = i & 31, j = (i >> 5) & 1, m = (i >> 6) % MT, w = (i >> 6) / MT;
        const int tile = (set * warps_m + w) * MT + m, r = 2 * (l & 3) + j;
        if (tile >= tiles || r >= n) continue;
        float lo = 0.f, hi = 0.f;
        for (int k = 0; k < p.warps_k; ++k) {
          const float* at = red + (((w * p.warps_k + k) * MT + m) * 4 + j) * 32 + l;
          lo += at[0], hi += at[64];
        }
        const float f = row_unscale<T>(tb, r);
        lo = lo * alpha * f, hi = hi * alpha * f;
        const int slot = tb->slot[first + r0 + r];
        if constexpr (kUp) {
          p.h[(int64_t)slot * (p.rows / 2) + tile * 8 + (l >> 2)] = lo / (1.f + expf(-lo)) * hi;
        } else {
          const float w8 = p.weights[slot];
          float* at = p.h + (int64_t)slot * p.rows + tile * 16 + (l >> 2);
          at[0] = w8 * lo, at[8] = w8 * hi;
        }
      }
    }
    if constexpr (!kUp) {
      // the last of the experts' CTAs to reach a set of columns adds up its tokens
      __threadfence();
      __syncthreads();
      if (tid == 0) tb->last = atomicAdd(&p.done[set], 1) == tb->num_live - 1;
      __syncthreads();
      if (tb->last) {
        __threadfence();
        const int col0 = set * warps_m * MT * 16, cols = min(warps_m * MT * 16, (int)p.rows - col0);
        for (int i = tid; i < p.tokens * cols; i += kMoeThreads) {
          const int token = i / cols, col = col0 + i % cols;
          float sum = 0.f;
          for (int j = 0; j < p.topk; ++j) {
            const int s = token * p.topk + j;
            if ((uint32_t)p.ids[s] < (uint32_t)p.experts) sum += __ldcg(p.h + (int64_t)s * p.rows + col);
          }
          static_cast<OutT*>(p.out)[(int64_t)token * p.rows + col] = ElemTraits<OutT>::from_f32(sum * p.factor);
        }
      }
    }
  }
  if constexpr (!kUp) {
    if (tb->num_live == 0)  // no expert is named: zeros
      for (int64_t i = blockIdx.x * kMoeThreads + tid; i < (int64_t)p.tokens * p.rows; i += (int64_t)gridDim.x * kMoeThreads)
        static_cast<OutT*>(p.out)[i] = ElemTraits<OutT>::from_f32(0.f);
  }
}

template <typename T, typename OutT, bool kUp, int MT, int D>
static int launch_experts(MoeParams& p, cudaStream_t st) {
  auto kern = fp4_experts_kernel<T, OutT, kUp, MT, D>;
  const size_t smem = (sizeof(MoeTables) + 15) / 16 * 16 + (size_t)kMoeWarps * D * MT * 1280 + kMoeWarps * MT * 512 +
                      (size_t)p.chunks * 4 * kMoeRows * 4 * 16;
  SGLB_REQUIRE(smem <= 227 * 1024, "fused_experts_fp4: %lld columns are too many", (long long)p.K);
  static thread_local size_t attr_set[64] = {0};
  int dev = 0;
  SGLB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || attr_set[dev] < smem) {
    SGLB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (dev >= 0 && dev < 64) attr_set[dev] = smem;
  }
  const int per_sm = std::max(1, std::min(4, (int)(224 * 1024 / (smem + 1024))));
  const int64_t most = (int64_t)std::min(p.slots, p.experts) * p.sets;
  const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, (int64_t)sm_count() * per_sm));
  SGLB_CUDA(launch_pdl(kern, grid, kMoeThreads, smem, st, p));
  return SGLB200_OK;
}

struct MoeShape {
  int64_t T, topk, H, I;
  int E;
};
constexpr int kMoeMT = 2, kMoeD = 3;
static int warps_k_for(int chunks) { return chunks >= 16 ? 8 : chunks >= 8 ? 4 : chunks >= 4 ? 2 : 1; }
static int64_t down_sets(int64_t H, int64_t I) {
  const int wm = kMoeWarps / warps_k_for((int)((I + kChunk - 1) / kChunk));
  return (H / 16 + wm * kMoeMT - 1) / (wm * kMoeMT);
}

}  // namespace fp4
}  // namespace sglb200

using namespace sglb200;

extern "C" {

int64_t sglb200_fused_experts_fp4_workspace_bytes(int64_t tokens, int64_t topk, int64_t hidden, int64_t intermediate) {
  if (tokens <= 0 || topk <= 0 || hidden <= 0 || intermediate <= 0) return 0;
  const int64_t slots = tokens * topk;
  return (slots * intermediate + slots * hidden) * 4 + (fp4::down_sets(hidden, intermediate) * 4 + 15) / 16 * 16;
}

int sglb200_fused_experts_fp4(const void* x, int dtype, const void* w13, const void* w13_scale, const float* w13_alpha, const void* w2,
                              const void* w2_scale, const float* w2_alpha, const float* topk_weights, const int32_t* topk_ids, void* out,
                              int64_t tokens, int64_t topk, int num_experts, int64_t hidden, int64_t intermediate, float factor,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype != 0 && dtype != 1) return fail(SGLB200_E_UNSUPPORTED, "fused_experts_fp4: activations must be bfloat16 or float16");
  SGLB_REQUIRE(tokens >= 0 && topk > 0 && hidden > 0 && intermediate > 0, "fused_experts_fp4: %lld tokens, topk %lld, hidden %lld, intermediate %lld",
               (long long)tokens, (long long)topk, (long long)hidden, (long long)intermediate);
  SGLB_REQUIRE(num_experts > 0 && num_experts <= fp4::kMoeMaxExperts, "fused_experts_fp4: %d experts (at most %d)", num_experts, fp4::kMoeMaxExperts);
  SGLB_REQUIRE(hidden % 32 == 0 && intermediate % 32 == 0, "fused_experts_fp4: hidden (%lld) and intermediate (%lld) must be divisible by 32",
               (long long)hidden, (long long)intermediate);
  SGLB_REQUIRE(tokens <= fp4::kMoeMaxSlots && topk <= fp4::kMoeMaxSlots && tokens * topk <= fp4::kMoeMaxSlots,
               "fused_experts_fp4: %lld tokens with %lld experts each: it is for at most %d of both together", (long long)tokens,
               (long long)topk, fp4::kMoeMaxSlots);
  if (tokens == 0) return SGLB200_OK;
  SGLB_REQUIRE(x && w13 && w13_scale && w2 && w2_scale && topk_weights && topk_ids && out, "fused_experts_fp4: null pointer");
  SGLB_REQUIRE(aligned16(x) && aligned16(w13) && aligned16(w13_scale) && aligned16(w2) && aligned16(w2_scale) && aligned16(out),
               "fused_experts_fp4: pointers must be 16-byte aligned");
  const int64_t need = sglb200_fused_experts_fp4_workspace_bytes(tokens, topk, hidden, intermediate);
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need)
    return fail(SGLB200_E_WORKSPACE, "fused_experts_fp4: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t slots = tokens * topk;
  float* h = static_cast<float*>(workspace);
  float* y = h + slots * intermediate;
  fp4::MoeParams p{};
  p.ids = topk_ids, p.weights = topk_weights;
  p.slots = (int)slots, p.topk = (int)topk, p.experts = num_experts, p.tokens = (int)tokens;
  p.done = reinterpret_cast<int32_t*>(y + slots * hidden), p.done_count = (int)fp4::down_sets(hidden, intermediate);
  p.factor = factor;
  const auto plan = [&](int64_t K, int64_t rows) {
    p.K = K, p.rows = rows, p.chunks = (int)((K + fp4::kChunk - 1) / fp4::kChunk), p.warps_k = fp4::warps_k_for(p.chunks);
    const int per = fp4::kMoeWarps / p.warps_k * fp4::kMoeMT;
    p.sets = (int)((rows / 16 + per - 1) / per);
  };
  p.x = x, p.w = static_cast<const uint8_t*>(w13), p.ws = static_cast<const uint8_t*>(w13_scale), p.alpha = w13_alpha, p.h = h;
  plan(hidden, 2 * intermediate);
  int rc = dtype == 0 ? fp4::launch_experts<__nv_bfloat16, __nv_bfloat16, true, fp4::kMoeMT, fp4::kMoeD>(p, st)
                      : fp4::launch_experts<__half, __half, true, fp4::kMoeMT, fp4::kMoeD>(p, st);
  if (rc) return rc;
  p.x = h, p.w = static_cast<const uint8_t*>(w2), p.ws = static_cast<const uint8_t*>(w2_scale), p.alpha = w2_alpha, p.h = y, p.out = out;
  plan(intermediate, hidden);
  return dtype == 0 ? fp4::launch_experts<float, __nv_bfloat16, false, fp4::kMoeMT, fp4::kMoeD>(p, st)
                    : fp4::launch_experts<float, __half, false, fp4::kMoeMT, fp4::kMoeD>(p, st);
}

}  // extern "C"
