// dx_int8.cuh — linear layers on 8-bit integer operands:
//   Y[m,n] = act(s_m t_n sum_k Xq[m,k] Wq[n,k] + bias[n]) (+ R[m,n])
//   Y[m,n] = act(s_m tg_n sum_k Xq Wgq + bg[n]) * (s_m tu_n sum_k Xq Wuq + bu[n])
// with Xq, Wq signed 8-bit, s (one per row of X: token) and t (one per output
// channel) fp32, fp16 / bf16 / fp32 out.  The sums are exact: 32-bit integer
// accumulators of tcgen05.mma kind::i8 (K <= 131071, so |sum| < 2^31 even where
// every product is 128 * 128); they become fp32 once, at the end.
//
// Both operands are K-major: rows of 128 bytes of K in 128-byte-swizzled
// shared memory, one MMA per 32 bytes.  Two kernels:
//
//   int8_pair_kernel  CTA pairs, 256 x bn tiles, persistent: the integer form
//     of umma2_fused_linear_kernel (same roles, barriers and raster).  Serves
//     more than 128 tokens (gated: 64).
//   int8_tile_kernel  one 128 (channels) x mn (tokens) tile per CTA with the
//     operands swapped — D^T[n, m] — so that a few tokens cost a narrow MMA
//     while W streams past once; K split over a cluster of C CTAs that add
//     their integer partial sums through distributed shared memory.  Integer
//     sums do not depend on their order.  Serves up to 128 tokens (gated: 64).
//
// Every mbarrier wait is bounded, as in dx_umma_gemm.cuh.
#pragma once

#include "dx_epilogue.cuh"
#include "dx_ptx.cuh"
#include "dx_umma_gemm.cuh"

namespace dx {

struct Int8Params {
  int M, N;
  int k_blocks;  // 128-byte blocks of K
  long long ldy, ldr;
  const float* sx;   // [M]
  const float* sw;   // [N]
  const float* sw2;  // gated: the up-projection's [N]
  const void* bias;
  const void* bias2;
  const void* residual;
  void* Y;
  int act;
  // tile kernel
  int nr;       // channels of a tile: up to 128 (gated: 64), a multiple of 8
  int mn;       // tokens of a tile: a multiple of 16 up to 128
  int cluster;  // CTAs that split K
  int w_early;  // the preceding launch wrote only X: W may be read before it ends
  int stages;   // of the operand ring (both kernels)
  // pair kernel
  int bn;       // accumulator columns of a tile: a multiple of 32 (gated: 64) up to 256
  int m_tiles, n_tiles, group_m, workers;
  int full_tiles;  // tiles [full_tiles, m_tiles * n_tiles) are done as two halves each
  int num_work;    // full_tiles + 2 * the others
  int has_residual;
  int tma_out;     // Y (and R) can be stored (and read) by TMA
};

__device__ __forceinline__ float ld_elem(const void* p, long long i, const __half*) {
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ float ld_elem(const void* p, long long i, const __nv_bfloat16*) {
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ float ld_elem(const void* p, long long i, const float*) {
  return static_cast<const float*>(p)[i];
}

// =====================================================================
// Tile kernel: 128 rows of W x mn tokens, operands swapped.
// =====================================================================
struct Int8TileShape {
  static constexpr int MAX_MN = 128;
  static constexpr int BK = 128;            // bytes of K a stage
  static constexpr int W_BYTES = 128 * BK;  // gated: 64 rows of Wg, 64 of Wu
  static constexpr int MAX_STAGES = 12;
  static constexpr int MAX_CLUSTER = 8;
  static constexpr int THREADS = 192;
  // Shared memory: the ring of `stages` W tiles, then as many X tiles, then
  static constexpr int OFF_DEST = MAX_MN * 4;  // (behind MAX_MN row scales)
  static constexpr int OFF_BAR = OFF_DEST + MAX_MN * 4;
  static constexpr int BAR_FULL = 0;
  static constexpr int BAR_EMPTY = MAX_STAGES;
  static constexpr int BAR_TFULL = 2 * MAX_STAGES;
  static constexpr int NUM_BARS = BAR_TFULL + 1;
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr int TAIL_BYTES = OFF_MISC + 16;
  static constexpr int stage_bytes(int mn) { return W_BYTES + mn * BK; }
  static constexpr int smem_bytes(int mn, int stages) {
    return 1024 + stages * stage_bytes(mn) + TAIL_BYTES;
  }
  static constexpr int HALF_SM = 115712;  // what each of two CTAs of an SM may have
  static constexpr int FULL_SM = 227 * 1024;
  // The partial sums received from a cluster of C CTAs, [source][row of this
  // CTA's share][128], lie in the idle ring: at most mn + C rows of 512 bytes.
  static constexpr int MIN_STAGES = 3;
  static constexpr int half_sm_stages(int mn) { return (HALF_SM - smem_bytes(mn, 0)) / stage_bytes(mn); }
};
static_assert(Int8TileShape::half_sm_stages(Int8TileShape::MAX_MN) >= Int8TileShape::MIN_STAGES &&
                  (16 + Int8TileShape::MAX_CLUSTER) * 512 <=
                      Int8TileShape::MIN_STAGES * Int8TileShape::stage_bytes(16) &&
                  (Int8TileShape::MAX_MN + Int8TileShape::MAX_CLUSTER) * 512 <=
                      Int8TileShape::MIN_STAGES * Int8TileShape::stage_bytes(Int8TileShape::MAX_MN),
              "receive area");

// First row (of `rows`) of the share that CTA c of C finishes.
__device__ __forceinline__ int int8_share(int c, int rows, int C) { return c * rows / C; }

template <typename T, bool kGated>
__global__ void __launch_bounds__(Int8TileShape::THREADS, 2)
    int8_tile_kernel(const __grid_constant__ CUtensorMap tmW,
                     const __grid_constant__ CUtensorMap tmW2,
                     const __grid_constant__ CUtensorMap tmX, const Int8Params p) {
  using S = Int8TileShape;
  using Tr = ElemTraits<T>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t base = (raw_u32 + 1023u) & ~1023u;
  uint8_t* const base_ptr = smem_raw + (base - raw_u32);
  const int stages = p.stages;
  const uint32_t x_bytes = static_cast<uint32_t>(p.mn) * S::BK;
  const uint32_t stage_bytes = S::W_BYTES + x_bytes;
  // What a stage loads: with fewer than 128 rows the MMA reads stale rows behind
  // them, whose results nobody uses.
  const uint32_t load_bytes = static_cast<uint32_t>(p.nr * (kGated ? 2 : 1)) * S::BK + x_bytes;
  const uint32_t sW = base;
  const uint32_t sX = base + static_cast<uint32_t>(stages) * S::W_BYTES;
  const uint32_t tail = static_cast<uint32_t>(stages) * stage_bytes;
  const uint32_t bars = base + tail + S::OFF_BAR;
  float* const s_sx = reinterpret_cast<float*>(base_ptr + tail);
  uint32_t* const s_dest = reinterpret_cast<uint32_t*>(base_ptr + tail + S::OFF_DEST);
  uint32_t* const tmem_word = reinterpret_cast<uint32_t*>(base_ptr + tail + S::OFF_MISC);
  volatile int* const abort_flag =
      reinterpret_cast<volatile int*>(base_ptr + tail + S::OFF_MISC + 4);
  const uint32_t tmem_cols = p.mn <= 32 ? 32u : (p.mn <= 64 ? 64u : 128u);
  auto bar = [bars](int i) { return bars + 8u * static_cast<uint32_t>(i); };

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int C = p.cluster;
  const int c = C > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int n0 = static_cast<int>(blockIdx.x) / C * p.nr;
  const int m0 = static_cast<int>(blockIdx.y) * p.mn;
  const int rows = min(p.mn, p.M - m0);
  const int kb0 = static_cast<int>(static_cast<long long>(c) * p.k_blocks / C);
  const int kb1 = static_cast<int>(static_cast<long long>(c + 1) * p.k_blocks / C);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(bar(S::BAR_FULL + s), 1);
      mbar_init(bar(S::BAR_EMPTY + s), 1);
    }
    mbar_init(bar(S::BAR_TFULL), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmW);
    if (kGated) tma_prefetch_desc(&tmW2);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_word), tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_word;

  auto load_w = [&](int s, int kb, uint32_t fb, uint64_t pol) {
    if constexpr (kGated) {
      tma_load_2d_hint(&tmW, sW + s * S::W_BYTES, fb, kb * S::BK, n0, pol);
      tma_load_2d_hint(&tmW2, sW + s * S::W_BYTES + S::W_BYTES / 2, fb, kb * S::BK, n0, pol);
    } else {
      tma_load_2d_hint(&tmW, sW + s * S::W_BYTES, fb, kb * S::BK, n0, pol);
    }
  };
  const bool producer = warp == 0 && lane == 0;
  // With one tile of tokens W is read once and leaves L2 first.
  const uint64_t pol_w =
      gridDim.y == 1 ? make_l2_policy_evict_first() : make_l2_policy_evict_normal();
  const int early = min(stages, kb1 - kb0);
  if (producer && p.w_early) {
    for (int i = 0; i < early; ++i) {
      mbar_arrive_expect_tx(bar(S::BAR_FULL + i), load_bytes);
      load_w(i, kb0 + i, bar(S::BAR_FULL + i), pol_w);
    }
  }
  __syncwarp();
  // Everything else in global memory may be the preceding launch's output.
  grid_dependency_wait();
  grid_launch_dependents();

  const int q = warp & 3;            // TMEM lane quarter of an epilogue warp
  const int et = threadIdx.x - 64;   // epilogue thread
  const uint32_t lane_addr = tmem + (static_cast<uint32_t>(q * 32) << 16);
  bool done = true;  // epilogue: the accumulator is complete
  // The channel this epilogue thread finishes, and its scales and biases.
  const bool via_smem = kGated || C > 1;
  const int nt = kGated ? (et & 63) : (via_smem ? et : q * 32 + lane);
  const int ncol = nt < p.nr ? n0 + nt : p.N;  // (p.N: none)
  float t0 = 0.0f, t1 = 0.0f, b0 = 0.0f, b1 = 0.0f;
  // The rows this CTA finishes, this thread's first one and its residual.
  const int my_row0 = int8_share(c, rows, C), my_rows = int8_share(c + 1, rows, C) - my_row0;
  const int my_first = kGated ? (et >> 6) & 1 : 0;
  float res0 = 0.0f;

  if (warp == 0) {
    // ------------------------------------------------------ TMA producer
    if (lane == 0) {
      uint32_t ph = 0;
      int s = 0, i = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++i) {
        const uint32_t fb = bar(S::BAR_FULL + s);
        if (!(p.w_early && i < early)) {
          if (!mbar_wait(bar(S::BAR_EMPTY + s), ph ^ 1u, abort_flag)) break;
          mbar_arrive_expect_tx(fb, load_bytes);
          load_w(s, kb, fb, pol_w);
        }
        tma_load_2d(&tmX, sX + s * x_bytes, fb, kb * S::BK, m0);
        if (++s == stages) {
          s = 0;
          ph ^= 1u;
        }
      }
      // Loads in flight land before the shared memory is used or released.
      const int n_drain = min(i, stages);
      for (int j = i - n_drain; j < i; ++j)
        mbar_wait_drain(bar(S::BAR_FULL + j % stages), (j / stages) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------- MMA issuer
    // The whole warp runs the loop and one lane issues: with every operand the
    // same in all lanes the descriptors stay in uniform registers.  A loop of
    // lane 0 alone took 165 ns a stage plus 29 ns an MMA to issue.
    const uint32_t idesc = umma_idesc_i8(128, p.mn);
    const bool issuer = elect_one();
    uint32_t ph = 0;
    int s = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(bar(S::BAR_FULL + s), ph, abort_flag)) break;
      const uint64_t ad = smem_desc_sw128(sW + s * S::W_BYTES, 16, 1024);
      const uint64_t bd = smem_desc_sw128(sX + s * x_bytes, 16, 1024);
      if (issuer) {
#pragma unroll
        for (int k = 0; k < S::BK / 32; ++k)
          umma_i8(tmem, ad + 2ull * k, bd + 2ull * k, idesc, (kb != kb0 || k != 0) ? 1u : 0u);
        umma_commit(bar(S::BAR_EMPTY + s));
      }
      __syncwarp();
      if (++s == stages) {
        s = 0;
        ph ^= 1u;
      }
    }
    if (issuer) umma_commit(bar(S::BAR_TFULL));  // also after a wait that gave up
    mbar_wait_drain(bar(S::BAR_TFULL), 0);
    __syncwarp();
  } else {
    // --------------------------------------------------------- epilogue
    if (et < rows) {
      s_sx[et] = p.sx[m0 + et];
      if (via_smem) {
        // Where this CTA's partial sums of row et go: the CTA whose share has the row.
        // (Found row by row behind the wait, 16 rows of 4096 x 4096 took 10.3 us, now 8.8.)
        const int dest = ((et + 1) * C - 1) / rows;
        const int first = int8_share(dest, rows, C);
        const int share = int8_share(dest + 1, rows, C) - first;
        const uint32_t at = base + static_cast<uint32_t>((c * share + et - first) * 512);
        s_dest[et] = mapa_shared(at, static_cast<uint32_t>(dest));
      }
    }
    if (ncol < p.N) {
      t0 = p.sw[ncol];
      if (p.bias != nullptr) b0 = ld_elem(p.bias, ncol, static_cast<const T*>(nullptr));
      if (kGated) {
        t1 = p.sw2[ncol];
        if (p.bias2 != nullptr) b1 = ld_elem(p.bias2, ncol, static_cast<const T*>(nullptr));
      }
    }
    if (via_smem && p.residual != nullptr && ncol < p.N && my_first < my_rows)
      res0 = ld_elem(p.residual, (m0 + my_row0 + my_first) * p.ldr + ncol,
                     static_cast<const T*>(nullptr));
    done = mbar_wait(bar(S::BAR_TFULL), 0, abort_flag) && *abort_flag == 0;
    done = __all_sync(0xffffffffu, done) != 0;  // (TMEM is read by whole warps)
    tc_fence_after();
    named_bar_sync(1, 128);  // s_sx
  }

  T* const Y = static_cast<T*>(p.Y);
  if (via_smem) {
    // Partial sums to the CTA that finishes the row, once every ring is idle.
    if (C > 1)
      cluster_sync();
    else
      __syncthreads();
    if (warp >= 2 && done) {
      const uint32_t mine = static_cast<uint32_t>((q * 32 + lane) * 4);
#pragma unroll 1
      for (int mc = 0; mc < rows; mc += 16) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(lane_addr + static_cast<uint32_t>(mc), r);
        uint32_t to[16];  // (behind the last row: not used)
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          *reinterpret_cast<uint4*>(to + j) = *reinterpret_cast<const uint4*>(s_dest + mc + j);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (mc + j < rows) st_shared_cluster_u32(to[j] + mine, r[j]);
      }
    }
    tc_fence_before();
    if (C > 1)
      cluster_sync();
    else
      __syncthreads();
    if (warp >= 2 && done && ncol < p.N) {
      const int* const recv = reinterpret_cast<const int*>(base_ptr);
      constexpr int kStep = kGated ? 2 : 1;
      float res = res0;
#pragma unroll 1
      for (int i = my_first; i < my_rows; i += kStep) {
        const long long m = m0 + my_row0 + i;
        float next = 0.0f;
        if (p.residual != nullptr && i + kStep < my_rows)
          next = ld_elem(p.residual, (m + kStep) * p.ldr + ncol, static_cast<const T*>(nullptr));
        int a0 = 0, a1 = 0;
#pragma unroll
        for (int s = 0; s < S::MAX_CLUSTER; ++s) {
          if (s < C) {
            const int* const src = recv + (s * my_rows + i) * 128 + (kGated ? (et & 63) : et);
            a0 += src[0];
            if (kGated) a1 += src[64];
          }
        }
        const float sx = s_sx[my_row0 + i];
        float v[1] = {fmaf(static_cast<float>(a0), sx * t0, b0)};
        act_values<sizeof(T) == 4>(v, p.act);
        if (kGated) v[0] *= fmaf(static_cast<float>(a1), sx * t1, b1);
        Y[m * p.ldy + ncol] = Tr::from_float(v[0] + res);
        res = next;
      }
    }
  } else if (warp >= 2 && done) {
#pragma unroll 1
    for (int mc = 0; mc < rows; mc += 16) {
      uint32_t r[16];
      tmem_ld_32x32b_x16(lane_addr + static_cast<uint32_t>(mc), r);
      float res[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        res[j] = (p.residual != nullptr && ncol < p.N && mc + j < rows)
                     ? ld_elem(p.residual, (m0 + mc + j) * p.ldr + ncol, static_cast<const T*>(nullptr))
                     : 0.0f;
      tmem_wait_ld();
      float v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float sx = mc + j < rows ? s_sx[mc + j] : 0.0f;
        v[j] = fmaf(static_cast<float>(static_cast<int>(r[j])), sx * t0, b0);
      }
      act_values<sizeof(T) == 4>(v, p.act);
      if (ncol < p.N) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (mc + j < rows) Y[(m0 + mc + j) * p.ldy + ncol] = Tr::from_float(v[j] + res[j]);
      }
    }
    tc_fence_before();
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// =====================================================================
// CTA-pair kernel: 256 x bn tiles, bn chosen for each problem.
// =====================================================================
struct Int8PairShape {
  static constexpr int BM = 128;  // rows per CTA
  static constexpr int BK = 128;
  static constexpr int MAX_BN = 256;
  static constexpr int A_BYTES = BM * BK;
  // The ring holds as many stages of A_BYTES + bn / 2 * BK as fit (5 at bn = 256).
  static constexpr int RING_BYTES = 5 * (A_BYTES + MAX_BN / 2 * BK);
  static constexpr int MAX_STAGES = 8;
  static constexpr int TMEM_COLS = 2 * MAX_BN;  // two accumulators
  static constexpr int THREADS = 64 + 32 * kEpiWarps;
  static constexpr int VEC_BYTES = 4 * 128 * 4;  // a warp's column scales and biases
  static constexpr int OFF_EPI = RING_BYTES;
  static constexpr int EPI_BUFS = 3;  // staging buffers of an epilogue warp
  static constexpr int OFF_VEC = OFF_EPI + kEpiWarps * EPI_BUFS * kEpiBufBytes;
  static constexpr int OFF_BAR = OFF_VEC + kEpiWarps * VEC_BYTES;
  static constexpr int BAR_FULL = 0;
  static constexpr int BAR_EMPTY = MAX_STAGES;
  static constexpr int BAR_TFULL = 2 * MAX_STAGES;
  static constexpr int BAR_TEMPTY = BAR_TFULL + 2;
  static constexpr int BAR_RES = BAR_TEMPTY + 2;
  static constexpr int BAR_DRAIN = BAR_RES + EPI_BUFS * kEpiWarps;
  static constexpr int NUM_BARS = BAR_DRAIN + 1;
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr int SMEM_BYTES = 1024 + OFF_MISC + 16;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
  static_assert(32 * 33 * 4 <= EPI_BUFS * kEpiBufBytes, "a chunk as fp32 rows");
};

// A pair's piece of work: a tile, or half the columns of one.
struct Int8Work {
  int mb, nb, half, bn;  // bn: accumulator columns (the tile's, or half of them)
};

__device__ __forceinline__ void int8_tile_coords(const Int8Params& p, int t, int& mb, int& nb);

__device__ __forceinline__ Int8Work int8_work(const Int8Params& p, int i) {
  Int8Work w;
  w.half = 0;
  w.bn = p.bn;
  int t = i;
  if (i >= p.full_tiles) {
    t = p.full_tiles + ((i - p.full_tiles) >> 1);
    w.half = (i - p.full_tiles) & 1;
    w.bn = p.bn / 2;
  }
  int8_tile_coords(p, t, w.mb, w.nb);
  return w;
}

// The t'th tile: m-tiles fastest inside groups of group_m (as umma_tile_coords).
__device__ __forceinline__ void int8_tile_coords(const Int8Params& p, int t, int& mb, int& nb) {
  const int per_group = p.group_m * p.n_tiles;
  const int g = t / per_group;
  const int r = t - g * per_group;
  const int m_first = g * p.group_m;
  const int gm = min(p.group_m, p.m_tiles - m_first);
  mb = m_first + r % gm;
  nb = r / gm;
}

// Scales and biases of a warp's columns, spread over its lanes: a register holds
// column lane + 32 k.  Asked for one tile ahead (short K loops do not hide the
// trip to memory), then put into the warp's shared arrays.
template <bool kGated>
struct Int8Columns {
  static constexpr int kPer = kGated ? 2 : 4;  // at most 64 / 128 columns
  float t[kPer], b[kPer], t2[kGated ? kPer : 1], b2[kGated ? kPer : 1];
  float sx;  // of the lane's row
};

template <typename T, bool kGated>
__device__ __forceinline__ void int8_fetch_columns(const Int8Params& p, int n, int cols, int row,
                                                   int lane, Int8Columns<kGated>& c) {
  const T* const bias = static_cast<const T*>(p.bias);
  const T* const bias2 = static_cast<const T*>(p.bias2);
  c.sx = row < p.M ? p.sx[row] : 0.0f;
#pragma unroll
  for (int k = 0; k < Int8Columns<kGated>::kPer; ++k) {
    const int j = n + lane + 32 * k;
    const bool in = 32 * k < cols && j < p.N;
    c.t[k] = in ? p.sw[j] : 0.0f;
    c.b[k] = in && bias != nullptr ? ElemTraits<T>::to_float(bias[j]) : 0.0f;
    if (kGated) {
      c.t2[k] = in ? p.sw2[j] : 0.0f;
      c.b2[k] = in && bias2 != nullptr ? ElemTraits<T>::to_float(bias2[j]) : 0.0f;
    }
  }
}

template <bool kGated>
__device__ __forceinline__ void int8_put_columns(const Int8Columns<kGated>& c, float* vec, int lane) {
  __syncwarp();  // the previous tile's values are no longer read
#pragma unroll
  for (int k = 0; k < Int8Columns<kGated>::kPer; ++k) {
    vec[lane + 32 * k] = c.t[k];
    vec[128 + lane + 32 * k] = c.b[k];
    if (kGated) {
      vec[256 + lane + 32 * k] = c.t2[k];
      vec[384 + lane + 32 * k] = c.b2[k];
    }
  }
  __syncwarp();
}

// v = acc * (sx * t) + b over the 32 columns at t, b (shared memory, read as
// broadcasts of four).
__device__ __forceinline__ void int8_scale(float (&v)[32], const uint32_t (&r)[32], float sx,
                                           const float* t, const float* b) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float4 tt = *reinterpret_cast<const float4*>(t + 4 * j);
    const float4 bb = *reinterpret_cast<const float4*>(b + 4 * j);
    v[4 * j + 0] = fmaf(static_cast<float>(static_cast<int>(r[4 * j + 0])), sx * tt.x, bb.x);
    v[4 * j + 1] = fmaf(static_cast<float>(static_cast<int>(r[4 * j + 1])), sx * tt.y, bb.y);
    v[4 * j + 2] = fmaf(static_cast<float>(static_cast<int>(r[4 * j + 2])), sx * tt.z, bb.z);
    v[4 * j + 3] = fmaf(static_cast<float>(static_cast<int>(r[4 * j + 3])), sx * tt.w, bb.w);
  }
}

// 32 finished columns v of a warp's 32 rows (lane: row) into any Y: through shared
// memory (33 floats a row: no bank conflicts), so that a store covers 32 columns
// of one row.  For outputs that TMA cannot store: fp32, or rows that do not start on
// 16 bytes.
template <typename T>
__device__ __forceinline__ void int8_store_rows(const Int8Params& p, const float (&v)[32], float* s,
                                                int row0, int col, int lane) {
  using Tr = ElemTraits<T>;
#pragma unroll
  for (int j = 0; j < 32; ++j) s[lane * 33 + j] = v[j];
  __syncwarp();
  col += lane;
  const int rows = col < p.N ? min(32, p.M - row0) : 0;
  T* y = static_cast<T*>(p.Y) + row0 * p.ldy + col;
  const T* res = static_cast<const T*>(p.residual);
  if (rows == 32 && res == nullptr) {
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      *y = Tr::from_float(s[r * 33 + lane]);
      y += p.ldy;
    }
  } else {
    if (res != nullptr) res += row0 * p.ldr + col;
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += 8) {
      float x[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        x[r] = s[(r0 + r) * 33 + lane];
        if (res != nullptr && r0 + r < rows) x[r] += Tr::to_float(res[r * p.ldr]);
      }
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r0 + r < rows) y[r * p.ldy] = Tr::from_float(x[r]);
      y += 8 * p.ldy;
      if (res != nullptr) res += 8 * p.ldr;
    }
  }
  __syncwarp();
}

template <typename T, bool kGated>
__global__ void __launch_bounds__(Int8PairShape::THREADS, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap tmA,
                     const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmB2,
                     const __grid_constant__ CUtensorMap tmY,
                     const __grid_constant__ CUtensorMap tmR, const Int8Params p) {
  using S = Int8PairShape;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t base = (raw_u32 + 1023u) & ~1023u;
  uint8_t* const base_ptr = smem_raw + (base - raw_u32);
  const uint32_t b_bytes = static_cast<uint32_t>(p.bn / 2) * S::BK;  // a stage's W rows, per CTA
  const int box_rows = p.bn / 4;                                     // per load
  const uint32_t sA = base;
  const uint32_t sB = base + static_cast<uint32_t>(p.stages) * S::A_BYTES;
  const uint32_t bars = base + S::OFF_BAR;
  uint32_t* const tmem_word = reinterpret_cast<uint32_t*>(base_ptr + S::OFF_MISC);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(base_ptr + S::OFF_MISC + 4);
  auto bar = [bars](int i) { return bars + 8u * static_cast<uint32_t>(i); };

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = static_cast<int>(blockIdx.x >> 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(bar(S::BAR_FULL + s), 1);
      mbar_init(bar(S::BAR_EMPTY + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(S::BAR_TFULL + b), 1);
      mbar_init(bar(S::BAR_TEMPTY + b), 2 * kEpiWarps);
    }
    for (int i = 0; i < S::EPI_BUFS * kEpiWarps; ++i) mbar_init(bar(S::BAR_RES + i), 1);
    mbar_init(bar(S::BAR_DRAIN), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if (kGated) tma_prefetch_desc(&tmB2);
    if (p.tma_out) tma_prefetch_desc(&tmY);
    if (p.has_residual) tma_prefetch_desc(&tmR);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_word), S::TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_word;
  grid_dependency_wait();
  grid_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------------ TMA producer
    if (lane == 0) {
      const uint64_t pol = make_l2_policy_evict_normal();
      int s = 0;
      uint32_t ph = 0, issued = 0;
      bool ok = true;
      for (int i = pair; ok && i < p.num_work; i += p.workers) {
        const Int8Work wk = int8_work(p, i);
        const int m0 = wk.mb * 2 * S::BM + static_cast<int>(rank) * S::BM;
        // Plain: a tile's columns are the leader's, then the peer's; gated: both
        // CTAs load the same columns, the leader of Wg and the peer of Wu.
        const int n0 = kGated ? wk.nb * (p.bn / 2) + wk.half * box_rows
                              : wk.nb * p.bn + wk.half * wk.bn + static_cast<int>(rank) * (wk.bn / 2);
        const bool wide = wk.bn == p.bn;
        const uint32_t bytes = 2 * (S::A_BYTES + static_cast<uint32_t>(wk.bn / 2) * S::BK);
        const CUtensorMap* const mapB = (kGated && rank != 0) ? &tmB2 : &tmB;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(bar(S::BAR_EMPTY + s), ph ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(bar(S::BAR_FULL + s), bytes);
          const uint32_t fb = mapa_shared(bar(S::BAR_FULL + s), 0);
          tma_load_2d_pair(&tmA, sA + s * S::A_BYTES, fb, kb * S::BK, m0, pol);
          tma_load_2d_pair(mapB, sB + s * b_bytes, fb, kb * S::BK, n0, pol);
          if (wide)
            tma_load_2d_pair(mapB, sB + s * b_bytes + b_bytes / 2, fb, kb * S::BK, n0 + box_rows,
                             pol);
          ++issued;
          if (++s == p.stages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      if (leader) {
        const uint32_t stages = static_cast<uint32_t>(p.stages);
        const uint32_t n_drain = issued < stages ? issued : stages;
        for (uint32_t i = issued - n_drain; i < issued; ++i)
          mbar_wait_drain(bar(S::BAR_FULL + static_cast<int>(i % stages)), (i / stages) & 1u);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ----------------------------------------------- MMA issuer (leader)
    if (leader) {
      const bool issuer = elect_one();
      int s = 0, local = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int i = pair; ok && i < p.num_work; i += p.workers, ++local) {
        const uint32_t idesc = umma_idesc_i8(256, i < p.full_tiles ? p.bn : p.bn / 2);
        const int b = local & 1;
        const uint32_t use_ph = (static_cast<uint32_t>(local) >> 1) & 1u;
        if (!mbar_wait_warp(bar(S::BAR_TEMPTY + b), use_ph ^ 1u, abort_flag)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(b * S::MAX_BN);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait_warp(bar(S::BAR_FULL + s), ph, abort_flag)) {
            ok = false;
            break;
          }
          const uint64_t ad = smem_desc_sw128(sA + s * S::A_BYTES, 16, 1024);
          const uint64_t bd = smem_desc_sw128(sB + s * b_bytes, 16, 1024);
          if (issuer) {
#pragma unroll
            for (int k = 0; k < S::BK / 32; ++k)
              umma_i8_pair(d_tmem, ad + 2ull * k, bd + 2ull * k, idesc,
                           (kb != 0 || k != 0) ? 1u : 0u);
            umma_commit_both(bar(S::BAR_EMPTY + s));
          }
          __syncwarp();
          if (++s == p.stages) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (ok && issuer) umma_commit_both(bar(S::BAR_TFULL + b));
        __syncwarp();
      }
      if (issuer) umma_commit_pair(mapa_shared(bar(S::BAR_DRAIN), 0));
      mbar_wait_drain(bar(S::BAR_DRAIN), 0);
    }
    __syncwarp();
  } else {
    // --------------------------------------------- epilogue (both CTAs)
    const int e = warp - 2;
    const int q = warp & 3;
    EpilogueCtx<T> c;
    c.tmY = &tmY;
    c.tmR = &tmR;
    c.bias = nullptr;
    c.M = p.M;
    c.N = p.N;
    c.has_residual = p.has_residual;
    c.ebuf0 = base + S::OFF_EPI + e * S::EPI_BUFS * kEpiBufBytes;
    c.ebuf_ptr0 = base_ptr + S::OFF_EPI + e * S::EPI_BUFS * kEpiBufBytes;
    c.rbar0 = bar(S::BAR_RES + e * S::EPI_BUFS);
    c.pol_stream = make_l2_policy_evict_first();
    float* const vec = reinterpret_cast<float*>(base_ptr + S::OFF_VEC + e * S::VEC_BYTES);
    uint32_t it = 0;
    int local = 0;
    // Where this warp works on the i'th piece: its first column and 32-column chunks
    // (half of the piece's), and the first of its 32 rows.
    auto place = [&](int i, Int8Work& wk, int& n0, int& c0, int& chunks, int& row_base) {
      wk = int8_work(p, i);
      const int out_cols = kGated ? wk.bn / 2 : wk.bn;
      const int half = (out_cols / 32 + 1) / 2;
      c0 = (e / 4) * half * 32;
      chunks = e / 4 == 0 ? half : out_cols / 32 - half;
      n0 = wk.nb * (kGated ? p.bn / 2 : p.bn) + wk.half * out_cols + c0;
      row_base = wk.mb * 2 * S::BM + static_cast<int>(rank) * S::BM + q * 32;
    };
    Int8Work wk;
    int n0, c0, chunks, row_base;
    Int8Columns<kGated> cols;
    if (pair < p.num_work) {
      place(pair, wk, n0, c0, chunks, row_base);
      int8_fetch_columns<T, kGated>(p, n0, 32 * chunks, row_base + lane, lane, cols);
    }
    for (int i = pair; i < p.num_work; i += p.workers, ++local) {
      const int b = local & 1;
      const uint32_t use_ph = (static_cast<uint32_t>(local) >> 1) & 1u;
      const float sx = cols.sx;
      int8_put_columns<kGated>(cols, vec, lane);
      if (i + p.workers < p.num_work) {
        place(i + p.workers, wk, n0, c0, chunks, row_base);
        int8_fetch_columns<T, kGated>(p, n0, 32 * chunks, row_base + lane, lane, cols);
      }
      place(i, wk, n0, c0, chunks, row_base);
      const int live =
          row_base < p.M && n0 < p.N ? min(chunks, (p.N - n0 + 31) / 32) : 0;
      // A chunk's staging buffer is free, and its residual on the way, one chunk
      // ahead (8192 x 14336 x 4096 with a residual: 363 us without).
      const bool ahead = p.tma_out && live > 0;
      if (ahead) epi_chunk_begin<S::EPI_BUFS>(c, n0, row_base, lane, it);
      if (!mbar_wait_warp(bar(S::BAR_TFULL + b), use_ph, abort_flag)) {
        if (ahead) epi_chunk_drain<S::EPI_BUFS>(c, it);
        break;
      }
      tc_fence_after();
      const uint32_t tempty = mapa_shared(bar(S::BAR_TEMPTY + b), 0);
      const uint32_t acc = tmem_base + static_cast<uint32_t>(b * S::MAX_BN) +
                           (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(c0);
      if (live == 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tempty);
        continue;
      }
      // (the first chunk's residual was asked for before the accumulator was ready)
      uint32_t r[32], u[32];
      tmem_ld_32x32b_x32(acc, r);
      if (kGated) tmem_ld_32x32b_x32(acc + static_cast<uint32_t>(wk.bn / 2), u);
      bool ok = true;
#pragma unroll 1
      for (int ch = 0; ch < live; ++ch) {
        if (ahead && ch + 1 < live)
          epi_chunk_begin<S::EPI_BUFS>(c, n0 + 32 * (ch + 1), row_base, lane, it + 1);
        tmem_wait_ld();
        float v[32], w[32];
        int8_scale(v, r, sx, vec + 32 * ch, vec + 128 + 32 * ch);
        if (kGated) int8_scale(w, u, sx, vec + 256 + 32 * ch, vec + 384 + 32 * ch);
        if (ch + 1 < live) {
          tmem_ld_32x32b_x32(acc + static_cast<uint32_t>(32 * (ch + 1)), r);
          if (kGated) tmem_ld_32x32b_x32(acc + static_cast<uint32_t>(wk.bn / 2 + 32 * (ch + 1)), u);
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(tempty);
        }
        act_values<sizeof(T) == 4>(v, p.act);
        if (kGated) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= w[j];
        }
        if (!ahead) {
          int8_store_rows<T>(p, v, reinterpret_cast<float*>(c.ebuf_ptr0), row_base, n0 + 32 * ch,
                             lane);
          continue;
        }
        if constexpr (sizeof(T) == 2) {
          if (!epi_chunk_store<S::EPI_BUFS>(c, v, n0 + 32 * ch, row_base, lane, it, abort_flag)) {
            if (ch + 1 < live) {
              tmem_wait_ld();
              epi_chunk_drain<S::EPI_BUFS>(c, it + 1);
            }
            ok = false;
            break;
          }
        }
      }
      if (!ok) break;
    }
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }

  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, S::TMEM_COLS);
  }
}

}  // namespace dx
