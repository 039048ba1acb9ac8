// dx_moe.cuh — a mixture-of-experts layer for the few tokens of a serving step:
//   l = x Wr + br;  the k experts of the largest l (ties: lowest number);
//   w_e = exp(l_e) / sum of exp(l) over the chosen (or over all) experts;
//   y = r + sum_e w_e ((act(x Wg_e + bg_e) * (x Wu_e + bu_e)) Wo_e + bo_e)
// with T <= 64 tokens, E <= 256 experts, fp16 / bf16 weights as they lie in
// memory (Wg, Wu [E][D][H], Wo [E][H][D]).
//
// Bound by the weights of the experts that some token chose, each read once.
// Two launches:
//
//   moe_router_kernel  clusters of 8 CTAs, 8 tokens each: the CTAs split D, add
//     their 64-bit partial logits through distributed shared memory, and CTA i
//     picks token i's experts.
//   moe_experts_kernel  one CTA per SM, all resident (cooperative launch).
//     Phase 1 computes h = act(gate) * up of every chosen expert, phase 2 the
//     output; each phase's work is dealt evenly over the CTAs down to single
//     64-deep K blocks of a tile (MoePhase), so every SM streams the same bytes
//     whatever the sizes.  As in the skinny-M decode kernel the operands are
//     swapped: 128 weight columns are the MMA's rows (an MN-major operand, as W
//     lies in memory) and the tokens its columns.  All tokens go through every
//     chosen expert — the MMA has columns to spare, and no gathering is needed —
//     and the epilogue uses a token's column only where the token chose the
//     expert, so nothing of an expert (an infinity, a NaN) reaches other tokens.
//     h is kept as two 16-bit values (MoeHidden), both multiplied by Wo: a relative
//     error of 2^-17 (bf16) or 2^-22 (fp16), where one value has 2^-9 or 2^-12.  In
//     fp16 it also has a step of 2^-36, and h has to stay below 65504.
//     A tile that several CTAs share leaves fp32 partial sums; when all are
//     there the CTAs that end in the tile finish a share of its rows each,
//     adding the partials in CTA order (results do not depend on timing).
//     Between the phases the CTAs wait for one another, with the first weights
//     of phase 2 already on their way.
//
// The hidden rows have a place for every token of every chosen expert, so that a token
// tile is one box; rows that nobody wrote are loaded and multiplied too (64 tokens: 16 KB
// of token tiles, from L2, beside 32 KB of weights).
//
// Both launches (us, weights from HBM; the chosen experts' bytes at the measured copy
// rate): 1 token, 2 of 8 experts of 4096 x 14336 117 (108); 8 tokens, 8 of 64 of 2048 x
// 1024 96 (81); 64 tokens of the same 145 (123); 33 tokens, 4 of 16 of 1032 x 2824 69 (43).
//
// Every wait is bounded, as in dx_umma_gemm.cuh.
#pragma once

#include <type_traits>

#include "dx_epilogue.cuh"
#include "dx_moe_plan.cuh"
#include "dx_ptx.cuh"

namespace dx {

constexpr int kMoeMaxT = 64;
constexpr int kMoeMaxE = 256;
constexpr int kMoeMaxTop = 32;

// ---------------------------------------------------------------- router
constexpr int kRouterTokens = 8;  // tokens of a cluster = its CTAs
constexpr int kRouterThreads = 512;
constexpr int kRouterBlock = 32;  // rows of Wr that a warp's loads cover at once
constexpr int kRouterBatch = 4;   // such blocks on their way to a warp, a sum each

struct MoeRouterParams {
  const void* X;
  const void* Wr;  // [D][E], pitch ldwr
  const void* br;  // [E] or nullptr
  long long ldx, ldwr;
  int T, D, E, top, renormalize;
  int* ids;        // [T][top]
  float* weights;  // [T][top]
  int* counters;   // zeroed for moe_experts_kernel
  int num_counters;
};

// Unsigned key in the order of the doubles (a NaN sorts by its sign and bits).
__device__ __forceinline__ unsigned long long moe_key(double f) {
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(f));
  return (u >> 63) != 0 ? ~u : (u | (1ull << 63));
}

// The logits are sums in 64 bits: which experts are chosen is decided next to a
// border, where fp32 sums may order two of them otherwise.  8 tokens x 8 experts x 4
// rows are one 64-bit matrix instruction (tcgen05 has none of that type), to which a
// lane gives one value of X and one of Wr, straight from memory.  Sums by multiply-adds,
// a thread an expert, are bound by the tokens' values coming out of shared memory: the
// layer for 8 tokens, 64 experts of 4096 x 256 took 62.6 us with fp32 ones, 71.7 with
// 64-bit ones, 61.2 with this; 8 tokens, 64 of 2048 x 1024 92.3, 98.9 and 92.2.
template <typename T>
__global__ void __launch_bounds__(kRouterThreads) moe_router_kernel(const MoeRouterParams p) {
  using Tr = ElemTraits<T>;
  constexpr int kWarps = kRouterThreads / 32;
  __shared__ double s_part[kMoeMaxE / 8][kRouterTokens][8];  // [row group, 8 experts][token][expert]
  static_assert(kMoeMaxE / 8 >= kWarps, "a part for each warp");
  __shared__ double s_sum[kRouterTokens][kMoeMaxE];
  __shared__ double s_logit[kMoeMaxE];
  const int tid = static_cast<int>(threadIdx.x);
  const int warp = tid >> 5, lane = tid & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int t0 = static_cast<int>(blockIdx.x) / kRouterTokens * kRouterTokens;
  const int tokens = min(kRouterTokens, p.T - t0);
  grid_dependency_wait();
  grid_launch_dependents();
  if (blockIdx.x == 0)
    for (int i = tid; i < p.num_counters; i += kRouterThreads) p.counters[i] = 0;

  // This CTA's rows of Wr, a multiple of 8; warps as row groups x tiles of 8 experts.
  const int slice = ((p.D + kRouterTokens - 1) / kRouterTokens + 7) / 8 * 8;
  const int k_begin = rank * slice, k_end = min(p.D, k_begin + slice);
  const int tiles = (p.E + 7) / 8;
  const int across = min(tiles, kWarps), groups = kWarps / across;
  const int group = warp / across;
  const int m = lane >> 2, j = lane & 3;  // the lane's token and expert of 8; its rows, 8 j on
  if (group < groups) {
    const T* const x_row = static_cast<const T*>(p.X) + static_cast<long long>(t0 + m) * p.ldx;
    for (int tile = warp % across; tile < tiles; tile += across) {
      const int e = tile * 8 + m;
      const T* const w_col = static_cast<const T*>(p.Wr) + e;
      double c[kRouterBatch][2] = {};  // (sums that do not wait for one another)
      for (int k0 = k_begin + group * kRouterBlock; k0 < k_end;
           k0 += groups * kRouterBlock * kRouterBatch) {
        T w[kRouterBatch][8];
        __align__(16) T x[kRouterBatch][8];
#pragma unroll
        for (int i = 0; i < kRouterBatch; ++i) {
          const int k = k0 + i * groups * kRouterBlock + 8 * j;
          const bool in = k < k_end;  // (all eight rows or none)
          *reinterpret_cast<uint4*>(x[i]) = in && m < tokens
                                                ? *reinterpret_cast<const uint4*>(x_row + k)
                                                : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int r = 0; r < 8; ++r)
            w[i][r] = in && e < p.E ? w_col[(k + r) * p.ldwr] : Tr::from_float(0.0f);
        }
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
          for (int i = 0; i < kRouterBatch; ++i)
            mma_f64(c[i], static_cast<double>(Tr::to_float(x[i][r])),
                    static_cast<double>(Tr::to_float(w[i][r])));
      }
      double* const to = &s_part[group * tiles + tile][m][2 * j];
#pragma unroll
      for (int h = 0; h < 2; ++h) to[h] = (c[0][h] + c[1][h]) + (c[2][h] + c[3][h]);
    }
  }
  __syncthreads();
  for (int i = tid; i < tokens * p.E; i += kRouterThreads) {
    const int t = i / p.E, e = i - t * p.E;
    double s = 0.0;
    for (int g = 0; g < groups; ++g) s += s_part[g * tiles + e / 8][t][e % 8];
    s_sum[t][e] = s;
  }
  cluster_sync();
  const int token = t0 + rank;
  if (rank < tokens) {
    for (int i = tid; i < p.E; i += kRouterThreads) {
      double s = 0.0;
#pragma unroll
      for (int c = 0; c < kRouterTokens; ++c)
        s += ld_shared_cluster_f64(
            mapa_shared(smem_u32(&s_sum[rank][i]), static_cast<uint32_t>(c)));
      if (p.br != nullptr) s += static_cast<double>(Tr::to_float(static_cast<const T*>(p.br)[i]));
      s_logit[i] = s;
    }
  }
  cluster_sync();  // no CTA leaves while its sums are read
  if (rank >= tokens || tid >= 32) return;

  // One warp: lane l holds experts l, l + 32, ...
  constexpr int kPer = kMoeMaxE / 32;
  unsigned long long key[kPer];  // 0: absent or taken (no number's key is 0, a NaN's may be)
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int ee = i * 32 + tid;
    key[i] = ee < p.E ? max(moe_key(s_logit[ee]), 1ull) : 0ull;
  }
  double top_logit = 0.0;
  float sum = 0.0f, mine = 0.0f;
  int my_id = 0;
  for (int j = 0; j < p.top; ++j) {
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) best = max(best, key[i]);
    const uint32_t high = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(best >> 32));
    const uint32_t low = __reduce_max_sync(
        0xffffffffu, static_cast<uint32_t>(best >> 32) == high ? static_cast<uint32_t>(best) : 0u);
    best = (static_cast<unsigned long long>(high) << 32) | low;
    uint32_t at = kMoeMaxE;
#pragma unroll
    for (int i = kPer - 1; i >= 0; --i)
      if (key[i] == best) at = static_cast<uint32_t>(i * 32 + tid);
    const int id = static_cast<int>(__reduce_min_sync(0xffffffffu, at));
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i * 32 + tid == id) key[i] = 0;
    const double l = s_logit[id];
    if (j == 0) top_logit = l;
    const float x = expf(static_cast<float>(l - top_logit));
    sum += x;
    if (tid == j) {
      mine = x;
      my_id = id;
    }
  }
  if (!p.renormalize) {
    sum = 0.0f;
    for (int ee = tid; ee < p.E; ee += 32) sum += expf(static_cast<float>(s_logit[ee] - top_logit));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if (tid < p.top) {
    p.ids[token * p.top + tid] = my_id;
    p.weights[token * p.top + tid] = mine / sum;
  }
}

// --------------------------------------------------------------- experts
struct MoeParams {
  int T, D, H, E, top, act;
  int kb_d, nt_h;  // phase 1: 64-deep blocks of D, 128-column tiles of H
  int kb_h, nt_d;  // phase 2: 64-deep blocks of H, 256-column tiles of D
  int mn;          // tokens padded to a multiple of 16
  int stages;
  const int* ids;
  const float* weights;
  const void *bg, *bu, *bo;  // [E][H], [E][H], [E][D] or nullptr
  const void* residual;
  long long ldr;
  void* Y;
  long long ldy;
  void *h_hi, *h_lo;  // [chosen experts][T][H]
  float* partials;    // [CTA][kMoeSlots][2][T][128]
  int* counters;      // [2 phases][CTA] tile arrivals, then the phase barrier; zero before
};

struct MoeShape {
  static constexpr int BK = 64;
  static constexpr int BOX_BYTES = 64 * BK * 2;  // [64 k x 64 n]
  static constexpr int W_BYTES = 4 * BOX_BYTES;  // 256 columns
  // 128 KB of weights in flight an SM; more of them only wait for one another (8
  // tokens, 64 experts: 3 us longer with 5 stages, 5 with 6, 11 with 2).
  static constexpr int MAX_STAGES = 4;
  static constexpr int THREADS = 192;
  // Behind the ring (W tiles, then token tiles):
  static constexpr int OFF_MASK = 0;                         // [E] tokens, 64 bits
  static constexpr int OFF_LIST = OFF_MASK + kMoeMaxE * 8;   // chosen experts
  static constexpr int OFF_ROWW = OFF_LIST + kMoeMaxE * 4;   // [2][64] weights of a run
  static constexpr int OFF_BAR = OFF_ROWW + 2 * kMoeMaxT * 4;
  static constexpr int BAR_FULL = 0;
  static constexpr int BAR_EMPTY = MAX_STAGES;
  static constexpr int BAR_TFULL = 2 * MAX_STAGES;
  static constexpr int BAR_TEMPTY = BAR_TFULL + 2;
  static constexpr int BAR_DRAIN = BAR_TEMPTY + 2;
  static constexpr int NUM_BARS = BAR_DRAIN + 1;
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;  // tmem base, abort flag, experts, ok
  static constexpr int OFF_IDS = OFF_MISC + 32;  // [T * top] experts, then as many weights
  static constexpr int stage_bytes(int mn) { return W_BYTES + 2 * mn * BK * 2; }
  static constexpr int smem_bytes(int mn, int stages, int pairs) {
    return 1024 + stages * stage_bytes(mn) + OFF_IDS + 8 * pairs;
  }
  static constexpr int max_stages(int mn, int pairs) {
    const int n = (227 * 1024 - smem_bytes(mn, 0, pairs)) / stage_bytes(mn);
    return n < MAX_STAGES ? n : MAX_STAGES;
  }
};

// Counts a CTA in: what it wrote before, and what threads wrote that it met at a barrier
// since, is seen by whoever sees the count.  (One release for the CTA: with a fence
// by each of 128 threads a call took 1.2 to 1.8 us longer.)
__device__ __forceinline__ void moe_arrive(int* ctr) {
  asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(ctr) : "memory");
}

// Bounded wait until *ctr reaches `target` (every CTA of the launch is resident).
__device__ __forceinline__ bool moe_wait(const int* ctr, int target, volatile int* abort_flag) {
  const uint64_t t0 = global_timer_ns();
  uint32_t spins = 0;
  while (true) {
    int n;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(n) : "l"(ctr) : "memory");
    if (n >= target) return true;
    __nanosleep(20);
    if ((++spins & 63u) == 0) {
      if (*abort_flag) return false;
      if (global_timer_ns() - t0 > kWaitLimitNs) {
        *abort_flag = 1;
        report_timeout();
        return false;
      }
    }
  }
}

// h as hi + lo / kScale of type T.  bf16's lo has the exponents it needs; fp16's is
// kept 2^11 times as large, about as large as hi, so that it does not end among the
// subnormals for every h below 2^-3, and has sums of its own in TMEM (X of scale 0.001
// and Wo 4000 times as large as usual: outputs 3% of their norm off otherwise, 0.02% so).
template <typename T>
struct MoeHidden {
  static constexpr bool kApart = !ElemTraits<T>::kIsBf16;
  static constexpr float kScale = kApart ? 2048.0f : 1.0f;
};

template <typename T>
__device__ __forceinline__ void moe_split(float h, T& hi, T& lo) {
  using Tr = ElemTraits<T>;
  hi = Tr::from_float(h);
  const float rest = h - Tr::to_float(hi);
  lo = Tr::from_float(rest - rest == 0.0f ? rest * MoeHidden<T>::kScale : 0.0f);  // an infinite hi has no lo
}

template <typename T>
__device__ __forceinline__ float moe_bias(const T* b, long long i) {
  return b != nullptr ? ElemTraits<T>::to_float(b[i]) : 0.0f;
}

template <int MN, typename T>
__global__ void __launch_bounds__(MoeShape::THREADS, 1)
    moe_experts_kernel(const __grid_constant__ CUtensorMap tmG,
                       const __grid_constant__ CUtensorMap tmU,
                       const __grid_constant__ CUtensorMap tmO,
                       const __grid_constant__ CUtensorMap tmX,
                       const __grid_constant__ CUtensorMap tmHi,
                       const __grid_constant__ CUtensorMap tmLo, const MoeParams p) {
  using S = MoeShape;
  using Tr = ElemTraits<T>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t base = (raw_u32 + 1023u) & ~1023u;
  uint8_t* const base_ptr = smem_raw + (base - raw_u32);
  const int stages = p.stages;
  const uint32_t t_bytes = static_cast<uint32_t>(p.mn) * S::BK * 2;  // one token tile
  const uint32_t sW = base;
  const uint32_t sT = base + static_cast<uint32_t>(stages) * S::W_BYTES;
  const uint32_t tail = static_cast<uint32_t>(stages) * (S::W_BYTES + 2 * t_bytes);
  uint8_t* const tail_ptr = base_ptr + tail;
  const uint32_t bars = base + tail + S::OFF_BAR;
  int* const s_ids = reinterpret_cast<int*>(tail_ptr + S::OFF_IDS);
  float* const s_wts = reinterpret_cast<float*>(s_ids + p.T * p.top);
  uint32_t* const s_mask = reinterpret_cast<uint32_t*>(tail_ptr + S::OFF_MASK);
  int* const s_list = reinterpret_cast<int*>(tail_ptr + S::OFF_LIST);
  float* const s_roww = reinterpret_cast<float*>(tail_ptr + S::OFF_ROWW);
  uint32_t* const tmem_word = reinterpret_cast<uint32_t*>(tail_ptr + S::OFF_MISC);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tail_ptr + S::OFF_MISC + 4);
  int* const s_chosen = reinterpret_cast<int*>(tail_ptr + S::OFF_MISC + 8);
  volatile int* const s_ok = reinterpret_cast<volatile int*>(tail_ptr + S::OFF_MISC + 12);
  auto bar = [bars](int i) { return bars + 8u * static_cast<uint32_t>(i); };
  // Two buffers x two halves, then the same for the lo sums where they are apart.
  constexpr bool kApart = MoeHidden<T>::kApart;
  constexpr uint32_t kTmemCols = (kApart ? 8 : 4) * MN;

  const int tid = static_cast<int>(threadIdx.x);
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int lane = tid & 31;
  const int g = static_cast<int>(blockIdx.x);

  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(bar(S::BAR_FULL + s), 1);
      mbar_init(bar(S::BAR_EMPTY + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(S::BAR_TFULL + b), 1);
      mbar_init(bar(S::BAR_TEMPTY + b), 4);
    }
    mbar_init(bar(S::BAR_DRAIN), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmG);
    tma_prefetch_desc(&tmU);
    tma_prefetch_desc(&tmO);
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmHi);
    tma_prefetch_desc(&tmLo);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_word), kTmemCols);
    tmem_relinquish();
  }
  for (int i = tid; i < 2 * p.E; i += S::THREADS) s_mask[i] = 0;
  // The routing, the zeroed counters and X come from launches before this one.
  grid_dependency_wait();
  const int pairs = p.T * p.top;
  __syncthreads();
  for (int i = tid; i < pairs; i += S::THREADS) {
    const int e = p.ids[i], t = i / p.top;
    s_ids[i] = e;
    s_wts[i] = p.weights[i];
    atomicOr(&s_mask[2 * e + (t >> 5)], 1u << (t & 31));
  }
  __syncthreads();
  if (warp == 0) {  // the chosen experts in order of their numbers
    int n = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      const bool c = e < p.E && (s_mask[2 * e] | s_mask[2 * e + 1]) != 0;
      const uint32_t vote = __ballot_sync(0xffffffffu, c);
      if (c) s_list[n + __popc(vote & ((1u << lane) - 1u))] = e;
      n += __popc(vote);
    }
    if (lane == 0) *s_chosen = n;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_word;
  const int chosen = *s_chosen;
  int* const barrier_ctr = p.counters + 2 * gridDim.x;

  if (warp == 0) {
    // ------------------------------------------------------ TMA producer
    if (lane == 0) {
      // One thread feeds the SM, so it steps through runs and counts stages: with
      // the divisions of MoePhase::item per unit it was what bound the kernel (8
      // tokens, 64 experts: 23 us longer with two more divisions).
      struct Cursor {
        MoeRun r;
        int at, i;  // the run's position in the phase, the block within the run
        int stage;
        uint32_t parity;
      };
      const uint64_t pol = make_l2_policy_evict_first();
      const uint64_t keep = make_l2_policy_evict_last();
      uint32_t issued = 0;
      bool ok = true;
      Cursor w{}, t{};  // the next weights and the next tokens to load
      auto seek = [](const MoePhase& f, Cursor& c) {
        c.at = c.i = 0;
        f.run(0, c.r);
      };
      auto advance = [stages](const MoePhase& f, Cursor& c) {
        if (++c.stage == stages) {
          c.stage = 0;
          c.parity ^= 1u;
        }
        if (++c.i == c.r.len) {
          c.at += c.r.len;
          c.i = 0;
          f.run(c.at, c.r);
        }
      };
      // The stage of w.i, when it is free, with the weights on their way.
      auto load_w = [&](const MoePhase& f, uint32_t bytes) {
        const int s = w.stage;
        if (!mbar_wait(bar(S::BAR_EMPTY + s), w.parity ^ 1u, abort_flag)) return false;
        const uint32_t fb = bar(S::BAR_FULL + s);
        mbar_arrive_expect_tx(fb, bytes);
        const int e = s_list[w.r.a];
        const int k = (w.r.kb0 + w.i) * S::BK;
        const uint32_t dst = sW + s * S::W_BYTES;
        if (!f.second) {
          const int n = (w.r.tile - w.r.a * f.nt) * 128;
          tma_load_3d_hint(&tmG, dst, fb, n, k, e, pol);
          tma_load_3d_hint(&tmG, dst + S::BOX_BYTES, fb, n + 64, k, e, pol);
          tma_load_3d_hint(&tmU, dst + 2 * S::BOX_BYTES, fb, n, k, e, pol);
          tma_load_3d_hint(&tmU, dst + 3 * S::BOX_BYTES, fb, n + 64, k, e, pol);
        } else {
          const int n = w.r.tile * 256;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            tma_load_3d_hint(&tmO, dst + j * S::BOX_BYTES, fb, n + 64 * j, k, e, pol);
        }
        advance(f, w);
        ++issued;
        return true;
      };
      auto load_t = [&](const MoePhase& f) {
        const uint32_t fb = bar(S::BAR_FULL + t.stage);
        const uint32_t dst = sT + static_cast<uint32_t>(t.stage) * 2 * t_bytes;
        const int k = (t.r.kb0 + t.i) * S::BK;
        if (!f.second) {
          tma_load_2d_hint(&tmX, dst, fb, k, 0, keep);
        } else {
          tma_load_2d_hint(&tmHi, dst, fb, k, t.r.a * p.T, keep);
          tma_load_2d_hint(&tmLo, dst + t_bytes, fb, k, t.r.a * p.T, keep);
        }
        advance(f, t);
      };
      for (int ph = 0; ok && ph < 2; ++ph) {
        const MoePhase f = moe_phase(p, chosen, ph != 0);
        const uint32_t bytes = S::W_BYTES + (ph != 0 ? 2 * t_bytes : t_bytes);
        const int items = f.count();
        seek(f, w);
        seek(f, t);
        int u = 0;
        if (ph != 0) {
          // A ring of phase 2's weights before every h is written.
          const int early = min(stages, items);
          while (u < early && load_w(f, bytes)) ++u;
          ok = u == early && moe_wait(barrier_ctr, static_cast<int>(gridDim.x), abort_flag);
          fence_proxy_async_global();
          // (also when giving up, so that the started stages complete)
          for (int i = 0; i < u; ++i) load_t(f);
        }
        for (; ok && u < items; ++u) {
          ok = load_w(f, bytes);
          if (ok) load_t(f);
        }
      }
      // Loads in flight land before the shared memory is released.
      const uint32_t n_drain = min(issued, static_cast<uint32_t>(stages));
      for (uint32_t i = issued - n_drain; i < issued; ++i)
        mbar_wait_drain(bar(S::BAR_FULL + static_cast<int>(i % stages)), (i / stages) & 1u);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------- MMA issuer
    const uint32_t idesc = umma_idesc_f16(Tr::kIsBf16, 128, p.mn, true, false);
    const bool issuer = elect_one();
    int s = 0, local = 0;
    uint32_t par = 0;
    bool ok = true;
    for (int ph = 0; ok && ph < 2; ++ph) {
      const MoePhase f = moe_phase(p, chosen, ph != 0);
      MoeRun r;
      for (int u = 0; ok && f.run(u, r); u += r.len, ++local) {
        const int b = local & 1;
        if (!mbar_wait_warp(bar(S::BAR_TEMPTY + b), ((static_cast<uint32_t>(local) >> 1) & 1u) ^ 1u,
                            abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(b * 2 * MN);
        for (int i = 0; i < r.len; ++i) {
          if (!mbar_wait_warp(bar(S::BAR_FULL + s), par, abort_flag)) {
            ok = false;
            break;
          }
          if (issuer) {
            const uint64_t td = smem_desc_sw128(sT + static_cast<uint32_t>(s) * 2 * t_bytes, 16, 1024);
            const uint64_t lo = smem_desc_sw128(sT + static_cast<uint32_t>(s) * 2 * t_bytes + t_bytes,
                                                16, 1024);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              // 128 columns of W: MN-major, two 64-wide groups one box apart,
              // 8-row K groups 1024 B apart; +2048 B per K = 16 step.
              const uint64_t wd =
                  smem_desc_sw128(sW + s * S::W_BYTES + h * 2 * S::BOX_BYTES, S::BOX_BYTES, 1024);
              const uint32_t dh = d + static_cast<uint32_t>(h * MN);
#pragma unroll
              for (int k = 0; k < S::BK / 16; ++k)
                umma_f16(dh, wd + 128ull * k, td + 2ull * k, idesc, (i != 0 || k != 0) ? 1u : 0u);
              if (ph != 0) {
#pragma unroll
                for (int k = 0; k < S::BK / 16; ++k)
                  umma_f16(kApart ? dh + 4 * MN : dh, wd + 128ull * k, lo + 2ull * k, idesc,
                           (!kApart || i != 0 || k != 0) ? 1u : 0u);
              }
            }
            umma_commit(bar(S::BAR_EMPTY + s));
          }
          __syncwarp();
          if (++s == stages) {
            s = 0;
            par ^= 1u;
          }
        }
        if (ok && issuer) umma_commit(bar(S::BAR_TFULL + b));
        __syncwarp();
      }
    }
    // Every MMA issued so far completes before TMEM can be freed.
    if (issuer) umma_commit(bar(S::BAR_DRAIN));
    mbar_wait_drain(bar(S::BAR_DRAIN), 0);
    __syncwarp();
  } else {
    // --------------------------------------------------------- epilogue
    const int q = warp & 3;
    const int et = tid - 64;
    const int n = q * 32 + lane;  // column within a 128-column half
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(q * 32) << 16);
    const T* const bg = static_cast<const T*>(p.bg);
    const T* const bu = static_cast<const T*>(p.bu);
    const T* const bo = static_cast<const T*>(p.bo);
    T* const h_hi = static_cast<T*>(p.h_hi);
    T* const h_lo = static_cast<T*>(p.h_lo);
    int local = 0;
    bool ok = true;
    auto chosen_by = [&](int e) {  // the tokens of expert e
      return s_mask[2 * e] | (static_cast<unsigned long long>(s_mask[2 * e + 1]) << 32);
    };
    // A slot of a CTA's partial sums (MoePhase::slot): [2][T][128].
    const long long slot_floats = static_cast<long long>(2 * p.T) * 128;
    auto part = [&](int cta, int slot) { return p.partials + (cta * kMoeSlots + slot) * slot_floats; };
    // The tile whose partial sums this CTA has just written: `peers` CTAs from
    // `first` on have a share of it, `sum` points at the first one's, and this CTA
    // finishes every shares'th row from `share` on (-1: none).  Counts the CTA in;
    // where the tile is its last one, waits until all are there.
    const float* sum = nullptr;
    int first = 0, peers = 1, share = 0, shares = 1;
    auto join = [&](const MoePhase& f, int tile, int slot, bool whole) {
      first = g;
      peers = shares = 1;
      share = 0;
      if (!whole) {
        const int us = (tile - f.whole) * f.per_tile, ue = us + f.per_tile;
        first = f.cta_of(us);
        const int last = f.cta_of(ue - 1);
        peers = last - first + 1;
        shares = last - first + (f.begin(last + 1) == ue ? 1 : 0);
        share = f.u1 <= ue ? g - first : -1;
        if (first != g) slot = f.slot_of(first, tile);
      }
      sum = part(first, slot);
      named_bar_sync(1, 128);
      if (et == 0) {
        int* const ctr = p.counters + (f.second ? gridDim.x : 0) + first;
        if (!whole) moe_arrive(ctr);
        *s_ok = whole || share < 0 || moe_wait(ctr, peers, abort_flag) ? 1 : 0;
      }
      named_bar_sync(1, 128);  // (behind it the partials are read from L2, past L1)
      return *s_ok != 0;
    };
    // Columns 4 lane .. 4 lane + 3 of kRows rows of the tile, `apart` rows apart, added
    // in CTA order.
    auto row_sums = [&](auto rows, int row, int apart, float4* t) {
      constexpr int kRows = decltype(rows)::value, kBatch = 8 / kRows;
      const long long at = static_cast<long long>(row) * 128 + 4 * lane;
      const float* const next = part(first + 1, 0) + at;
#pragma unroll
      for (int j = 0; j < kRows; ++j)
        t[j] = __ldcg(reinterpret_cast<const float4*>(sum + at + j * apart * 128));
#pragma unroll 1
      for (int i = 0; i < peers - 1; i += kBatch) {
        float4 v[kBatch][kRows];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
          for (int j = 0; j < kRows; ++j)
            v[k][j] = i + k < peers - 1
                          ? __ldcg(reinterpret_cast<const float4*>(
                                next + kMoeSlots * slot_floats * (i + k) + j * apart * 128))
                          : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
          for (int j = 0; j < kRows; ++j) {
            t[j].x += v[k][j].x;
            t[j].y += v[k][j].y;
            t[j].z += v[k][j].z;
            t[j].w += v[k][j].w;
          }
      }
    };

    {  // ---- phase 1: h
      const MoePhase f = moe_phase(p, chosen, false);
      MoeRun r;
      for (int u = 0; ok && f.run(u, r); u += r.len, ++local) {
        const int b = local & 1;
        const int e = s_list[r.a];
        const int col0 = (r.tile - r.a * f.nt) * 128;
        const unsigned long long mask = chosen_by(e);
        const bool whole = r.len == f.per_tile;
        const int slot = f.slot(r.tile, whole);
        const bool live = col0 + n < p.H;
        float vg = 0.0f, vu = 0.0f;
        if (whole && live) {
          vg = moe_bias(bg, static_cast<long long>(e) * p.H + col0 + n);
          vu = moe_bias(bu, static_cast<long long>(e) * p.H + col0 + n);
        }
        // (the vote keeps the four warps together where a wait gives up)
        ok = named_bar_all(1, 128, mbar_wait(bar(S::BAR_TFULL + b),
                                             (static_cast<uint32_t>(local) >> 1) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = lane_addr + static_cast<uint32_t>(b * 2 * MN);
#pragma unroll 1
        for (int mc = 0; mc < p.T; mc += 16) {
          const uint32_t some = static_cast<uint32_t>(mask >> mc) & 0xffffu;
          if (some == 0) continue;
          uint32_t a0[16], a1[16];
          tmem_ld_32x32b_x16(acc + static_cast<uint32_t>(mc), a0);
          tmem_ld_32x32b_x16(acc + static_cast<uint32_t>(MN + mc), a1);
          tmem_wait_ld();
          if (!whole) {
            float* const to = part(g, slot) + mc * 128 + n;
            float* const to1 = to + p.T * 128;
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if ((some >> j) & 1u) {
                to[j * 128] = __uint_as_float(a0[j]);
                to1[j * 128] = __uint_as_float(a1[j]);
              }
          } else {
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(a0[j]) + vg;
            act_values<false>(v, p.act);
            const long long at = (static_cast<long long>(r.a) * p.T + mc) * p.H + col0 + n;
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (((some >> j) & 1u) && live) {
                T hi, lo;
                moe_split(v[j] * (__uint_as_float(a1[j]) + vu), hi, lo);
                h_hi[at + static_cast<long long>(j) * p.H] = hi;
                h_lo[at + static_cast<long long>(j) * p.H] = lo;
              }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(S::BAR_TEMPTY + b));
        if (whole) continue;
        // (loaded before the wait for the other CTAs' sums)
        const int col = col0 + 4 * lane;
        float vg4[4] = {0.0f, 0.0f, 0.0f, 0.0f}, vu4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (col < p.H) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            vg4[k] = moe_bias(bg, static_cast<long long>(e) * p.H + col + k);
            vu4[k] = moe_bias(bu, static_cast<long long>(e) * p.H + col + k);
          }
        }
        ok = join(f, r.tile, slot, false);
        if (!ok || share < 0) continue;
        // This CTA's share of the tokens, a warp each; a lane has four columns.
        int i = 0;
#pragma unroll 1
        for (unsigned long long left = mask; left != 0; left &= left - 1, ++i) {
          if (i % (4 * shares) != share * 4 + q) continue;
          const int m = __ffsll(static_cast<long long>(left)) - 1;
          float4 t[2];  // gate, up
          row_sums(std::integral_constant<int, 2>(), m, p.T, t);
          if (col >= p.H) continue;
          float v[4] = {t[0].x, t[0].y, t[0].z, t[0].w}, w[4] = {t[1].x, t[1].y, t[1].z, t[1].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[k] += vg4[k];
            w[k] += vu4[k];
          }
          act_values<false>(v, p.act);
          __align__(8) T hi[4];
          __align__(8) T lo[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) moe_split(v[k] * w[k], hi[k], lo[k]);
          const long long at = (static_cast<long long>(r.a) * p.T + m) * p.H + col;
          *reinterpret_cast<uint2*>(h_hi + at) = *reinterpret_cast<const uint2*>(hi);
          *reinterpret_cast<uint2*>(h_lo + at) = *reinterpret_cast<const uint2*>(lo);
        }
      }
    }
    // Everything this CTA wrote of h, before any CTA reads it by TMA (the proxies'
    // fence is the reader's, behind its wait).
    named_bar_sync(1, 128);
    if (et == 0 && ok) moe_arrive(barrier_ctr);

    {  // ---- phase 2: the output
      const MoePhase f = moe_phase(p, chosen, true);
      T* const Y = static_cast<T*>(p.Y);
      const T* const res = static_cast<const T*>(p.residual);
      float y[2][MN];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < MN; ++m) y[h][m] = 0.0f;
      MoeRun r;
      for (int u = 0; ok && f.run(u, r); u += r.len, ++local) {
        const int b = local & 1;
        const int e = s_list[r.a];
        const unsigned long long mask = chosen_by(e);
        // The tokens' weights for this expert.
        float* const roww = s_roww + b * kMoeMaxT;
        if (et < p.T) {
          float w = 0.0f;
#pragma unroll 4
          for (int j = 0; j < p.top; ++j) {
            const float wj = s_wts[et * p.top + j];
            w = s_ids[et * p.top + j] == e ? wj : w;
          }
          roww[et] = w;
        }
        float vb[2] = {0.0f, 0.0f};
        if (r.kb0 == 0) {  // (each expert's bias once a tile)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int c = r.tile * 256 + 128 * h + n;
            if (c < p.D) vb[h] = moe_bias(bo, static_cast<long long>(e) * p.D + c);
          }
        }
        ok = named_bar_all(1, 128, mbar_wait(bar(S::BAR_TFULL + b),
                                             (static_cast<uint32_t>(local) >> 1) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = lane_addr + static_cast<uint32_t>(b * 2 * MN);
#pragma unroll
        for (int mc = 0; mc < MN; mc += 16) {
          const uint32_t some = static_cast<uint32_t>(mask >> mc) & 0xffffu;
          if (some != 0) {
            float w[16];
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<float4*>(w + j) = *reinterpret_cast<const float4*>(roww + mc + j);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t v[16], l[kApart ? 16 : 1];
              tmem_ld_32x32b_x16(acc + static_cast<uint32_t>(h * MN + mc), v);
              if constexpr (kApart)
                tmem_ld_32x32b_x16(acc + static_cast<uint32_t>(4 * MN + h * MN + mc), l);
              tmem_wait_ld();
              if constexpr (kApart) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  v[j] = __float_as_uint(fmaf(__uint_as_float(l[j]), 1.0f / MoeHidden<T>::kScale,
                                              __uint_as_float(v[j])));
              }
#pragma unroll
              for (int j = 0; j < 16; ++j) {  // (a branch a token: 64 tokens 1 us longer)
                const float sum = fmaf(w[j], __uint_as_float(v[j]) + vb[h], y[h][mc + j]);
                y[h][mc + j] = ((some >> j) & 1u) != 0 ? sum : y[h][mc + j];
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(S::BAR_TEMPTY + b));
        // More of this tile to come?
        MoeRun after;
        if (f.run(u + r.len, after) && after.tile == r.tile) continue;
        const int us = (r.tile - f.whole) * f.per_tile;
        const bool whole = r.tile < f.whole || (f.u0 <= us && f.u1 >= us + f.per_tile);
        const int slot = f.slot(r.tile, whole);
        float* const to = part(g, slot) + n;
        float* const to1 = to + p.T * 128;
#pragma unroll
        for (int m = 0; m < MN; ++m) {
          if (m < p.T) {
            to[m * 128] = y[0][m];
            to1[m * 128] = y[1][m];
          }
          y[0][m] = y[1][m] = 0.0f;
        }
        ok = join(f, r.tile, slot, whole);
        if (!ok || share < 0) continue;
        // This CTA's share of the rows (halves of a token's 256 columns), a warp each.
#pragma unroll 1
        for (int row = share * 4 + q; row < 2 * p.T; row += 4 * shares) {
          const int h = row >= p.T ? 1 : 0, m = row - h * p.T;
          const int c = r.tile * 256 + 128 * h + 4 * lane;
          float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          if (res != nullptr && c < p.D) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = Tr::to_float(res[m * p.ldr + c + k]);
          }
          float4 t;
          row_sums(std::integral_constant<int, 1>(), row, 0, &t);
          if (c >= p.D) continue;
          const float s[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) Y[m * p.ldy + c + k] = Tr::from_float(s[k] + v[k]);
        }
      }
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

}  // namespace dx
