// dx_int8_api.cuh — host side of the 8-bit integer linear layers: argument
// checks, kernel choice, TMA descriptors and launches.  Part of dx_api.cu
// (it uses that file's helpers).
#pragma once

#include "dx_int8.cuh"
#include "dx_pack.cuh"
#include "dx_quant.cuh"

namespace {

using dx::Int8PairShape;
using dx::Int8Params;
using dx::Int8TileShape;
using dx::QuantParams;

// |sum| <= K * 128 * 128 < 2^31.
constexpr int64_t kInt8MaxK = 131071;

int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

int elem_size(int dtype) { return dtype == DX_DTYPE_F32 ? 4 : 2; }

// Whether every pointer is at a multiple of `size` bytes, as its elements have to be.
template <typename... P>
bool element_aligned(int size, P... p) {
  return ((reinterpret_cast<uintptr_t>(p) | ...) & static_cast<uintptr_t>(size - 1)) == 0;
}

bool float_dtype(int dtype) { return dtype >= DX_DTYPE_F32 && dtype <= DX_DTYPE_BF16; }

// 8-bit matrix of `rows` rows of `k` bytes, a [box_rows x 128 byte] box.
int make_tmap_i8(CUtensorMap* m, const void* ptr, int64_t k, int64_t rows, int64_t ld,
                 uint32_t box_rows, const char* name) {
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {128, box_rows};
  cuuint32_t es[2] = {1, 1};
  const CUresult r = g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims,
                              strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(DX_ERR_CUDA, "cuTensorMapEncodeTiled(%s) failed with CUresult %d", name,
                static_cast<int>(r));
  return DX_OK;
}

// ---------------------------------------------------------- quantisation
template <typename T, int THREADS, bool kVec>
int launch_quantize(const QuantParams& p, int sms, cudaStream_t s) {
  // 1024 threads an SM, each CTA taking every grid'th row.
  const int grid = std::min(p.M, sms * (1024 / THREADS));
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = launch_config(grid, THREADS, 0, s, 1, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, dx::quantize_rows_kernel<T, THREADS, kVec>, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch quantize_rows_kernel");
  return DX_OK;
}

template <typename T, bool kVec>
int quantize_typed(const QuantParams& p, int sms, cudaStream_t s) {
  // Few rows: the latency of a row counts, one vector a thread; many: all that
  // its registers hold, so that a row takes few threads and many are in flight.
  constexpr int kRegs = dx::kQuantRegsOf<T>;
  const int vectors = (p.K + dx::kQuantVec - 1) / dx::kQuantVec;
  const int threads = p.M <= 4 * sms ? vectors : (vectors + kRegs - 1) / kRegs;
  if (threads <= 128) return launch_quantize<T, 128, kVec>(p, sms, s);
  if (threads <= 256) return launch_quantize<T, 256, kVec>(p, sms, s);
  if (threads <= 512) return launch_quantize<T, 512, kVec>(p, sms, s);
  return launch_quantize<T, 1024, kVec>(p, sms, s);
}

int run_quantize(const void* X, void* Q, float* scale, int64_t M, int64_t K, int64_t ldx,
                 int64_t ldq, int dtype, int sms, cudaStream_t s) {
  QuantParams p{};
  p.X = X;
  p.Q = static_cast<int8_t*>(Q);
  p.scale = scale;
  p.M = static_cast<int>(M);
  p.K = static_cast<int>(K);
  p.ldx = ldx;
  p.ldq = ldq;
  const bool vec = K % dx::kQuantVec == 0 && aligned16(X) && (ldx * elem_size(dtype)) % 16 == 0 &&
                   aligned16(Q) && ldq % 8 == 0;
  if (dtype == DX_DTYPE_F32)
    return vec ? quantize_typed<float, true>(p, sms, s) : quantize_typed<float, false>(p, sms, s);
  if (dtype == DX_DTYPE_F16)
    return vec ? quantize_typed<__half, true>(p, sms, s) : quantize_typed<__half, false>(p, sms, s);
  return vec ? quantize_typed<__nv_bfloat16, true>(p, sms, s)
             : quantize_typed<__nv_bfloat16, false>(p, sms, s);
}

// --------------------------------------------------------------- problem
struct Int8Problem {
  const void* X;       // 8-bit rows, or a float type that is quantised first
  int x_dtype;
  const float* x_scale;
  const void *W, *W2;
  const float *w_scale, *w2_scale;
  const void *bias, *bias2, *R;
  void* Y;
  int64_t M, N, K, ldx, ldw, ldw2, ldr, ldy;
  int dtype, act, kernel;
  bool gated;
  void* ws;
  size_t ws_bytes;
  cudaStream_t stream;
  bool w_early = false;
};

size_t int8_scale_bytes(int64_t M) { return static_cast<size_t>(round_up(M * 4, 256)); }

size_t int8_workspace(int64_t M, int64_t K) {
  return int8_scale_bytes(M) + static_cast<size_t>(M) * static_cast<size_t>(round_up(K, 16));
}

int int8_validate(const Int8Problem& p) {
  if (!float_dtype(p.dtype)) return fail(DX_ERR_INVALID_ARGUMENT, "unknown dtype %d", p.dtype);
  if (p.x_dtype != DX_DTYPE_I8 && !float_dtype(p.x_dtype))
    return fail(DX_ERR_INVALID_ARGUMENT, "unknown x_dtype %d", p.x_dtype);
  if (p.act < DX_ACT_NONE || p.act > DX_ACT_SILU)
    return fail(DX_ERR_INVALID_ARGUMENT, "unknown activation %d", p.act);
  if (p.kernel != DX_KERNEL_AUTO && p.kernel != DX_KERNEL_UMMA && p.kernel != DX_KERNEL_DECODE)
    return fail(DX_ERR_INVALID_ARGUMENT, "unknown kernel variant %d", p.kernel);
  if (p.M < 0 || p.N < 0 || p.K < 1)
    return fail(DX_ERR_INVALID_ARGUMENT, "shape M=%lld N=%lld K=%lld: M, N >= 0 and K >= 1",
                (long long)p.M, (long long)p.N, (long long)p.K);
  if (p.K > kInt8MaxK)
    return fail(DX_ERR_UNSUPPORTED, "K=%lld above %lld, where a 32-bit sum may overflow",
                (long long)p.K, (long long)kInt8MaxK);
  if (p.M > (int64_t(1) << 22) || p.N > (int64_t(1) << 24))
    return fail(DX_ERR_UNSUPPORTED, "M above 2^22 or N above 2^24");
  if (p.M == 0 || p.N == 0) return DX_OK;
  if (p.Y == nullptr) return fail(DX_ERR_INVALID_ARGUMENT, "Y is NULL");
  if (p.X == nullptr || p.W == nullptr || p.w_scale == nullptr ||
      (p.x_dtype == DX_DTYPE_I8 && p.x_scale == nullptr))
    return fail(DX_ERR_INVALID_ARGUMENT, "X, W or a scale is NULL");
  if (p.gated && (p.W2 == nullptr || p.w2_scale == nullptr))
    return fail(DX_ERR_INVALID_ARGUMENT, "Wu or its scale is NULL");
  if (p.ldx < p.K)
    return fail(DX_ERR_INVALID_ARGUMENT, "ldx=%lld < K=%lld", (long long)p.ldx, (long long)p.K);
  if (p.ldw < p.K || (p.gated && p.ldw2 < p.K))
    return fail(DX_ERR_INVALID_ARGUMENT, "a weight's pitch is below K=%lld (weights are [N, K])",
                (long long)p.K);
  if (p.ldy < p.N)
    return fail(DX_ERR_INVALID_ARGUMENT, "ldy=%lld < N=%lld", (long long)p.ldy, (long long)p.N);
  if (p.R != nullptr && p.ldr < p.N)
    return fail(DX_ERR_INVALID_ARGUMENT, "ldr=%lld < N=%lld", (long long)p.ldr, (long long)p.N);
  if (!aligned16(p.W) || p.ldw % 16 != 0 || (p.gated && (!aligned16(p.W2) || p.ldw2 % 16 != 0)) ||
      (p.x_dtype == DX_DTYPE_I8 && (!aligned16(p.X) || p.ldx % 16 != 0)))
    return fail(DX_ERR_UNSUPPORTED,
                "8-bit operands need 16-byte-aligned pointers and pitches that are multiples of 16");
  if (!element_aligned(4, p.x_scale, p.w_scale, p.w2_scale) ||
      !element_aligned(elem_size(p.dtype), p.bias, p.bias2, p.R, p.Y) ||
      (p.x_dtype != DX_DTYPE_I8 && !element_aligned(elem_size(p.x_dtype), p.X)))
    return fail(DX_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its elements");
  return DX_OK;
}

// Whether the pair kernel can store Y (and read R) by TMA.
bool int8_tma_out(const Int8Problem& p) {
  return p.dtype != DX_DTYPE_F32 && tma_ok(p.Y, p.ldy) && (p.R == nullptr || tma_ok(p.R, p.ldr));
}

struct Int8Plan {
  bool pair = false;
  int bn = 256;               // pair
  bool halves = false;        // pair: the last wave's tiles as two halves each
  int workers = 0;            // pair
  int nr = 128, mn = 16, cluster = 1, stages = 3;  // tile
};

// Tile kernel: tokens and channels per tile, CTAs per cluster and ring depth (B200;
// us, W in L2 unless it says otherwise).  Two CTAs fit an SM, so a wave is 2 * SMs tiles.
//   tokens: the smallest of 16 / 32 / 64 / 128 whose tiles make one wave, then
//   evened out.  M = 64, N = 4096: 10.0 with 32 a tile against 11.6 with 64;
//   M = 512: 17.2 with 64, 19.3 with 128; M = 1024: 24.9 with 128 against 33.5
//   with 64, which make two waves.
//   With several token tiles, clusters of 4 or more that leave an eighth of the wave
//   free, or none: M = 80, K = N = 4096 11.6 with none, 15.1 with 3 CTAs; N = 3000,
//   M = 96 14.8 with 4 CTAs in 97% of the wave, M = 128 11.5 with none.
//   cluster: as many CTAs as fill a wave, up to 6, with some six K blocks each where
//   there are that many; none where the tiles alone keep two thirds of the SMs busy.
//   M = 1, weights from HBM: K = N = 4096 6.6-6.9 us for C = 4 to 8, 7.0-7.5 for 3
//   (11.6 for 1, in L2); K = 14336 13.5 for 5 and 6, 13.9 for 8, 14.4 for 3;
//   K = N = 8192 14.7 for 3, 15.0 for 2, 18.3 for 1; N = 14336 12.9 for 1, 14.0 for 2.
//   ring: all of the SM's shared memory when each CTA has an SM to itself.
//   channels: 128, or fewer where that evens out one or two CTAs an SM
//   (16 x 8192 x 28672: 40.2 us with 104 a tile, 41.5 with 128).
Int8Plan int8_tile_plan(const Int8Problem& p, int sms) {
  using S = Int8TileShape;
  Int8Plan pl;
  pl.nr = p.gated ? 64 : 128;
  int64_t n_tiles = (p.N + pl.nr - 1) / pl.nr;
  int64_t mn = 16;
  while (mn < S::MAX_MN && mn < p.M &&
         ((p.M + mn - 1) / mn > 1 && (mn < 32 || n_tiles * ((p.M + mn - 1) / mn) > 2 * sms)))
    mn *= 2;
  const int64_t m_tiles = (p.M + mn - 1) / mn;
  pl.mn = static_cast<int>(round_up((p.M + m_tiles - 1) / m_tiles, 16));
  int64_t tiles = n_tiles * m_tiles;
  const int64_t k_blocks = (p.K + 127) / 128;
  const int64_t most = std::min<int64_t>(
      std::min<int64_t>(6, (m_tiles > 1 ? 7 * sms / 4 : 2 * sms) / tiles),
      std::min<int64_t>(std::max<int64_t>(4, k_blocks / 6), k_blocks / 2));
  if (3 * tiles < 2 * sms && most >= (m_tiles > 1 ? 4 : 2)) pl.cluster = static_cast<int>(most);
  if (pl.cluster == 1 && tiles > sms && tiles <= 2 * sms) {
    // One or two CTAs an SM: the channels per tile that leave the busiest SM least.
    int64_t best = 2 * pl.nr;
    for (int nr = pl.nr - 8; nr >= pl.nr / 2; nr -= 8) {
      const int64_t t = (p.N + nr - 1) / nr * m_tiles;
      if (t > 2 * sms) break;
      if (2 * nr < best) {
        best = 2 * nr;
        pl.nr = nr;
        tiles = t;
      }
    }
  }
  const int room = tiles * pl.cluster <= sms ? S::FULL_SM : S::HALF_SM;
  pl.stages = std::min<int>(S::MAX_STAGES, (room - S::smem_bytes(pl.mn, 0)) / S::stage_bytes(pl.mn));
  return pl;
}

template <typename T, bool G>
int launch_int8_tile(const Int8Problem& pr, int dev, const Int8Plan& pl) {
  using S = Int8TileShape;
  auto kern = dx::int8_tile_kernel<T, G>;
  int rc = ensure_smem_attr(dev, reinterpret_cast<const void*>(kern), S::FULL_SM, true);
  if (rc) return rc;
  const int NT = pl.nr;
  CUtensorMap tW, tW2, tX;
  if ((rc = make_tmap_i8(&tW, pr.W, pr.K, pr.N, pr.ldw, NT, "W"))) return rc;
  if (G) {
    if ((rc = make_tmap_i8(&tW2, pr.W2, pr.K, pr.N, pr.ldw2, NT, "W2"))) return rc;
  } else {
    tW2 = tW;  // never read
  }
  if ((rc = make_tmap_i8(&tX, pr.X, pr.K, pr.M, pr.ldx, static_cast<uint32_t>(pl.mn), "X"))) return rc;
  Int8Params p{};
  p.M = static_cast<int>(pr.M);
  p.N = static_cast<int>(pr.N);
  p.k_blocks = static_cast<int>((pr.K + 127) / 128);
  p.ldy = pr.ldy;
  p.ldr = pr.ldr;
  p.sx = pr.x_scale;
  p.sw = pr.w_scale;
  p.sw2 = pr.w2_scale;
  p.bias = pr.bias;
  p.bias2 = pr.bias2;
  p.residual = pr.R;
  p.Y = pr.Y;
  p.act = pr.act;
  p.nr = pl.nr;
  p.mn = pl.mn;
  p.stages = pl.stages;
  p.cluster = pl.cluster;
  p.w_early = pr.w_early ? 1 : 0;
  const int n_tiles = static_cast<int>((pr.N + NT - 1) / NT);
  const int m_tiles = static_cast<int>((pr.M + pl.mn - 1) / pl.mn);
  set_plan_ints(G ? "int8_tile_gated tile=%dx%d stages=%d grid=%dx%d cluster=%d early=%d smem=%d"
                  : "int8_tile tile=%dx%d stages=%d grid=%dx%d cluster=%d early=%d smem=%d",
                NT, pl.mn, pl.stages, n_tiles * pl.cluster, m_tiles, pl.cluster, p.w_early,
                S::smem_bytes(pl.mn, pl.stages));
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = launch_config(n_tiles * pl.cluster, S::THREADS,
                                         S::smem_bytes(pl.mn, pl.stages), pr.stream, pl.cluster,
                                         attr);
  cfg.gridDim.y = static_cast<unsigned>(m_tiles);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tW, tW2, tX, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch int8_tile_kernel");
  return DX_OK;
}

template <typename T, bool G>
int launch_int8_pair(const Int8Problem& pr, int dev, const Int8Plan& pl) {
  using S = Int8PairShape;
  auto kern = dx::int8_pair_kernel<T, G>;
  int rc = ensure_smem_attr(dev, reinterpret_cast<const void*>(kern), S::SMEM_BYTES, false);
  if (rc) return rc;
  CUtensorMap tA, tB, tB2, tY, tR;
  if ((rc = make_tmap_i8(&tA, pr.X, pr.K, pr.M, pr.ldx, 128, "X"))) return rc;
  if ((rc = make_tmap_i8(&tB, pr.W, pr.K, pr.N, pr.ldw, static_cast<uint32_t>(pl.bn / 4), "W"))) return rc;
  if (G) {
    if ((rc = make_tmap_i8(&tB2, pr.W2, pr.K, pr.N, pr.ldw2, static_cast<uint32_t>(pl.bn / 4), "W2"))) return rc;
  } else {
    tB2 = tB;  // never read
  }
  const CUtensorMapDataType dt = tma_dtype(pr.dtype);
  const bool tma_out = int8_tma_out(pr);
  if (!tma_out) {
    tY = tA;  // never read
  } else if ((rc = make_tmap_2d(&tY, pr.Y, dt, pr.N, pr.M, pr.ldy, 32, 32,
                                CU_TENSOR_MAP_SWIZZLE_64B, "Y"))) {
    return rc;
  }
  if (tma_out && pr.R != nullptr) {
    if ((rc = make_tmap_2d(&tR, pr.R, dt, pr.N, pr.M, pr.ldr, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B,
                           "R")))
      return rc;
  } else {
    tR = tY;  // never read
  }
  const int NT = G ? pl.bn / 2 : pl.bn;
  Int8Params p{};
  p.bn = pl.bn;
  p.stages = std::min(S::MAX_STAGES, S::RING_BYTES / (S::A_BYTES + pl.bn / 2 * S::BK));
  p.M = static_cast<int>(pr.M);
  p.N = static_cast<int>(pr.N);
  p.k_blocks = static_cast<int>((pr.K + 127) / 128);
  p.sx = pr.x_scale;
  p.sw = pr.w_scale;
  p.sw2 = pr.w2_scale;
  p.bias = pr.bias;
  p.bias2 = pr.bias2;
  p.act = pr.act;
  p.tma_out = tma_out ? 1 : 0;
  p.has_residual = tma_out && pr.R != nullptr ? 1 : 0;
  p.residual = pr.R;
  p.ldr = pr.ldr;
  p.Y = pr.Y;
  p.ldy = pr.ldy;
  p.m_tiles = static_cast<int>((pr.M + 255) / 256);
  p.n_tiles = static_cast<int>((pr.N + NT - 1) / NT);
  const int tiles = p.m_tiles * p.n_tiles;
  p.full_tiles = pl.halves ? tiles / pl.workers * pl.workers : tiles;
  p.num_work = p.full_tiles + 2 * (tiles - p.full_tiles);
  p.group_m = pick_group_m(p.m_tiles, 256, (pr.K + 1) / 2);
  p.workers = std::min(pl.workers, p.num_work);
  set_plan_ints(
      G ? "int8_pair_gated tile=256x%d tma_out=%d stages=%d grid=%d tiles=%d full=%d group_m=%d smem=%d"
        : "int8_pair tile=256x%d tma_out=%d stages=%d grid=%d tiles=%d full=%d group_m=%d smem=%d",
      NT, p.tma_out, p.stages, 2 * p.workers, tiles, p.full_tiles, p.group_m, S::SMEM_BYTES);
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg =
      launch_config(2 * p.workers, S::THREADS, S::SMEM_BYTES, pr.stream, 2, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tA, tB, tB2, tY, tR, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch int8_pair_kernel");
  return DX_OK;
}

template <bool G>
int dispatch_int8(const Int8Problem& p, int dev, const Int8Plan& pl) {
  if (pl.pair) {
    if (p.dtype == DX_DTYPE_F32) return launch_int8_pair<float, G>(p, dev, pl);
    return p.dtype == DX_DTYPE_F16 ? launch_int8_pair<__half, G>(p, dev, pl)
                                   : launch_int8_pair<__nv_bfloat16, G>(p, dev, pl);
  }
  if (p.dtype == DX_DTYPE_F32) return launch_int8_tile<float, G>(p, dev, pl);
  return p.dtype == DX_DTYPE_F16 ? launch_int8_tile<__half, G>(p, dev, pl)
                                 : launch_int8_tile<__nv_bfloat16, G>(p, dev, pl);
}

// Accumulator columns of the pair kernel's tiles.  A wave of tiles takes about
// max(bn + 134, 268) (a narrow tile is bound by its X rows: K = 4096, sustained,
// us a wave: 8.0 at 128, 8.8 at 160, 9.6 at 192, 10.7 at 224, 11.6 at 256), and
// the last tile's epilogue, about bn, is not overlapped.  M = N = K = 4096: 45 us
// at 256 (4 waves), 47 at 192 (5), 56 at 128 (7); M = 512: 12.4 at 128, 15.4 at
// 256, 18.1 at 64 (2 waves); M = 3000, N = 5000: 43.5 at 224, 46 at 256.
// Where the tiles of the last wave fill at most half the pairs, they are done as
// two halves of bn / 2 columns each: 3.7 waves' time instead of 4 for M = N = 4096.
void int8_pair_tiles(const Int8Problem& p, int workers, Int8Plan* pl) {
  const int step = p.gated ? 64 : 32, wide = p.gated ? 2 : 1;
  const int64_t m_tiles = (p.M + 255) / 256;
  auto wave = [](int bn) { return std::max(bn + 134, 268); };
  int64_t best = -1;
  for (int bn = 256; bn >= 64; bn -= step) {
    const int64_t tiles = m_tiles * ((wide * p.N + bn - 1) / bn);
    const int64_t waves = tiles / workers, rest = tiles % workers;
    int64_t cost = waves * wave(bn) + bn;
    const bool halves = bn % (2 * step) == 0 && rest > 0 && 2 * rest <= workers &&
                        waves > 0 && wave(bn / 2) < wave(bn);
    if (rest > 0) cost += halves ? wave(bn / 2) - bn / 2 : wave(bn);
    if (best < 0 || cost < best) {
      best = cost;
      pl->bn = bn;
      pl->halves = halves;
    }
  }
}

// Pairs from 129 tokens on, gated from 65 (us, W from HBM, tile kernel against pairs).
// M = 128: K = N = 4096 11.8 and 13.2; K x N = 14336 x 4096 29.4 and 32.8; 8192 x 28672
// 49.3 and 53.8; 4096 x 14336 19.6 and 18.3.  M = 96: 4096 x 14336 17.4 and 18.3.
// M = 256, K = N = 4096, W in L2: 13.8 and 11.2.  Gated, M = 64: 4096 x 14336 28.8 and
// 32.4; 2056 x 5464 16.6 and 15.1; M = 128: 37.2 and 31.3, 22.0 and 15.2.
Int8Plan int8_plan(const Int8Problem& p, int dev, int sms) {
  Int8Plan pl = int8_tile_plan(p, sms);
  if (p.kernel == DX_KERNEL_DECODE || (p.kernel == DX_KERNEL_AUTO && p.M <= (p.gated ? 64 : 128))) return pl;
  const int slots = std::min(pair_slots<256, __nv_bfloat16>(dev, sms), sms / 2);
  if (slots < 1) return pl;
  pl.pair = true;
  pl.workers = slots;
  int8_pair_tiles(p, slots, &pl);
  return pl;
}

int run_int8(Int8Problem& p) {
  t_last_error.clear();
  int rc = int8_validate(p);
  if (rc) return rc;
  if (p.M == 0 || p.N == 0) return DX_OK;
  if (p.x_dtype != DX_DTYPE_I8) {
    const size_t need = int8_workspace(p.M, p.K);
    if (p.ws == nullptr || p.ws_bytes < need || !aligned16(p.ws))
      return fail(DX_ERR_WORKSPACE, "a %s X needs a 16-byte-aligned workspace of %zu bytes",
                  "floating-point", need);
  }
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  int sms = 0;
  if ((rc = stream_sms(p.stream, dev, &sms))) return rc;
  if ((rc = install_status_mirror(dev, p.stream))) return rc;
  if ((rc = check_status_mirror(dev))) return rc;
  if (!load_encode_fn())
    return fail(DX_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  if (p.x_dtype != DX_DTYPE_I8) {
    float* const scale = static_cast<float*>(p.ws);
    void* const q = static_cast<char*>(p.ws) + int8_scale_bytes(p.M);
    const int64_t ldq = round_up(p.K, 16);
    if ((rc = run_quantize(p.X, q, scale, p.M, p.K, p.ldx, ldq, p.x_dtype, sms, p.stream)))
      return rc;
    p.X = q;
    p.x_scale = scale;
    p.ldx = ldq;
    // The launch before the product is the quantisation, which itself waited
    // for everything before it and writes nothing but q and scale.
    p.w_early = true;
  }
  const Int8Plan pl = int8_plan(p, dev, sms);
  return p.gated ? dispatch_int8<true>(p, dev, pl) : dispatch_int8<false>(p, dev, pl);
}

}  // namespace

extern "C" {

int dx_quantize_rows(const void* X, void* Q, float* scale, int64_t M, int64_t K, int64_t ldx,
                     int64_t ldq, int dtype, void* stream) {
  t_last_error.clear();
  if (!float_dtype(dtype)) return fail(DX_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
  if (M < 0 || K < 0)
    return fail(DX_ERR_INVALID_ARGUMENT, "negative shape M=%lld K=%lld", (long long)M, (long long)K);
  if (M > 0x7fffffffLL || K > 0x3fffffffLL)
    return fail(DX_ERR_UNSUPPORTED, "M above 2^31-1 or K above 2^30-1");
  if (M == 0) return DX_OK;
  if (scale == nullptr || (K > 0 && (X == nullptr || Q == nullptr)))
    return fail(DX_ERR_INVALID_ARGUMENT, "X, Q or scale is NULL");
  if (ldx < K || ldq < K)
    return fail(DX_ERR_INVALID_ARGUMENT, "ldx=%lld or ldq=%lld below K=%lld", (long long)ldx,
                (long long)ldq, (long long)K);
  if (!element_aligned(elem_size(dtype), X) || !element_aligned(4, scale))
    return fail(DX_ERR_INVALID_ARGUMENT, "X or scale is not aligned to its elements");
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  int sms = 0;
  int rc = device_sms(dev, &sms);
  if (rc) return rc;
  return run_quantize(X, Q, scale, M, K, ldx, ldq, dtype, sms, static_cast<cudaStream_t>(stream));
}

int dx_pack_int8_rows(const void* src, void* dst, int64_t rows, int64_t K, int64_t ld_src,
                      int64_t ld_dst, void* stream) {
  t_last_error.clear();
  if (rows < 0 || K < 0)
    return fail(DX_ERR_INVALID_ARGUMENT, "negative shape rows=%lld K=%lld", (long long)rows,
                (long long)K);
  if (rows > 0x7fffffffLL || K > 0x3fffffffLL)
    return fail(DX_ERR_UNSUPPORTED, "rows above 2^31-1 or K above 2^30-1");
  if (rows == 0 || K == 0) return DX_OK;
  if (src == nullptr || dst == nullptr)
    return fail(DX_ERR_INVALID_ARGUMENT, "src or dst is NULL");
  if (ld_src < K || ld_dst < round_up(K, 16))
    return fail(DX_ERR_INVALID_ARGUMENT, "ld_src=%lld or ld_dst=%lld too small for K=%lld",
                (long long)ld_src, (long long)ld_dst, (long long)K);
  if (!aligned16(dst) || ld_dst % 16 != 0)
    return fail(DX_ERR_INVALID_ARGUMENT, "dst needs a 16-byte-aligned pointer and pitch");
  dx::PackParams p{};
  p.src = static_cast<const uint8_t*>(src);
  p.dst = static_cast<uint8_t*>(dst);
  p.rows = static_cast<int>(rows);
  p.K = static_cast<int>(K);
  p.chunks = static_cast<int>((K + 15) / 16);
  p.rows_per_cta = std::max(1, dx::kPackThreads * dx::kPackBatch / p.chunks);
  p.ld_src = ld_src;
  p.ld_dst = ld_dst;
  const int grid = static_cast<int>((rows + p.rows_per_cta - 1) / p.rows_per_cta);
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = launch_config(grid, dx::kPackThreads, 0,
                                         static_cast<cudaStream_t>(stream), 1, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, dx::pack_rows_kernel, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch pack_rows_kernel");
  return DX_OK;
}

size_t dx_int8_workspace_size(int64_t M, int64_t K) {
  if (M <= 0 || K <= 0 || K > kInt8MaxK || M > (int64_t(1) << 22)) return 0;
  return int8_workspace(M, K);
}

int dx_int8_linear(const void* X, int x_dtype, const float* x_scale, const void* W,
                   const float* w_scale, const void* bias, const void* R, void* Y, int64_t M,
                   int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t ldr, int64_t ldy,
                   int dtype, int act, int kernel, void* workspace, size_t workspace_bytes,
                   void* stream) {
  Int8Problem p{X,       x_dtype, x_scale, W,   nullptr, w_scale, nullptr, bias, nullptr, R,
                Y,       M,       N,       K,   ldx,     ldw,     0,       ldr,  ldy,     dtype,
                act,     kernel,  false,   workspace, workspace_bytes,
                static_cast<cudaStream_t>(stream)};
  return run_int8(p);
}

int dx_int8_gated_linear(const void* X, int x_dtype, const float* x_scale, const void* Wg,
                         const float* wg_scale, const void* Wu, const float* wu_scale,
                         const void* bias_g, const void* bias_u, void* Y, int64_t M, int64_t N,
                         int64_t K, int64_t ldx, int64_t ldwg, int64_t ldwu, int64_t ldy, int dtype,
                         int act, int kernel, void* workspace, size_t workspace_bytes,
                         void* stream) {
  Int8Problem p{X,       x_dtype, x_scale, Wg,  Wu,      wg_scale, wu_scale, bias_g, bias_u, nullptr,
                Y,       M,       N,       K,   ldx,     ldwg,     ldwu,     0,      ldy,    dtype,
                act,     kernel,  true,    workspace, workspace_bytes,
                static_cast<cudaStream_t>(stream)};
  return run_int8(p);
}

}  // extern "C"
