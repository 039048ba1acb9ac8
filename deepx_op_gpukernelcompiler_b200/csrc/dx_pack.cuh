// dx_pack.cuh — rows of bytes at any pitch and alignment into rows that start on
// 16 bytes, which TMA asks of the 8-bit operands.
//
// Bound by memory: every byte is read once and written once.  A thread moves 16
// bytes: the two aligned vectors around its source, shifted together in registers.
// A source vector is read whole only where it lies inside the matrix (from its first
// to its last byte, gaps between rows included); the few at its ends go byte by byte.
// 28672 x 8191: 75 us, 6.2 TB/s of bytes read and written; 5464 x 2056: 5.3 us; 2049 x
// 1000: 2.4 us.
#pragma once

#include "dx_ptx.cuh"

namespace dx {

struct PackParams {
  const uint8_t* src;
  uint8_t* dst;
  int rows, K;
  int chunks;        // 16-byte pieces of a row of dst
  int rows_per_cta;
  long long ld_src, ld_dst;
};

constexpr int kPackThreads = 256;
constexpr int kPackBatch = 4;  // pieces a thread has in flight

__global__ void __launch_bounds__(kPackThreads) pack_rows_kernel(const PackParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const uint8_t* const begin = p.src;
  const uint8_t* const end = p.src + (p.rows - 1) * p.ld_src + p.K;
  const long long row0 = static_cast<long long>(blockIdx.x) * p.rows_per_cta;
  const int rows = static_cast<int>(min(static_cast<long long>(p.rows_per_cta), p.rows - row0));
  const int pieces = rows * p.chunks;
  for (int i0 = static_cast<int>(threadIdx.x); i0 < pieces; i0 += kPackThreads * kPackBatch) {
    const uint8_t* from[kPackBatch];
    uint4 lo[kPackBatch], hi[kPackBatch];
    bool whole[kPackBatch];
#pragma unroll
    for (int j = 0; j < kPackBatch; ++j) {
      const int i = min(i0 + j * kPackThreads, pieces - 1);
      const int r = i / p.chunks;
      from[j] = p.src + (row0 + r) * p.ld_src + 16 * (i - r * p.chunks);
      const uintptr_t skew = reinterpret_cast<uintptr_t>(from[j]) & 15u;
      const uint8_t* const a = from[j] - skew;
      whole[j] = a >= begin && a + (skew != 0 ? 32 : 16) <= end;
      lo[j] = hi[j] = make_uint4(0u, 0u, 0u, 0u);
      if (whole[j]) {
        lo[j] = *reinterpret_cast<const uint4*>(a);
        if (skew != 0) hi[j] = *reinterpret_cast<const uint4*>(a + 16);
      }
    }
#pragma unroll
    for (int j = 0; j < kPackBatch; ++j) {
      const int i = i0 + j * kPackThreads;
      if (i >= pieces) break;
      const int r = i / p.chunks, c = i - r * p.chunks;
      uint32_t w[8] = {lo[j].x, lo[j].y, lo[j].z, lo[j].w, hi[j].x, hi[j].y, hi[j].z, hi[j].w};
      if (whole[j]) {
        const uint32_t skew = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from[j])) & 15u;
#pragma unroll
        for (int k = 0; k < 6; ++k) w[k] = (skew & 8u) != 0 ? w[k + 2] : w[k];
#pragma unroll
        for (int k = 0; k < 5; ++k) w[k] = (skew & 4u) != 0 ? w[k + 1] : w[k];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 8u * (skew & 3u));
      } else {
        const int n = min(16, p.K - 16 * c);
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (k < n) w[k >> 2] |= static_cast<uint32_t>(from[j][k]) << (8 * (k & 3));
      }
      *reinterpret_cast<uint4*>(p.dst + (row0 + r) * p.ld_dst + 16 * c) =
          make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

}  // namespace dx
