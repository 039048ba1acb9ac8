// dx_quant.cuh — symmetric 8-bit quantisation of matrix rows:
//   a_m = max(max_k |x_mk|, 2^-100),  s_m = a_m / 127,
//   q_mk = the integer nearest 127 x_mk / a_m, halves to even,
// so x_mk is close to q_mk * s_m.  A row that holds an infinity or a NaN gets
// the scale NaN (and q = 0), which makes every product with it NaN.
//
// Bound by memory: a row is read once into registers (rows of more than
// kQuantRegs vectors a thread are read twice, the second time from L2), its
// largest magnitude found on the integer bit patterns (ordered as the
// magnitudes are, and a NaN stays the largest), and one byte a value written.
//
// The rounding is exact.  v = x * (127 / a) in fp32 is off by at most
// 127 * 1.5 * 2^-23 < 3e-5, so the nearest integer of v is the right one
// unless v lies within that of a half; those few values (|v - rint(v)| above
// 0.4999) are rounded from the quotient in 64 bits, where 127 x is exact and a
// quotient that is not a half differs from one by more than 2^-35.
// Rows of 2^100 and more are scaled by 2^-64 first (exact) so that nothing
// overflows.
#pragma once

#include "dx_epilogue.cuh"
#include "dx_ptx.cuh"

namespace dx {

constexpr int kQuantVec = 8;   // values a vector: one 16-byte load of a 16-bit type
constexpr int kQuantRegs = 4;  // vectors of a row that a thread keeps in registers

struct QuantParams {
  const void* X;
  int8_t* Q;
  float* scale;
  int M, K;
  long long ldx, ldq;
  int vec;  // X, Q and their pitches allow vector accesses
};

// One vector of 8 values as it lies in memory: 4 words of a 16-bit type, 8 of fp32.
template <typename T>
struct QuantVec {
  static constexpr int kWords = kQuantVec * sizeof(T) / 4;
  uint32_t w[kWords];
};

// The vector at x, `n` values of it (zeros behind them).
template <typename T>
__device__ __forceinline__ QuantVec<T> quant_load(const T* x, int n, bool vec) {
  QuantVec<T> v;
  if (vec && n >= kQuantVec) {
#pragma unroll
    for (int i = 0; i < QuantVec<T>::kWords; i += 4) {
      const uint4 u = reinterpret_cast<const uint4*>(x)[i / 4];
      v.w[i] = u.x, v.w[i + 1] = u.y, v.w[i + 2] = u.z, v.w[i + 3] = u.w;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < kQuantVec; ++i) v.w[i] = i < n ? __float_as_uint(x[i]) : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < kQuantVec / 2; ++i) {
      const uint16_t* const u = reinterpret_cast<const uint16_t*>(x);
      const uint32_t lo = 2 * i < n ? u[2 * i] : 0u, hi = 2 * i + 1 < n ? u[2 * i + 1] : 0u;
      v.w[i] = lo | (hi << 16);
    }
  }
  return v;
}

template <typename T>
__device__ __forceinline__ void quant_floats(const QuantVec<T>& v, float (&f)[kQuantVec]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < kQuantVec; ++i) f[i] = __uint_as_float(v.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kQuantVec / 2; ++i) {
      const float2 p = ElemTraits<T>::unpack2(v.w[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}

template <typename T>
__device__ __forceinline__ uint32_t quant_max(uint32_t m, const QuantVec<T>& v) {
  float f[kQuantVec];
  quant_floats(v, f);
#pragma unroll
  for (int i = 0; i < kQuantVec; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m;
}

// The nearest integer of 127 x / a; c = 127 / a in fp32.
__device__ __forceinline__ int quant_one(float x, float a, float c) {
  const float v = x * c;
  // Adding 1.5 * 2^23 leaves the nearest integer in the low mantissa bits.
  const float t = v + 12582912.0f;
  int q = static_cast<int>(__float_as_uint(t)) - 0x4b400000;
  if (fabsf(v - (t - 12582912.0f)) > 0.4999f)
    q = static_cast<int>(rint(127.0 * static_cast<double>(x) / static_cast<double>(a)));
  return q;
}

template <typename T>
__device__ __forceinline__ void quant_store(int8_t* q, int n, bool vec, const QuantVec<T>& x,
                                            float pre, float a, float c) {
  float f[kQuantVec];
  quant_floats(x, f);
  uint32_t b[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < kQuantVec; ++i) {
    const uint32_t v = static_cast<uint32_t>(quant_one(f[i] * pre, a, c)) & 0xffu;
    b[i >> 2] |= v << (8 * (i & 3));
  }
  if (c == 0.0f) b[0] = b[1] = 0u;  // a row with an infinity or a NaN
  if (vec && n >= kQuantVec) {
    *reinterpret_cast<uint2*>(q) = make_uint2(b[0], b[1]);
  } else {
#pragma unroll
    for (int i = 0; i < kQuantVec; ++i)
      if (i < n) q[i] = static_cast<int8_t>(b[i >> 2] >> (8 * (i & 3)));
  }
}

// One row per CTA.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) quantize_rows_kernel(const QuantParams p) {
  constexpr int kWarps = THREADS / 32;
  __shared__ uint32_t s_max[kWarps];
  grid_dependency_wait();
  grid_launch_dependents();
  const long long row = blockIdx.x;
  const T* const x = static_cast<const T*>(p.X) + row * p.ldx;
  int8_t* const q = p.Q + row * p.ldq;
  const int vectors = (p.K + kQuantVec - 1) / kQuantVec;
  const bool vec = p.vec != 0;

  QuantVec<T> f[kQuantRegs];
  uint32_t m = 0;
#pragma unroll
  for (int r = 0; r < kQuantRegs; ++r) {
    const int i = r * THREADS + static_cast<int>(threadIdx.x);
    if (i < vectors) {
      f[r] = quant_load(x + static_cast<long long>(i) * kQuantVec, p.K - i * kQuantVec, vec);
      m = quant_max(m, f[r]);
    }
  }
  for (int i = kQuantRegs * THREADS + static_cast<int>(threadIdx.x); i < vectors; i += THREADS)
    m = quant_max(m, quant_load(x + static_cast<long long>(i) * kQuantVec, p.K - i * kQuantVec, vec));
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();
  m = s_max[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) m = max(m, s_max[w]);

  const bool finite = m < 0x7f800000u;
  const float top = fmaxf(__uint_as_float(finite ? m : 0u), 0x1p-100f);
  if (threadIdx.x == 0)
    p.scale[row] = finite ? __fdiv_rn(top, 127.0f) : __uint_as_float(0x7fc00000u);
  const float pre = top >= 0x1p100f ? 0x1p-64f : 1.0f;
  const float a = top * pre;
  const float c = finite ? __fdiv_rn(127.0f, a) : 0.0f;
#pragma unroll
  for (int r = 0; r < kQuantRegs; ++r) {
    const int i = r * THREADS + static_cast<int>(threadIdx.x);
    if (i < vectors)
      quant_store(q + static_cast<long long>(i) * kQuantVec, p.K - i * kQuantVec, vec, f[r], pre, a,
                  c);
  }
  for (int i = kQuantRegs * THREADS + static_cast<int>(threadIdx.x); i < vectors; i += THREADS)
    quant_store(q + static_cast<long long>(i) * kQuantVec, p.K - i * kQuantVec, vec,
                quant_load(x + static_cast<long long>(i) * kQuantVec, p.K - i * kQuantVec, vec), pre,
                a, c);
}

}  // namespace dx
