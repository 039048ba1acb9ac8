// dx_quant.cuh — symmetric 8-bit quantisation of matrix rows:
//   a_m = max(max_k |x_mk|, 2^-100),  s_m = a_m / 127,
//   q_mk = the integer nearest 127 x_mk / a_m, halves to even,
// so x_mk is close to q_mk * s_m.  A row that holds an infinity or a NaN gets
// the scale NaN (and q = 0), which makes every product with it NaN.
//
// Bound by memory: a row is read once into registers (rows of more than
// the threads' registers hold are read twice, the second time from L2), its
// largest magnitude found (a NaN counts as the largest), and one byte a value
// written.
//
// The rounding is exact.  With c = 127 / a in fp32, x c is off by 2^-23 of the
// quotient; one residual step, x c + (127 x - x c a) / a, leaves a half exactly a
// half and anything else within 2^-24.  Between 16-bit values a quotient that is
// not a half differs from one by more than 2^-20 of itself (127 x / a - (n + 1/2) =
// (254 X - (2n + 1) 2^j A) / (2^(j+1) A) with integers X, A < 2^11), so adding
// 1.5 * 2^23 rounds it as the exact quotient.  fp32 values can lie closer: those
// within 1e-4 of a half are decided by the sign of 127 x - (k + 1/2) a in 64 bits,
// where both products are exact.  127 x and a are taken times 2^-8, so that rows
// near the end of bf16's range do not overflow.  Deciding the halves of 16-bit
// rows in 64 bits too cost 21 instructions a value and 109 us for 8192 x 14336
// (bf16 rows hold many exact halves).
#pragma once

#include "dx_epilogue.cuh"
#include "dx_ptx.cuh"

namespace dx {

constexpr int kQuantVec = 8;   // values a vector: one 16-byte load of a 16-bit type
// 16-byte words of a row that a thread keeps in registers: 4 vectors of a 16-bit
// type, 2 of fp32.
constexpr int kQuantWords = 4;
template <typename T>
constexpr int kQuantRegsOf = kQuantWords * 2 / static_cast<int>(sizeof(T));

struct QuantParams {
  const void* X;
  int8_t* Q;
  float* scale;
  int M, K;
  long long ldx, ldq;
};

// One vector of 8 values as it lies in memory: 4 words of a 16-bit type, 8 of fp32.
template <typename T>
struct QuantVec {
  static constexpr int kWords = kQuantVec * sizeof(T) / 4;
  uint32_t w[kWords];
};

// Eight values: kVec: of the vector at x, else every kStride'th from x on, those
// before `n` (zeros behind them).
template <bool kVec, int kStride, typename T>
__device__ __forceinline__ QuantVec<T> quant_load(const T* x, int n) {
  QuantVec<T> v;
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < QuantVec<T>::kWords; i += 4) {
      const uint4 u = reinterpret_cast<const uint4*>(x)[i / 4];
      v.w[i] = u.x, v.w[i + 1] = u.y, v.w[i + 2] = u.z, v.w[i + 3] = u.w;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < kQuantVec; ++i) v.w[i] = i * kStride < n ? __float_as_uint(x[i * kStride]) : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < kQuantVec / 2; ++i) {
      const uint16_t* const u = reinterpret_cast<const uint16_t*>(x);
      const uint32_t lo = 2 * i * kStride < n ? u[2 * i * kStride] : 0u;
      const uint32_t hi = (2 * i + 1) * kStride < n ? u[(2 * i + 1) * kStride] : 0u;
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

// The larger of the magnitudes m (a pair of a 16-bit type, or one fp32) and w; a NaN
// is the largest.
__device__ __forceinline__ uint32_t quant_max_word(uint32_t m, uint32_t w, const __half*) {
  const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&m),
                                __habs2(*reinterpret_cast<const __half2*>(&w)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t quant_max_word(uint32_t m, uint32_t w, const __nv_bfloat16*) {
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&m),
                                       __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t quant_max_word(uint32_t m, uint32_t w, const float*) {
  return max(m, w & 0x7fffffffu);
}

template <typename T>
__device__ __forceinline__ uint32_t quant_max(uint32_t m, const QuantVec<T>& v) {
#pragma unroll
  for (int i = 0; i < QuantVec<T>::kWords; ++i)
    m = quant_max_word(m, v.w[i], static_cast<const T*>(nullptr));
  return m;
}

// A quant_max as the bit pattern of an fp32 magnitude (ordered as magnitudes are).
template <typename T>
__device__ __forceinline__ uint32_t quant_max_bits(uint32_t m) {
  if constexpr (sizeof(T) == 4) {
    return m;
  } else {
    const float2 p = ElemTraits<T>::unpack2(m);
    return max(__float_as_uint(p.x) & 0x7fffffffu, __float_as_uint(p.y) & 0x7fffffffu);
  }
}

// What turns a row's values into integers.
struct QuantRow {
  float c;      // 127 / a; 0 for a row with an infinity or a NaN
  float a;      // 2^-8 a
  float inv_a;  // 1 / (2^-8 a)
};

__device__ __forceinline__ QuantRow quant_row(float top, bool finite) {
  QuantRow r;
  r.c = finite ? __fdiv_rn(127.0f, top) : 0.0f;
  r.a = top * 0x1p-8f;
  r.inv_a = __frcp_rn(r.a);
  return r;
}

// The integers nearest to 127 x / a of eight values, stored as bytes where
// quant_load found them.
template <bool kVec, int kStride, typename T>
__device__ __forceinline__ void quant_store(int8_t* q, int n, const QuantVec<T>& x,
                                            const QuantRow& row) {
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: the integer ends up in the low bits
  float f[kQuantVec];
  quant_floats(x, f);
  uint32_t t[kQuantVec];
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < kQuantVec; ++i) {
      const float v = f[i] * row.c;
      const float rest = fmaf(-v, row.a, f[i] * (127.0f * 0x1p-8f));
      t[i] = __float_as_uint(fmaf(rest, row.inv_a, v) + kMagic);
    }
  } else {
    float off = 0.0f;
#pragma unroll
    for (int i = 0; i < kQuantVec; ++i) {
      const float r = fmaf(f[i], row.c, kMagic);
      off = fmaxf(off, fabsf(fmaf(f[i], row.c, kMagic - r)));
      t[i] = __float_as_uint(r);
    }
    if (off > 0.4999f) {
#pragma unroll
      for (int i = 0; i < kQuantVec; ++i) {
        const float k = floorf(f[i] * row.c);
        const double d = (127.0 / 256.0) * static_cast<double>(f[i]) -
                         (static_cast<double>(k) + 0.5) * static_cast<double>(row.a);
        const int q0 = static_cast<int>(k);
        t[i] = static_cast<uint32_t>(q0 + ((d > 0.0 || (d == 0.0 && (q0 & 1))) ? 1 : 0));
      }
    }
  }
  uint32_t b[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    b[i] = __byte_perm(__byte_perm(t[4 * i], t[4 * i + 1], 0x0040),
                       __byte_perm(t[4 * i + 2], t[4 * i + 3], 0x0040), 0x5410);
  if (row.c == 0.0f) b[0] = b[1] = 0u;  // a row with an infinity or a NaN
  if constexpr (kVec) {
    *reinterpret_cast<uint2*>(q) = make_uint2(b[0], b[1]);
  } else {
#pragma unroll
    for (int i = 0; i < kQuantVec; ++i)
      if (i * kStride < n) q[i * kStride] = static_cast<int8_t>(b[i >> 2] >> (8 * (i & 3)));
  }
}

// A row per CTA at a time, rows gridDim.x apart.  The next row's loads are issued
// before this row's maximum is joined, so that they are in flight through the
// barriers, the arithmetic and the stores.  kVec: every row consists of whole,
// aligned vectors, a thread taking every THREADS'th; else a thread takes every
// THREADS'th value, so that a warp's loads and stores are contiguous all the same
// (8192 x 4099 bf16: 67 us with eight neighbouring values a thread).
template <typename T, int THREADS, bool kVec>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
    quantize_rows_kernel(const QuantParams p) {
  constexpr int kWarps = THREADS / 32;
  constexpr int kRegs = kQuantRegsOf<T>;
  constexpr int kBlock = THREADS * kQuantVec;  // values of a row that one step covers
  __shared__ uint32_t s_max[2][kWarps];
  grid_dependency_wait();
  grid_launch_dependents();
  const int tid = static_cast<int>(threadIdx.x);
  const int lead = kVec ? tid * kQuantVec : tid;  // this thread's first value of a step
  const T* const X = static_cast<const T*>(p.X) + lead;
  auto load = [&](const T* x, int at) {  // x: of the row, at `lead`; at: the step's first value
    return quant_load<kVec, THREADS>(x + at, p.K - lead - at);
  };
  auto load_row = [&](long long row, QuantVec<T> (&f)[kRegs]) {
    const T* const x = X + row * p.ldx;
#pragma unroll
    for (int r = 0; r < kRegs; ++r)
      if (r * kBlock + lead < p.K) f[r] = load(x, r * kBlock);
  };
  QuantVec<T> next[kRegs];
  load_row(blockIdx.x, next);
  int half = 0;
  for (long long row = blockIdx.x; row < p.M; row += gridDim.x, half ^= 1) {
    QuantVec<T> f[kRegs];
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < kRegs; ++r) {
      f[r] = next[r];
      if (r * kBlock + lead < p.K) m = quant_max(m, f[r]);
    }
    if (row + gridDim.x < p.M) load_row(row + gridDim.x, next);
    const T* const x = X + row * p.ldx;
    int8_t* const q = p.Q + row * p.ldq + lead;
    for (int at = kRegs * kBlock; at + lead < p.K; at += kBlock) m = quant_max(m, load(x, at));
    m = __reduce_max_sync(0xffffffffu, quant_max_bits<T>(m));
    // Two arrays in turn: a warp may be a row ahead of one still reading.
    if ((tid & 31) == 0) s_max[half][tid >> 5] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, s_max[half][tid & (kWarps - 1)]);

    const bool finite = m < 0x7f800000u;
    const float top = fmaxf(__uint_as_float(finite ? m : 0u), 0x1p-100f);
    if (tid == 0)
      p.scale[row] = finite ? __fdiv_rn(top, 127.0f) : __uint_as_float(0x7fc00000u);
    const QuantRow qr = quant_row(top, finite);
#pragma unroll
    for (int r = 0; r < kRegs; ++r)
      if (r * kBlock + lead < p.K)
        quant_store<kVec, THREADS>(q + r * kBlock, p.K - lead - r * kBlock, f[r], qr);
    for (int at = kRegs * kBlock; at + lead < p.K; at += kBlock)
      quant_store<kVec, THREADS>(q + at, p.K - lead - at, load(x, at), qr);
  }
}

}  // namespace dx
