// fp8.h — e4m3 blocks of 128 with an e8m0 scale, as the kernels that write them form them, and
// rows of fp32 or bf16 read 8 elements at a time.
#pragma once

#include "common.h"

namespace nl {

constexpr int kB = 128;  // elements per scale

// |x| as ordered bits, and with 0 for a value that is not finite (it has no part in the scale).
constexpr uint32_t kInfBits = 0x7f800000u;
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t finite_abs_bits(float x) {
  const uint32_t u = abs_bits(x);
  return u < kInfBits ? u : 0u;
}

// The e8m0 byte (e + 127) of a block whose largest |x| has these bits: with |x| =
// 1.f * 2^(E-127), 448 = 1.75 * 2^8 gives e = E - 135, one more above 1.75.
// Blocks below 2^-119 stay at 2^-127, a block of zeros is at 1.
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  const int b = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return amax == 0 ? 127 : (b > 0 ? b : 0);
}

// Four values divided by 2^(byte - 127) to four e4m3 bytes (an infinity or a NaN gives NaN). The
// conversion reads the scale from a float's exponent, 0 being 2^-127 (the same bytes as x * 2^-e
// converted, for every byte up to 253 and subnormal x), and rounds once.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d, int byte) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  const float scale = __uint_as_float((uint32_t)byte << 23);
  s16x2 r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, scale, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, scale, true);
  return __builtin_bit_cast(uint32_t, r);
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
// max over the 16 lanes of a row of lanes (the exchanges of wave_sum in common.h)
__device__ __forceinline__ uint32_t max16(uint32_t v) {
  v = max(v, dpp_u<0xB1>(v));
  v = max(v, dpp_u<0x4E>(v));
  v = max(v, dpp_u<0x141>(v));
  return max(v, dpp_u<0x140>(v));
}

typedef u32x4 __attribute__((aligned(2))) u32x4_any;  // 16 bytes at any address of an element
typedef f32x4 __attribute__((aligned(4))) f32x4_any;

// 8 elements as they are stored
template <typename T>
struct Vec {
  u32x4 v[sizeof(T) / 2];
};

// elements p[0 .. n-1] of up to 8, zero behind them
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p, int n) {
  Vec<T> o;
  constexpr int kParts = sizeof(T) / 2;
  if (n >= 8) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) o.v[i] = reinterpret_cast<const u32x4_any*>(p)[i];
    return o;
  }
#pragma unroll
  for (int i = 0; i < kParts; ++i) o.v[i] = u32x4{0u, 0u, 0u, 0u};
  if (n > 0) {
#pragma unroll
    for (int k = 0; k < 7; ++k) {
      if (k >= n) continue;
      if constexpr (sizeof(T) == 2) o.v[0][k >> 1] |= (uint32_t)p[k] << (16 * (k & 1));
      else o.v[k >> 2][k & 3] = __float_as_uint(p[k]);
    }
  }
  return o;
}

template <typename T>
__device__ __forceinline__ void unpack(const Vec<T>& o, float f[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (sizeof(T) == 2) f[k] = k & 1 ? bf16_hi(o.v[0][k >> 1]) : bf16_lo(o.v[0][k >> 1]);
    else f[k] = __uint_as_float(o.v[k >> 2][k & 3]);
  }
}

// The same of a row, `n` elements of which are the row's (0 or less: none). `over`: what lies behind
// the row may be read (the next row, of 8 elements at least): one load then, and what is not the
// row's is cleared by clear_tail. Element by element a row's last vector waits for each: the norm of
// 100,663 rows of 333 bf16 took 99 us with the residual for 58, its gradients 162 for 57.
template <typename T>
__device__ __forceinline__ Vec<T> load_row(const T* p, int n, bool over) {
  return load_vec(p, over && n > 0 ? 8 : n);
}
__device__ __forceinline__ void clear_tail(float (&f)[8], int n) {
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = k < n ? f[k] : 0.f;
}

}  // namespace nl
