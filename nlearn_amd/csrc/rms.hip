// rms.hip — root-mean-square norm of rows, with the residual's addition folded in
// and the result in the input's type or in 8 bits with a scale for each block of
// 128 (what an 8-bit product reads), and its gradients.
//
//   s    = x (+ r, rounded to the type of x: the residual stream the next block reads)
//   rstd = 1 / sqrt(mean(s^2) + eps),   xh = s * rstd,   y = xh * gamma
//   dx   = rstd * (g - xh * mean(g * xh)) (+ ds),   g = dy * gamma
//   dgamma = sum over the rows of dy * xh
// (nlearn/model.py:228-241 normalises like this; its residual adds are
// model.py:315-324.)
//
// A row is read once and kept in registers, 8 columns a lane and vector, by 16
// lanes up to 128 columns, a wave up to 2048, 256 threads up to 8192 and 512 up to
// 16384 (1024 threads of two vectors spilled registers). Vectors are loaded and stored
// at whatever alignment the rows have (the hardware takes any multiple of the element).
// Bound by HBM where there are many rows (medians of a kernel trace over three sets of
// inputs in turn; a large copy reaches 5.1 TB/s): with the residual 16384 x 512 bf16 14.9 us
// (67 MB, 4.5 TB/s), its gradients 13.9 us (67 MB) and 3.9 us for the sum of dgamma's
// partial rows (over the same rows again, which the 256 MB cache holds, 12.0, 10.9 and 4.3);
// 16384 x 2048 bf16 to 8 bits 46 us (235 MB, 5.1 TB/s). By the chain load -> sum -> store
// where there are few: one row of 512 2.0 us, 8 rows of 2048 to 8 bits 5.0 us, 777 x 1001
// fp32 4.0 us and 5.1 + 3.3 us. A backward in
// one launch for few rows, each workgroup summing dgamma of its own columns over all rows,
// took 17 us there.
#include <type_traits>

#include "fp8.h"

namespace nl {
namespace {

constexpr int kMaxRms = 16384;    // columns
constexpr int kBwdBlocks = 1024;  // most workgroups of the backward, which leave a partial row of dgamma each

template <typename T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& o, int n) {
  if (n >= 8) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<u32x4_any*>(p)[i] = o.v[i];
    return;
  }
#pragma unroll
  for (int k = 0; k < 7; ++k) {
    if (k >= n) continue;
    if constexpr (sizeof(T) == 2) p[k] = (uint16_t)(o.v[0][k >> 1] >> (16 * (k & 1)));
    else p[k] = __uint_as_float(o.v[k >> 2][k & 3]);
  }
}

template <typename T>
__device__ __forceinline__ Vec<T> pack(const float f[8]) {
  Vec<T> o;
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    if constexpr (sizeof(T) == 2) {
      o.v[0][k >> 1] = pack_bf16x2(f[k], f[k + 1]);
    } else {
      o.v[k >> 2][k & 3] = __float_as_uint(f[k]);
      o.v[k >> 2][(k & 3) + 1] = __float_as_uint(f[k + 1]);
    }
  }
  return o;
}

// gamma[c .. c+7], zero past the last column (any alignment of a float)
__device__ __forceinline__ void load_gamma(const float* p, int n, float f[8]) {
  if (n >= 8) {
    const f32x4 a = reinterpret_cast<const f32x4_any*>(p)[0], b = reinterpret_cast<const f32x4_any*>(p)[1];
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = a[k], f[4 + k] = b[k];
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = k < n ? p[k] : 0.f;
}

// The sum over the TPR threads of a row, on each of them; `red` holds a float for each wave.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  if constexpr (TPR == 16) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    return v + dpp<0x140>(v);
  } else if constexpr (TPR == 64) {
    return wave_sum(v);
  } else {
    v = wave_sum(v);
    __syncthreads();  // whoever read the last row's sum has it
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) t += red[w];
    return t;
  }
}
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, float* red) {
  v = max16(v);
  if constexpr (TPR > 16) {
    const auto r16 = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)r16[0], (uint32_t)r16[1]);
    const auto r32 = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max((uint32_t)r32[0], (uint32_t)r32[1]);
  }
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = __uint_as_float(v);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) v = max(v, __float_as_uint(red[w]));
  }
  return v;
}

// The sum of a thread's squares, those of a vector by pairs, then the vectors: at most VPL + 3 roundings stand
// behind a square. (In one chain 31 squares below half a step of a first one were all lost: y off by 16 u, u = 2^-24,
// for 1.2. 8 sums side by side are as good, but with 129 registers for 127 the norm of 2048 columns to 8 bits
// would run 3 waves a SIMD for 4.)
template <int VPL, class F>
__device__ __forceinline__ float thread_squares(const float (&f)[VPL][8], F&& scaled) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    float p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = scaled(f[i][2 * j]), b = scaled(f[i][2 * j + 1]);
      p[j] = __builtin_fmaf(a, a, b * b);
    }
    const float t = (p[0] + p[1]) + (p[2] + p[3]);
    s = i == 0 ? t : s + t;
  }
  return s;
}

// 1 / sqrt(mean + eps) of a row whose squares add up to ss. Squares of finite values may
// pass fp32 (above 2^64): such a row is summed again divided by a power of two.
template <int TPR, int VPL>
__device__ __forceinline__ float row_rstd(float ss, const float (&f)[VPL][8], int D, float eps, float* red) {
  if (__builtin_expect(ss < __uint_as_float(kInfBits), 1)) return rsqrtf(ss / (float)D + eps);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < VPL; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, abs_bits(f[i][j]));
  m = row_max<TPR>(m, red);
  if (m >= kInfBits) return rsqrtf(ss);  // an infinity or a NaN among them: 0 or NaN
  const int e = (int)(m >> 23) - 127;    // the largest value's, about 63 and above
  const float t = thread_squares(f, [&](float x) { return __builtin_ldexpf(x, -e); });
  // eps * 2^-2e is far below one unit of the mean
  return __builtin_ldexpf(rsqrtf(row_sum<TPR>(t, red) / (float)D), -e);
}

struct RmsArgs {
  int rows, D;
  const void* x;
  int64_t ldx;
  const void* r;  // may be null
  int64_t ldr;
  void* s;        // x + r, where there is r
  int64_t lds;
  const float* gamma;
  float eps;
  void* y;        // in the type of x, or null
  int64_t ldy;
  float* rstd;    // may be null
  uint8_t* q;     // in 8 bits, or null
  int64_t ldq;
  uint8_t* sc;
  int64_t ldsc;
};

template <typename T, int TPR, int VPL, bool kF8>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_fwd_kernel(RmsArgs a) {
  constexpr int kThreads = TPR > 256 ? TPR : 256, RPB = kThreads / TPR;
  __shared__ float red[kThreads / 64];
  const int l = threadIdx.x % TPR;
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < a.rows; row += (int64_t)gridDim.x * RPB) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
    const bool over = a.D >= 8 && row + 1 < a.rows;
    Vec<T> xv[VPL], rv[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = (i * TPR + l) * 8;
      xv[i] = load_row(x + c, a.D - c, over);
    }
    if (a.r) {
      const T* r = reinterpret_cast<const T*>(a.r) + row * a.ldr;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int c = (i * TPR + l) * 8;
        rv[i] = load_row(r + c, a.D - c, over);
      }
    }
    float gam[VPL][8], f[VPL][8];
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = (i * TPR + l) * 8;
      load_gamma(a.gamma + c, a.D - c, gam[i]);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) unpack(xv[i], f[i]);
    if (a.r) {
      T* s = reinterpret_cast<T*>(a.s) + row * a.lds;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        float g[8];
        unpack(rv[i], g);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i][j] += g[j];
        const Vec<T> o = pack<T>(f[i]);
        const int c = (i * TPR + l) * 8;
        store_vec(s + c, o, a.D - c);
        unpack(o, f[i]);  // the norm is of what was stored
      }
    }
    if (a.D & 7) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) clear_tail(f[i], a.D - (i * TPR + l) * 8);
    }
    const float ss = thread_squares(f, [](float x) { return x; });
    const float rstd = row_rstd<TPR, VPL>(row_sum<TPR>(ss, red), f, a.D, a.eps, red);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = (i * TPR + l) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[i][j] = f[i][j] * rstd * gam[i][j];
      if constexpr (kF8) {
        // a block of 128 is 16 lanes' vectors; not rounded before it is quantised
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, c + j < a.D ? finite_abs_bits(f[i][j]) : 0u);
        const int byte = scale_byte(max16(m));
        if (c < (a.D + kB - 1) / kB * kB) {
#pragma unroll
          for (int j = 0; j < 8; ++j) f[i][j] = c + j < a.D ? f[i][j] : 0.f;
          *reinterpret_cast<u32x2*>(a.q + row * a.ldq + c) = u32x2{
              pack_e4m3x4(f[i][0], f[i][1], f[i][2], f[i][3], byte), pack_e4m3x4(f[i][4], f[i][5], f[i][6], f[i][7], byte)};
          if ((l & 15) == 0) a.sc[row * a.ldsc + c / kB] = (uint8_t)byte;
        }
      } else {
        store_vec(reinterpret_cast<T*>(a.y) + row * a.ldy + c, pack<T>(f[i]), a.D - c);
      }
    }
    if (a.rstd && l == 0) a.rstd[row] = rstd;
  }
}

struct RmsBwdArgs {
  int rows, D;
  const void* dy;
  int64_t lddy;
  const void* x;
  int64_t ldx;
  const float* rstd;
  const float* gamma;
  const void* dres;  // may be null
  int64_t lddres;
  void* dx;
  int64_t lddx;
  float* part;       // a partial row of dgamma for each workgroup, or null
};

template <typename T, int TPR, int VPL>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_bwd_kernel(RmsBwdArgs a) {
  constexpr int kThreads = TPR > 256 ? TPR : 256, RPB = kThreads / TPR;
  constexpr bool kAhead = VPL * sizeof(T) <= 4;  // the next row in flight while this one is computed
  constexpr int PITCH = TPR + 8;                 // writes of a wave and reads along columns on different banks
  __shared__ float red[kThreads / 64];
  __shared__ float sums[RPB > 1 ? RPB * 8 * PITCH : 1];
  const int l = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float gam[VPL][8], ag[VPL][8];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int c = (i * TPR + l) * 8;
    load_gamma(a.gamma + c, a.D - c, gam[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) ag[i][j] = 0.f;
  }
  struct Row {
    Vec<T> d[VPL], x[VPL], r[VPL];
    float rs;
  };
  auto fetch = [&](int64_t row, Row& w) __attribute__((always_inline)) {
    const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.lddy;
    const bool over = a.D >= 8 && row + 1 < a.rows;
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = (i * TPR + l) * 8;
      w.d[i] = load_row(dy + c, a.D - c, over);
      w.x[i] = load_row(x + c, a.D - c, over);
    }
    if (a.dres) {
      const T* r = reinterpret_cast<const T*>(a.dres) + row * a.lddres;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int c = (i * TPR + l) * 8;
        w.r[i] = load_row(r + c, a.D - c, over);
      }
    }
    w.rs = a.rstd[row];
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + sub;
  Row w, n;
  if (kAhead && row < a.rows) fetch(row, w);
  for (; row < a.rows; row += step) {
    if constexpr (kAhead) {
      if (row + step < a.rows) fetch(row + step, n);
    } else {
      fetch(row, w);
    }
    float xh[VPL][8], g[VPL][8];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      unpack(w.d[i], g[i]);
      unpack(w.x[i], xh[i]);
      if (a.D & 7) {
        clear_tail(g[i], a.D - (i * TPR + l) * 8);
        clear_tail(xh[i], a.D - (i * TPR + l) * 8);
      }
      float p[4];  // by pairs, as a row's squares are
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[i][j] *= w.rs;
        ag[i][j] = __builtin_fmaf(g[i][j], xh[i][j], ag[i][j]);
        g[i][j] *= gam[i][j];
        p[j >> 1] = j & 1 ? __builtin_fmaf(g[i][j], xh[i][j], p[j >> 1]) : g[i][j] * xh[i][j];
      }
      m += (p[0] + p[1]) + (p[2] + p[3]);
    }
    m = row_sum<TPR>(m, red) / (float)a.D;
    T* dx = reinterpret_cast<T*>(a.dx) + row * a.lddx;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int c = (i * TPR + l) * 8;
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = w.rs * (g[i][j] - xh[i][j] * m);
      if (a.dres) {
        float r[8];
        unpack(w.r[i], r);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += r[j];
      }
      store_vec(dx + c, pack<T>(o), a.D - c);
    }
    if constexpr (kAhead) w = n;
  }
  if (!a.part) return;
  float* part = a.part + (int64_t)blockIdx.x * a.D;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    if constexpr (RPB == 1) {
      const int c = (i * TPR + l) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < a.D) part[c + j] = ag[i][j];
    } else {
      // the rows' sums of a workgroup, added in order
      if (i > 0) __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) sums[(sub * 8 + j) * PITCH + l] = ag[i][j];
      __syncthreads();
      for (int e = threadIdx.x; e < TPR * 8; e += kThreads) {
        const int c = i * TPR * 8 + e;
        if (c >= a.D) break;
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < RPB; ++k) t += sums[(k * 8 + (e & 7)) * PITCH + (e >> 3)];
        part[c] = t;
      }
    }
  }
}

// out (+)= the sum of P partial rows (of dgamma, of a bias gradient), in a fixed order: a workgroup
// takes 16 columns, thread (ph, q) the rows ph, ph + 256, ... of columns 4q .. 4q+3; then the 16
// phases of a wave, then the 16 waves.
__global__ __launch_bounds__(1024) void row_sums_kernel(int P, int D, const float* __restrict__ part,
                                                       void* __restrict__ out, int bf16, int accumulate) {
  __shared__ float sums[16][17];
  const int q = threadIdx.x & 3, ph = threadIdx.x >> 2, c = blockIdx.x * 16 + q * 4, n = D - c;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (n >= 4) {
#pragma unroll 4
    for (int p = ph; p < P; p += 256) {
      const f32x4 v = *reinterpret_cast<const f32x4_any*>(part + (int64_t)p * D + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] += v[j];
    }
  } else {
    for (int p = ph; p < P; p += 256)
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (j < n) a[j] += part[(int64_t)p * D + c + j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    for (int o = 4; o < 64; o <<= 1) a[j] += __shfl_xor(a[j], o, 64);
    if ((threadIdx.x & 63) < 4) sums[threadIdx.x >> 6][q * 4 + j] = a[j];
  }
  __syncthreads();
  const int col = blockIdx.x * 16 + threadIdx.x;
  if (threadIdx.x < 16 && col < D) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += sums[w][threadIdx.x];
    if (bf16) {
      reinterpret_cast<uint16_t*>(out)[col] = f32_to_bf16(t);
    } else {
      float* o = reinterpret_cast<float*>(out) + col;
      *o = accumulate ? *o + t : t;
    }
  }
}

// Threads and vectors a row takes: 16 lanes up to 128 columns, a wave of as few vectors a lane as hold
// it up to 2048, beyond that 256 and from 8193 on 512 threads of up to 4.
template <class F>
void by_width(int D, F&& go) {
#define NL_W(TPR, VPL) go(std::integral_constant<int, TPR>{}, std::integral_constant<int, VPL>{})
  if (D <= 128) NL_W(16, 1);
  else if (D <= 512) NL_W(64, 1);
  else if (D <= 1024) NL_W(64, 2);
  else if (D <= 2048) NL_W(64, 4);
  else if (D <= 4096) NL_W(256, 2);
  else if (D <= 8192) NL_W(256, 4);
  else NL_W(512, 4);
#undef NL_W
}

int rows_per_block(int D) { return D <= 128 ? 16 : D <= 2048 ? 4 : 1; }

int bwd_blocks(int rows, int D) {
  // A partial row of dgamma each, written and read again. Measured (us, the gradients and the sum of
  // the partial rows) with 1024, 512 and 256 workgroups: 16384 x 512 bf16 10.9 + 4.3, 12.0 + 4.0,
  // 15.6 + 3.9; 16384 x 4096 92 + 7, 83 + 5, 110 + 5; 2048 x 8192 39 + 11, 28 + 7, 27 + 4.
  const int rpb = rows_per_block(D);
  return std::min((rows - 1) / rpb + 1, D <= 512 ? kBwdBlocks : D <= 4096 ? 512 : 256);
}

int check_rows(const char* what, int rows, int D, int dtype) {
  if (rows < 0 || D < 1 || D > kMaxRms)
    return nl_set_error(NL_EINVAL, std::string(what) + ": need rows >= 0 and 1 <= D <= 16384");
  if (dtype != NL_DTYPE_F32 && dtype != NL_DTYPE_BF16)
    return nl_set_error(NL_EINVAL, std::string(what) + ": rows are fp32 or bf16");
  return NL_OK;
}

// A matrix of `rows` rows of D elements: there, a row stride that keeps rows apart, aligned to its elements.
int check_matrix(const char* what, const char* name, const void* p, int64_t ld, int rows, int D, int elem) {
  if (!p) return nl_set_error(NL_EINVAL, std::string(what) + ": null " + name);
  if (rows > 1 && ld < D) return nl_set_error(NL_EINVAL, std::string(what) + ": rows of " + name + " overlap");
  if ((uintptr_t)p % elem) return nl_set_error(NL_EALIGN, std::string(what) + ": " + name + " is not aligned to its type");
  return NL_OK;
}

#define NL_TRY(x)          \
  do {                     \
    const int rc_ = (x);   \
    if (rc_) return rc_;   \
  } while (0)

int rms_forward(const char* what, void* stream, int dtype, bool f8, const RmsArgs& a) {
  NL_TRY(check_rows(what, a.rows, a.D, dtype));
  if (!(a.eps > 0.f) || !(a.eps <= 1.f)) return nl_set_error(NL_EINVAL, std::string(what) + ": need 0 < eps <= 1");
  if (a.rows == 0) return NL_OK;
  const int e = dtype == NL_DTYPE_BF16 ? 2 : 4;
  NL_TRY(check_matrix(what, "x", a.x, a.ldx, a.rows, a.D, e));
  NL_TRY(check_matrix(what, "gamma", a.gamma, a.D, 1, a.D, 4));
  if (a.r) {
    NL_TRY(check_matrix(what, "residual", a.r, a.ldr, a.rows, a.D, e));
    NL_TRY(check_matrix(what, "sum_out", a.s, a.lds, a.rows, a.D, e));
  }
  if (f8) {
    const int kb = (a.D + kB - 1) / kB;
    if (!a.q || !a.sc) return nl_set_error(NL_EINVAL, std::string(what) + ": null output");
    if (a.ldq < (int64_t)kb * kB || a.ldsc < kb)
      return nl_set_error(NL_EINVAL, std::string(what) + ": output rows hold whole blocks of 128 and their scales");
    if (a.ldq % 16 || ((uintptr_t)a.q & 15))
      return nl_set_error(NL_EALIGN, std::string(what) + ": values need 16-byte aligned rows");
  } else {
    NL_TRY(check_matrix(what, "y", a.y, a.ldy, a.rows, a.D, e));
  }
  by_width(a.D, [&](auto tpr, auto vpl) {
    constexpr int TPR = decltype(tpr)::value, VPL = decltype(vpl)::value;
    constexpr int kThreads = TPR > 256 ? TPR : 256, RPB = kThreads / TPR;
    const dim3 grid((unsigned)std::min<int64_t>(((int64_t)a.rows + RPB - 1) / RPB, 1 << 20)), block(kThreads);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == NL_DTYPE_BF16) {
      if (f8) hipLaunchKernelGGL((rms_fwd_kernel<uint16_t, TPR, VPL, true>), grid, block, 0, st, a);
      else hipLaunchKernelGGL((rms_fwd_kernel<uint16_t, TPR, VPL, false>), grid, block, 0, st, a);
    } else {
      if (f8) hipLaunchKernelGGL((rms_fwd_kernel<float, TPR, VPL, true>), grid, block, 0, st, a);
      else hipLaunchKernelGGL((rms_fwd_kernel<float, TPR, VPL, false>), grid, block, 0, st, a);
    }
  });
  return nl_check_launch(what);
}

}  // namespace
}  // namespace nl

void nl::launch_partial_sums(hipStream_t st, int P, int D, const float* part, void* out, int dtype, int accumulate) {
  hipLaunchKernelGGL(row_sums_kernel, dim3((unsigned)(((int64_t)D + 15) / 16)), dim3(1024), 0, st, P, D, part, out,
                     dtype == NL_DTYPE_BF16 ? 1 : 0, accumulate);
}

using namespace nl;

extern "C" int nl_rms_norm_fwd(void* stream, int rows, int D, int dtype, const void* x, int64_t ldx,
                               const void* residual, int64_t ldr, void* sum_out, int64_t ld_sum, const float* gamma,
                               float eps, void* y, int64_t ldy, float* rstd) {
  return rms_forward("nl_rms_norm_fwd", stream, dtype, false,
                     RmsArgs{rows, D, x, ldx, residual, ldr, sum_out, ld_sum, gamma, eps, y, ldy, rstd, nullptr, 0,
                             nullptr, 0});
}

extern "C" int nl_rms_norm_fp8(void* stream, int rows, int D, int dtype, const void* x, int64_t ldx,
                               const void* residual, int64_t ldr, void* sum_out, int64_t ld_sum, const float* gamma,
                               float eps, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds) {
  return rms_forward("nl_rms_norm_fp8", stream, dtype, true,
                     RmsArgs{rows, D, x, ldx, residual, ldr, sum_out, ld_sum, gamma, eps, nullptr, 0, nullptr, q, ldq,
                             scale, lds});
}

extern "C" size_t nl_rms_norm_bwd_ws_bytes(int rows, int D) {
  if (rows <= 0 || D < 1 || D > kMaxRms) return 0;
  return (size_t)bwd_blocks(rows, D) * D * sizeof(float);
}

extern "C" int nl_rms_norm_bwd(void* stream, int rows, int D, int dtype, const void* dy, int64_t lddy, const void* x,
                               int64_t ldx, const float* rstd, const float* gamma, const void* dres, int64_t lddres,
                               void* dx, int64_t lddx, float* dgamma, int accumulate, void* ws, size_t ws_bytes) {
  const char* what = "nl_rms_norm_bwd";
  NL_TRY(check_rows(what, rows, D, dtype));
  const int e = dtype == NL_DTYPE_BF16 ? 2 : 4;
  if (rows > 0) {
    NL_TRY(check_matrix(what, "dy", dy, lddy, rows, D, e));
    NL_TRY(check_matrix(what, "x", x, ldx, rows, D, e));
    NL_TRY(check_matrix(what, "dx", dx, lddx, rows, D, e));
    NL_TRY(check_matrix(what, "rstd", rstd, 1, 1, 1, 4));
    NL_TRY(check_matrix(what, "gamma", gamma, D, 1, D, 4));
    if (dres) NL_TRY(check_matrix(what, "dres", dres, lddres, rows, D, e));
    if (dgamma && (!ws || ws_bytes < nl_rms_norm_bwd_ws_bytes(rows, D)))
      return nl_set_error(NL_EINVAL, "nl_rms_norm_bwd: workspace smaller than nl_rms_norm_bwd_ws_bytes()");
    if ((uintptr_t)ws & 15) return nl_set_error(NL_EALIGN, "nl_rms_norm_bwd: workspace not 16-byte aligned");
  }
  if (dgamma && ((uintptr_t)dgamma & 3)) return nl_set_error(NL_EALIGN, "nl_rms_norm_bwd: dgamma is not aligned");
  if (rows == 0 && (!dgamma || accumulate)) return NL_OK;
  const int blocks = rows > 0 ? bwd_blocks(rows, D) : 0;
  const hipStream_t st = (hipStream_t)stream;
  if (rows > 0) {
    const RmsBwdArgs a{rows, D, dy, lddy, x, ldx, rstd, gamma, dres, lddres, dx, lddx, dgamma ? (float*)ws : nullptr};
    by_width(D, [&](auto tpr, auto vpl) {
      constexpr int TPR = decltype(tpr)::value, VPL = decltype(vpl)::value;
      const dim3 grid((unsigned)blocks), block(TPR > 256 ? TPR : 256);
      if (dtype == NL_DTYPE_BF16) hipLaunchKernelGGL((rms_bwd_kernel<uint16_t, TPR, VPL>), grid, block, 0, st, a);
      else hipLaunchKernelGGL((rms_bwd_kernel<float, TPR, VPL>), grid, block, 0, st, a);
    });
  }
  if (dgamma)
    launch_partial_sums(st, blocks, D, (const float*)ws, dgamma, NL_DTYPE_F32, accumulate);
  return nl_check_launch(what);
}
