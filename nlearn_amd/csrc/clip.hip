// clip.hip — the global L2 norm of many tensors of unlike sizes and types, and
// their clipping by it, as optax.clip_by_global_norm in front of AdamW has it
// (nlearn/train.py:502-506), for gradients that lie in tensors of their own:
//   n = sqrt(sum over all elements of g^2),   g -> g while n < max_norm, else (g / n) * max_norm
//
// Two passes over the gradients (the second needs the first one's sum), bound by
// HBM; the second starts where the first ended, with what the 256 MB cache still
// holds. The tensors' addresses travel as a kernel's arguments, 72 in a launch, so
// nothing is copied to the device and a captured graph keeps them; up to 72 tensors
// are two launches. The squares are summed in fp64 (a square passes fp32 at 2^64
// and vanishes below 2^-75; at 4 elements a clock and CU the fp64 units wait for
// HBM all the same), each workgroup's walk and the workgroups in a fixed order.
#include "common.h"

namespace nl {
namespace {

constexpr int kMost = 72;       // tensors in a launch: their table and the rest fit the 4 KiB of arguments
constexpr int kGrid = 1024;     // workgroups of the sums, a partial sum each
constexpr int kUnroll = 4;      // 16-byte vectors a thread has in flight
constexpr int kChunk = 256 * kUnroll * 2;  // vectors of one tensor that a workgroup takes at a time

typedef u32x4 __attribute__((aligned(2))) u32x4_any;

struct Leaf {
  const void* g;
  void* out;
  int64_t cols, ld, ldo;
  uint32_t rows;
  uint32_t chunk0_bf16;  // first chunk of this leaf * 2, + 1 for bf16
};
struct Table {
  Leaf leaf[kMost];
  int n;
  uint32_t chunks;
};
static_assert(sizeof(Table) <= 3700, "a kernel has 4 KiB of arguments");

// Calls go(leaf, bf16, vectors of a row, first vector, vectors) for the chunks b, b + step, ... of the table.
template <bool kBack, class F>
__device__ __forceinline__ void walk(const Table& t, F&& go) {
  for (uint32_t b = blockIdx.x; b < t.chunks; b += gridDim.x) {
    const uint32_t chunk = kBack ? t.chunks - 1 - b : b;
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((t.leaf[mid].chunk0_bf16 >> 1) <= chunk) lo = mid;
      else hi = mid - 1;
    }
    const Leaf& f = t.leaf[lo];
    const bool bf16 = f.chunk0_bf16 & 1;
    const int64_t vpr = (f.cols + (bf16 ? 7 : 3)) / (bf16 ? 8 : 4);
    const int64_t first = (int64_t)(chunk - (f.chunk0_bf16 >> 1)) * kChunk;
    const int64_t all = vpr * f.rows;
    go(f, bf16, vpr, first, (int)(all - first < kChunk ? all - first : kChunk));
  }
}

// Where vector i of a chunk lies: its row, its first column. Rows are counted from the chunk's first.
struct Place {
  int64_t row0, col0;  // of the chunk's first vector
  uint32_t vpr;        // 0: one row
};
__device__ __forceinline__ Place place(const Leaf& f, int64_t vpr, int64_t first) {
  if (f.rows == 1) return {0, first, 0};
  const int64_t r = first / vpr;
  return {r, first - r * vpr, (uint32_t)vpr};
}
__device__ __forceinline__ void at(const Place& p, int i, int64_t& row, int64_t& col) {
  row = p.row0;
  col = p.col0 + i;
  if (p.vpr) {
    const uint32_t d = (uint32_t)col / p.vpr;
    row += d;
    col = (uint32_t)col - d * p.vpr;
  }
}

// 16 bytes of a row's vector, zero past its end
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p, int64_t left) {
  constexpr int V = 16 / sizeof(T);
  if (left >= V) return *reinterpret_cast<const u32x4_any*>(p);
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int k = 0; k < V - 1; ++k) {
    if (k >= left) continue;
    if constexpr (sizeof(T) == 2) v[k >> 1] |= (uint32_t)p[k] << (16 * (k & 1));
    else v[k] = __float_as_uint(p[k]);
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const u32x4& v, int64_t left) {
  constexpr int V = 16 / sizeof(T);
  if (left >= V) {
    *reinterpret_cast<u32x4_any*>(p) = v;
    return;
  }
#pragma unroll
  for (int k = 0; k < V - 1; ++k) {
    if (k >= left) continue;
    if constexpr (sizeof(T) == 2) p[k] = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
    else p[k] = __uint_as_float(v[k]);
  }
}

template <typename T>
__device__ __forceinline__ double squares(const u32x4& v) {
  double s = 0.0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (sizeof(T) == 2) {
      const double a = bf16_lo(v[q]), b = bf16_hi(v[q]);
      s = __builtin_fma(a, a, s);
      s = __builtin_fma(b, b, s);
    } else {
      const double a = __uint_as_float(v[q]);
      s = __builtin_fma(a, a, s);
    }
  }
  return s;
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const Leaf& f, int64_t vpr, int64_t first, int n) {
  const Place p = place(f, vpr, first);
  const T* g = reinterpret_cast<const T*>(f.g);
  double s = 0.0;
  for (int i0 = threadIdx.x; i0 < n; i0 += 256 * kUnroll) {
    u32x4 v[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int i = i0 + k * 256;
      int64_t row, col;
      at(p, i, row, col);
      col *= 16 / (int)sizeof(T);
      v[k] = i < n ? load16<T>(g + row * f.ld + col, f.cols - col) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) s += squares<T>(v[k]);
  }
  return s;
}

// The sum over a workgroup of 256, on every thread.
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// part[b] (+)= the squares of workgroup b's chunks
__global__ __launch_bounds__(256) void norm_parts_kernel(Table t, double* __restrict__ part, int add) {
  __shared__ double red[4];
  double s = 0.0;
  walk<false>(t, [&](const Leaf& f, bool bf16, int64_t vpr, int64_t first, int n) __attribute__((always_inline)) {
    s += bf16 ? chunk_squares<uint16_t>(f, vpr, first, n) : chunk_squares<float>(f, vpr, first, n);
  });
  s = block_sum(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = add ? part[blockIdx.x] + s : s;
}

// sqrt of the sum of the partial sums, the same on every thread of every workgroup
__device__ __forceinline__ float norm_of(const double* __restrict__ part, int parts, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) s += part[i];
  return (float)__builtin_sqrt(block_sum(s, red));
}

__global__ __launch_bounds__(256) void norm_kernel(const double* __restrict__ part, int parts, float* __restrict__ out) {
  __shared__ double red[4];
  const float n = norm_of(part, parts, red);
  if (threadIdx.x == 0) *out = n;
}

template <typename T>
__device__ __forceinline__ void chunk_clip(const Leaf& f, int64_t vpr, int64_t first, int n, bool clip, float norm,
                                           float most) {
  const Place p = place(f, vpr, first);
  const T* g = reinterpret_cast<const T*>(f.g);
  T* out = reinterpret_cast<T*>(f.out);
  auto scaled = [&](float x) { return clip ? (x / norm) * most : x; };
  for (int i0 = threadIdx.x; i0 < n; i0 += 256 * kUnroll) {
    u32x4 v[kUnroll];
    int64_t row[kUnroll], col[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const int i = i0 + k * 256;
      at(p, i, row[k], col[k]);
      col[k] *= 16 / (int)sizeof(T);
      v[k] = i < n ? load16<T>(g + row[k] * f.ld + col[k], f.cols - col[k]) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      if (i0 + k * 256 >= n) continue;
      u32x4 o;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if constexpr (sizeof(T) == 2) o[q] = pack_bf16x2(scaled(bf16_lo(v[k][q])), scaled(bf16_hi(v[k][q])));
        else o[q] = __float_as_uint(scaled(__uint_as_float(v[k][q])));
      }
      store16<T>(out + row[k] * f.ldo + col[k], o, f.cols - col[k]);
    }
  }
}

__global__ __launch_bounds__(256) void clip_kernel(Table t, const double* __restrict__ part, int parts, float most,
                                                   float* __restrict__ norm_out, int in_place) {
  __shared__ double red[4];
  const float norm = norm_of(part, parts, red);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  const bool clip = !(norm < most);
  if (!clip && in_place) return;
  walk<true>(t, [&](const Leaf& f, bool bf16, int64_t vpr, int64_t first, int n) __attribute__((always_inline)) {
    if (bf16) chunk_clip<uint16_t>(f, vpr, first, n, clip, norm, most);
    else chunk_clip<float>(f, vpr, first, n, clip, norm, most);
  });
}

int check_leaf(const nl_grad_tensor& t, bool out) {
  if (t.rows < 0 || t.cols < 0) return nl_set_error(NL_EINVAL, "global_norm: negative size");
  if (t.dtype != NL_DTYPE_F32 && t.dtype != NL_DTYPE_BF16)
    return nl_set_error(NL_EINVAL, "global_norm: tensors are fp32 or bf16");
  if (t.rows == 0 || t.cols == 0) return NL_OK;
  const int e = t.dtype == NL_DTYPE_BF16 ? 2 : 4;
  if (!t.g || (out && !t.out)) return nl_set_error(NL_EINVAL, "global_norm: null pointer");
  if ((uintptr_t)t.g % e || (out && (uintptr_t)t.out % e))
    return nl_set_error(NL_EALIGN, "global_norm: a tensor is not aligned to its type");
  if (t.rows > 1 && (t.ld < t.cols || (out && t.ld_out < t.cols)))
    return nl_set_error(NL_EINVAL, "global_norm: rows overlap");
  if (out && t.out == t.g && t.rows > 1 && t.ld != t.ld_out)
    return nl_set_error(NL_EINVAL, "global_norm: a result in place has the input's row stride");
  // rows are counted in 32 bits, and a chunk's vectors within its rows
  if (t.rows > INT32_MAX || (t.rows > 1 && t.cols > INT32_MAX) || t.cols > (int64_t)1 << 40)
    return nl_set_error(NL_EUNSUPPORTED, "global_norm: rows of a matrix and their lengths are below 2^31");
  return NL_OK;
}

// The tables of all launches, one after the other: go(table) for each, at least one.
template <class F>
int tables(int n, const nl_grad_tensor* tensors, F&& go) {
  Table t;
  t.n = 0;
  t.chunks = 0;
  bool any = false;
  for (int i = 0; i < n; ++i) {
    const nl_grad_tensor& s = tensors[i];
    if (s.rows == 0 || s.cols == 0) continue;
    const int v = s.dtype == NL_DTYPE_BF16 ? 8 : 4;
    const int64_t chunks = (s.rows * ((s.cols + v - 1) / v) + kChunk - 1) / kChunk;
    if (t.n == kMost || (t.n && t.chunks + chunks > INT32_MAX)) {
      go(t);
      any = true;
      t.n = 0;
      t.chunks = 0;
    }
    if (chunks > INT32_MAX) return nl_set_error(NL_EUNSUPPORTED, "global_norm: a tensor of more than 2^44 bytes");
    t.leaf[t.n++] = Leaf{s.g, s.out, s.cols, s.ld, s.ld_out, (uint32_t)s.rows,
                         t.chunks << 1 | (s.dtype == NL_DTYPE_BF16 ? 1u : 0u)};
    t.chunks += (uint32_t)chunks;
  }
  if (t.n || !any) go(t);
  return NL_OK;
}

int check_all(int n, const nl_grad_tensor* tensors, bool out, float* norm, void* ws, size_t ws_bytes) {
  if (n < 0 || (n > 0 && !tensors)) return nl_set_error(NL_EINVAL, "global_norm: bad table");
  if (!norm) return nl_set_error(NL_EINVAL, "global_norm: null norm");
  if ((uintptr_t)norm & 3) return nl_set_error(NL_EALIGN, "global_norm: norm is not aligned");
  if (!ws || ws_bytes < NL_GLOBAL_NORM_MULTI_WS)
    return nl_set_error(NL_EINVAL, "global_norm: workspace smaller than NL_GLOBAL_NORM_MULTI_WS");
  if ((uintptr_t)ws & 7) return nl_set_error(NL_EALIGN, "global_norm: workspace not 8-byte aligned");
  for (int i = 0; i < n; ++i)
    if (int rc = check_leaf(tensors[i], out)) return rc;
  return NL_OK;
}

static_assert(NL_GLOBAL_NORM_MULTI_WS == kGrid * sizeof(double), "a partial sum for each workgroup");

// The partial sums of all tensors; *parts: how many there are. Every launch has the same workgroups.
int sums(hipStream_t st, int n, const nl_grad_tensor* tensors, double* part, int* parts) {
  uint32_t most = 1;
  if (int rc = tables(n, tensors, [&](const Table& t) { most = std::max(most, t.chunks); })) return rc;
  *parts = (int)std::min<uint32_t>(most, kGrid);
  int add = 0;
  return tables(n, tensors, [&](const Table& t) {
    hipLaunchKernelGGL(norm_parts_kernel, dim3((unsigned)*parts), dim3(256), 0, st, t, part, add);
    add = 1;
  });
}

}  // namespace
}  // namespace nl

using namespace nl;

extern "C" int nl_global_norm_multi(void* stream, int n, const nl_grad_tensor* tensors, float* norm, void* ws,
                                    size_t ws_bytes) {
  if (int rc = check_all(n, tensors, false, norm, ws, ws_bytes)) return rc;
  int parts = 0;
  if (int rc = sums((hipStream_t)stream, n, tensors, (double*)ws, &parts)) return rc;
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, (const double*)ws, parts, norm);
  return nl_check_launch("nl_global_norm_multi");
}

extern "C" int nl_clip_by_global_norm(void* stream, int n, const nl_grad_tensor* tensors, float max_norm, float* norm,
                                      void* ws, size_t ws_bytes) {
  if (!(max_norm > 0.f)) return nl_set_error(NL_EINVAL, "clip_by_global_norm: max_norm must be > 0");
  if (int rc = check_all(n, tensors, true, norm, ws, ws_bytes)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  int parts = 0, in_place = 1;
  for (int i = 0; i < n; ++i) in_place &= tensors[i].out == tensors[i].g;
  if (int rc = sums(st, n, tensors, (double*)ws, &parts)) return rc;
  if (int rc = tables(n, tensors, [&](const Table& t) {
        hipLaunchKernelGGL(clip_kernel, dim3(std::max(1u, std::min<uint32_t>(t.chunks, 2 * kGrid))), dim3(256), 0, st,
                           t, (const double*)ws, parts, max_norm, norm, in_place);
      }))
    return rc;
  return nl_check_launch("nl_clip_by_global_norm");
}
