// clip.hip — the global L2 norm of many tensors of unlike sizes and types, and
// their clipping by it, as optax.clip_by_global_norm in front of AdamW has it
// (nlearn/train.py:502-506), for gradients that lie in tensors of their own:
//   n = sqrt(sum over all elements of g^2),   g -> g while n < max_norm, else (g / n) * max_norm
//
// Two passes over the gradients (the second needs the first one's sum), bound by
// HBM (medians of a kernel trace over three sets of tensors in turn): 46 tensors of 263 MB,
// fp32 and bf16, 50 us for the sums (5.2 TB/s; at least 47) and 85 us for the second pass
// (527 MB, 6.2 TB/s with what the 256 MB cache still holds of them: it starts where the
// first ended; at least 82). Results are stored past the caches: the
// sums of the next call took 99 us, not 72, beside the write-back of dirty lines.
// Rows that end inside a vector read into the next row: element by element the sums
// took 70 us. The tensors' addresses travel as a kernel's arguments, 64 in a launch,
// so nothing is copied to the device and a captured graph keeps them; up to 64
// tensors are two launches (18 small ones: 4.2 + 5.7 us). The squares are summed in
// fp64 (a square passes fp32 at 2^64 and vanishes below 2^-75; at 4 elements a clock
// and CU the fp64 units wait for HBM all the same), each workgroup's walk and the
// workgroups in a fixed order.
#include "common.h"

namespace nl {
namespace {

constexpr int kMost = 64;       // tensors in a launch: one a lane, and their table fits the 4 KiB of arguments
constexpr int kGrid = 1024;     // workgroups of the sums, a partial sum each
constexpr int kVecs = 4;        // 16-byte vectors of a chunk that a thread takes, all in flight together
constexpr int kChunk = 256 * kVecs;  // vectors of one tensor that a workgroup takes at a time

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
  // each lane knows a leaf's first chunk: one comparison finds a chunk's leaf
  const int lane = threadIdx.x & 63;
  const uint32_t start = lane < t.n ? t.leaf[lane].chunk0_bf16 >> 1 : 0xffffffffu;
  for (uint32_t b = blockIdx.x; b < t.chunks; b += gridDim.x) {
    const uint32_t chunk = kBack ? t.chunks - 1 - b : b;
    const int lo = __builtin_amdgcn_readfirstlane(__popcll(__ballot(start <= chunk)) - 1);
    const Leaf& f = t.leaf[lo];
    const bool bf16 = f.chunk0_bf16 & 1;
    const int64_t vpr = (f.cols + (bf16 ? 7 : 3)) / (bf16 ? 8 : 4);
    const int64_t first = (int64_t)(chunk - (f.chunk0_bf16 >> 1)) * kChunk;
    const int64_t all = vpr * f.rows;
    go(f, bf16, vpr, first, (int)(all - first < kChunk ? all - first : kChunk));
  }
}

// Where a thread's vectors of a chunk lie: their row and first column, and the elements of the row
// from there on (0 or less: no such vector). go(k, row, column, left) for each.
template <int V, class F>
__device__ __forceinline__ void places(const Leaf& f, int64_t vpr, int64_t first, int n, F&& go) {
  const uint32_t tid = threadIdx.x;
  if (f.rows == 1) {
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
      const int64_t col = (first + tid + k * 256) * V;
      go(k, (int64_t)0, col, (int)(tid + k * 256) < n ? f.cols - col : 0);
    }
    return;
  }
  // rows and columns (in vectors) counted from the chunk's first row, where 32 bits hold them
  const int64_t row0 = first / vpr;
  const uint32_t w = (uint32_t)vpr;
  const uint32_t at = (uint32_t)(first - row0 * vpr) + tid;
  uint32_t row = at / w, col = at - row * w;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    go(k, row0 + row, (int64_t)col * V, (int)(tid + k * 256) < n ? f.cols - (int64_t)col * V : 0);
    col += 256;
    if (w >= 256) {  // the next row at most
      if (col >= w) col -= w, ++row;
    } else {
      const uint32_t d = col / w;
      row += d;
      col -= d * w;
    }
  }
}

// 16 bytes at p, `left` elements of which are the row's (0 or less: none). `over`: what lies behind a
// row may be read (it is the next row's): a load element by element waits for each, and where rows
// are a few vectors long one of them ends in most waves' loads.
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p, int64_t left, bool over) {
  constexpr int V = 16 / sizeof(T);
  if (left >= V || (over && left > 0)) return *reinterpret_cast<const u32x4_any*>(p);
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
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(p));
    return;
  }
#pragma unroll
  for (int k = 0; k < V - 1; ++k) {
    if (k >= left) continue;
    if constexpr (sizeof(T) == 2) p[k] = (uint16_t)(v[k >> 1] >> (16 * (k & 1)));
    else p[k] = __uint_as_float(v[k]);
  }
}

// zero past the row's last element
template <typename T>
__device__ __forceinline__ void mask16(u32x4& v, int left) {
  constexpr int V = 16 / sizeof(T);
  if (left >= V) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (sizeof(T) == 2) v[q] = left >= 2 * q + 2 ? v[q] : left == 2 * q + 1 ? v[q] & 0xffffu : 0u;
    else v[q] = left > q ? v[q] : 0u;
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

// Whether a chunk is whole vectors of one row
template <int V>
__device__ __forceinline__ bool plain(const Leaf& f, int64_t first, int n) {
  return f.rows == 1 && n == kChunk && (first + kChunk) * V <= f.cols;
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const Leaf& f, int64_t vpr, int64_t first, int n) {
  constexpr int V = 16 / sizeof(T);
  const T* g = reinterpret_cast<const T*>(f.g);
  u32x4 v[kVecs];
  if (plain<V>(f, first, n)) {
    const T* p = g + first * V + threadIdx.x * V;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) v[k] = *reinterpret_cast<const u32x4_any*>(p + k * 256 * V);
  } else {
    int rest[kVecs];
    places<V>(f, vpr, first, n, [&](int k, int64_t row, int64_t col, int64_t left) __attribute__((always_inline)) {
      v[k] = load16<T>(g + row * f.ld + col, left, f.cols >= V && row + 1 < f.rows);
      rest[k] = (int)(left < V ? left : V);
    });
#pragma unroll
    for (int k = 0; k < kVecs; ++k) mask16<T>(v[k], rest[k]);
  }
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) s += squares<T>(v[k]);
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
  constexpr int V = 16 / sizeof(T);
  const T* g = reinterpret_cast<const T*>(f.g);
  T* out = reinterpret_cast<T*>(f.out);
  auto scaled = [&](const u32x4& v) __attribute__((always_inline)) {
    auto one = [&](float x) __attribute__((always_inline)) { return clip ? (x / norm) * most : x; };
    u32x4 o;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (sizeof(T) == 2) o[q] = pack_bf16x2(one(bf16_lo(v[q])), one(bf16_hi(v[q])));
      else o[q] = __float_as_uint(one(__uint_as_float(v[q])));
    }
    return o;
  };
  u32x4 v[kVecs];
  if (plain<V>(f, first, n)) {
    const int64_t at = first * V + threadIdx.x * V;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) v[k] = *reinterpret_cast<const u32x4_any*>(g + at + k * 256 * V);
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
      __builtin_nontemporal_store(scaled(v[k]), reinterpret_cast<u32x4_any*>(out + at + k * 256 * V));
    return;
  }
  places<V>(f, vpr, first, n, [&](int k, int64_t row, int64_t col, int64_t left) __attribute__((always_inline)) {
    v[k] = load16<T>(g + row * f.ld + col, left, f.cols >= V && row + 1 < f.rows);
  });
  places<V>(f, vpr, first, n, [&](int k, int64_t row, int64_t col, int64_t left) __attribute__((always_inline)) {
    store16<T>(out + row * f.ldo + col, scaled(v[k]), left);
  });
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
        const dim3 grid(std::max(1u, std::min<uint32_t>(t.chunks, 2 * kGrid)));
        hipLaunchKernelGGL(clip_kernel, grid, dim3(256), 0, st, t, (const double*)ws, parts, max_norm, norm, in_place);
      }))
    return rc;
  return nl_check_launch("nl_clip_by_global_norm");
}
